// The paged cache's index rules (csrc/paged.hpp) for a test to ask.
#include "paged.hpp"

extern "C" {
int log2_block(int bs) { return nnhip::log2_block(bs); }
double block_scale(double amax) { return nnhip::block_scale(amax); }
int slot_ok(int blocks, int bs, int slot) {
  nnhip::PagedPool p;
  p.blocks = blocks; p.bs = bs; p.lbs = nnhip::log2_block(bs);
  return nnhip::slot_ok(p, slot);
}
int block_ok(int block, int blocks) { return nnhip::block_ok(block, blocks); }
long long head_offset(int blocks, int bs, int Hkv, int D, int block, int kv, int h) {
  nnhip::PagedPool p;
  p.blocks = blocks; p.bs = bs; p.lbs = nnhip::log2_block(bs); p.Hkv = Hkv; p.D = D;
  return nnhip::head_offset(p, block, kv, h);
}
void request_rows(const int *row_start, int b, int rows, int *out) {
  const nnhip::RowRange r = nnhip::request_rows(row_start, b, rows);
  out[0] = r.first; out[1] = r.last;
}
long long request_len(int len, int max_blocks, int lbs) {
  return nnhip::request_len(len, max_blocks, lbs);
}
int tables_status(int B, const int *cached, const int *added, const int *held, int bs,
                  int max_blocks, long long room, long long free_count, int blocks) {
  long long rows = 0, back = 0, take = 0;
  int worst = 0;
  for (int b = 0; b < B; ++b) {
    const nnhip::BlockNeed n =
        nnhip::block_need(cached[b], added[b], held[b], nnhip::log2_block(bs), max_blocks);
    if (n.status && (!worst || n.status < worst)) worst = n.status;
    rows += added[b]; back += n.back; take += n.take;
  }
  return nnhip::tables_status(worst, rows, room, back, take, free_count, blocks);
}
}
