// Index rules of the paged int8 KV cache, apart from the kernels: plain
// arithmetic that the kernels run and a host test can ask without a GPU.
//
// A pool of `blocks` blocks of bs tokens (bs 16, 32, 64 or 128).  Block i holds
// codes [k, v][Hkv][bs * D], k as [bs][D] and v as [D][bs], and scales
// [k, v][Hkv].  Token slot s is entry s % bs of block s / bs.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define NNHIP_HD __host__ __device__
#else
#define NNHIP_HD
#endif

namespace nnhip {

// Most requests of one call: their offsets lie in LDS.
constexpr int kMaxRequests = 4096;

struct PagedPool {
  int blocks = 0, bs = 0, lbs = 0, Hkv = 0, D = 0;  // lbs: log2(bs)
};

NNHIP_HD inline int log2_block(int bs) {
  return bs == 16 ? 4 : bs == 32 ? 5 : bs == 64 ? 6 : bs == 128 ? 7 : -1;
}

// Codes of one (block, head) of k or v.
NNHIP_HD inline int64_t head_elems(const PagedPool &p) { return (int64_t)p.D << p.lbs; }
// First code of (block, kv, head); kv 0: k, 1: v.
NNHIP_HD inline int64_t head_offset(const PagedPool &p, int block, int kv, int h) {
  return (((int64_t)block * 2 + kv) * p.Hkv + h) * head_elems(p);
}
NNHIP_HD inline int64_t scale_offset(const PagedPool &p, int block, int kv, int h) {
  return ((int64_t)block * 2 + kv) * p.Hkv + h;
}
NNHIP_HD inline bool slot_ok(const PagedPool &p, int slot) {
  return slot >= 0 && slot < ((int64_t)p.blocks << p.lbs);
}
NNHIP_HD inline bool block_ok(int block, int blocks) { return block >= 0 && block < blocks; }

// Rows [first, last) of request b, of `rows` rows in all; row_start is read as
// it comes: rows outside [0, rows) are no rows.
struct RowRange { int first, last; };
NNHIP_HD inline RowRange request_rows(const int32_t *row_start, int b, int rows) {
  int a = row_start[b], z = row_start[b + 1];
  a = a < 0 ? 0 : a > rows ? rows : a;
  z = z < a ? a : z > rows ? rows : z;
  return RowRange{a, z};
}
// Tokens of a request that its table row can name.
NNHIP_HD inline int64_t request_len(int len, int max_blocks, int lbs) {
  const int64_t most = (int64_t)max_blocks << lbs;
  return len < 0 ? 0 : len > most ? most : len;
}

// What one request asks of the block tables: the status it alone would give
// (0: none), the blocks it needs, returns and takes.
struct BlockNeed { int status, need, back, take; };
NNHIP_HD inline BlockNeed block_need(int cached, int added, int held, int lbs, int max_blocks) {
  if (cached < 0 || added < 0) return BlockNeed{1, 0, 0, 0};
  const int64_t len = (int64_t)cached + added;
  if (len > (int64_t)max_blocks << lbs) return BlockNeed{2, 0, 0, 0};
  if (held < 0 || held > max_blocks) return BlockNeed{5, 0, 0, 0};
  const int need = (int)((len + (1 << lbs) - 1) >> lbs);
  return BlockNeed{0, need, held > need ? held - need : 0, need > held ? need - held : 0};
}
// Status of a whole call from the requests' lowest nonzero one and the totals.
NNHIP_HD inline int tables_status(int worst, int64_t rows, int64_t room, int64_t back, int64_t take,
                                  int64_t free_count, int blocks) {
  if (worst == 1 || worst == 2) return worst;
  if (rows > room) return 3;
  if (worst || free_count < 0 || free_count + back > blocks) return 5;
  return take > free_count + back ? 4 : 0;
}

// The scale of a (block, k or v, head): the smallest power of two 2^e, e >=
// -126, with amax <= 127 * 2^e, and 0 for amax = 0.  A power of two, so that a
// code times its scale and a code moved to a larger scale are exact but for the
// one rounding to a whole code, and the older codes of a block that grows
// several times are off by less than one step in all (1/2 + 1/4 + ...).
NNHIP_HD inline double block_scale(double amax) {
  if (!(amax > 0)) return 0.0;
  union { double d; uint64_t u; } a{amax}, s;
  int e = (int)(a.u >> 52) - 1023 - 6;             // amax in [64, 128) * 2^e
  s.u = (uint64_t)(e + 1023) << 52;
  if (amax > 127.0 * s.d) ++e;
  if (e < -126) e = -126;
  s.u = (uint64_t)(e + 1023) << 52;
  return s.d;
}

}  // namespace nnhip
