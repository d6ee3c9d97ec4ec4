// C ABI of the paged int8 KV cache (include/nnhip.h, "paged int8 KV cache"):
// argument checks; the kernels are in paged.hip.
#include "api_common.hpp"

#include <climits>

using nnhip::guard;

namespace {

#define REQ(cond, msg) NNHIP_REQUIRE((cond), nnhip::kErrArg, (msg))

void set_device(const nnhip_ctx *ctx) { NNHIP_CHECK(hipSetDevice(ctx->c.device)); }

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int block_shift(int block_size, const char *what) {
  const int l = nnhip::log2_block(block_size);
  REQ(l > 0, std::string(what) + ": block_size must be 16, 32, 64 or 128");
  return l;
}

nnhip::PagedPool pool_of(int block_size, int num_blocks, int Hkv, int D, const void *codes,
                         const void *scales, const char *what) {
  nnhip::PagedPool p;
  p.bs = block_size;
  p.lbs = block_shift(block_size, what);
  p.blocks = num_blocks;
  p.Hkv = Hkv;
  p.D = D;
  REQ(codes && scales, std::string(what) + ": NULL argument");
  REQ(num_blocks > 0 && (int64_t)num_blocks * block_size <= INT32_MAX,
      std::string(what) + ": num_blocks must be positive, with at most 2^31 - 1 token slots");
  REQ(Hkv > 0 && Hkv <= 4096, std::string(what) + ": Hkv out of range");
  REQ((int64_t)num_blocks * 2 * Hkv <= INT32_MAX,
      std::string(what) + ": num_blocks * Hkv must be below 2^30");
  NNHIP_REQUIRE(D == 32 || D == 64 || D == 128, nnhip::kErrUnsupported,
                std::string(what) + ": head dim must be 32, 64 or 128");
  REQ(aligned(codes, 16) && aligned(scales, 4), std::string(what) + ": codes must be aligned to 16 bytes");
  return p;
}

// n zeros in `b`, which is set only once they are under way.
void zeroed(nnhip::DevBuf<unsigned> &b, size_t n, hipStream_t st) {
  nnhip::DevBuf<unsigned> z(n);
  NNHIP_CHECK(hipMemsetAsync(z.p, 0, z.bytes(), st));
  b = std::move(z);
}

void check_heads(int H, int Hkv, const char *what) {
  REQ(H > 0 && H <= 65535 && H % Hkv == 0, std::string(what) + ": H must be a multiple of Hkv");
}

}  // namespace

extern "C" {

int nnhip_block_tables(nnhip_ctx *ctx, int B, const int32_t *cached, const int32_t *added,
                       int block_size, int max_blocks, int32_t *tables, int32_t *held,
                       int num_blocks, int32_t *free_list, int32_t *free_count, int T,
                       int32_t *row_start, int32_t *lens, int32_t *pos, int32_t *slots,
                       int32_t *status) {
  return guard([&] {
    const char *what = "nnhip_block_tables";
    REQ(B > 0 && B <= nnhip::kMaxRequests, "nnhip_block_tables: B must be in [1, 4096]");
    const int lbs = block_shift(block_size, what);
    REQ(num_blocks > 0 && (int64_t)num_blocks * block_size <= INT32_MAX,
        "nnhip_block_tables: num_blocks must be positive, with at most 2^31 - 1 token slots");
    REQ(max_blocks > 0 && (int64_t)max_blocks * block_size <= 1 << 30,
        "nnhip_block_tables: max_blocks must be positive, with at most 2^30 tokens a request");
    REQ(T >= 0, "nnhip_block_tables: T is negative");
    REQ(ctx && cached && added && tables && held && free_list && free_count && row_start && lens &&
            status && ((pos && slots) || T == 0),
        "nnhip_block_tables: NULL argument");
    set_device(ctx);
    hipStream_t st = ctx->c.stream;
    if (!ctx->ticket.p) zeroed(ctx->ticket, 1, st);
    nnhip::launch_block_tables(st, B, cached, added, lbs, max_blocks, tables, held, num_blocks,
                               free_list, free_count, T, row_start, lens, pos, slots, status,
                               ctx->ticket.p);
  });
}

int nnhip_rope_kv_append_paged_q8(nnhip_ctx *ctx, const float *qkv, int T, int H, int Hkv, int D,
                                  const int32_t *pos, const int32_t *slots, const float *cos_t,
                                  const float *sin_t, int n_pos, float *q_out, int8_t *codes,
                                  float *scales, int block_size, int num_blocks) {
  return guard([&] {
    const char *what = "nnhip_rope_kv_append_paged_q8";
    const nnhip::PagedPool p = pool_of(block_size, num_blocks, Hkv, D, codes, scales, what);
    check_heads(H, Hkv, what);
    REQ(n_pos > 0 && !cos_t == !sin_t,
        "nnhip_rope_kv_append_paged_q8: n_pos must be positive, cos and sin both given or neither");
    REQ(aligned(qkv, 16) && aligned(q_out, 16) && aligned(cos_t, 8) && aligned(sin_t, 8),
        "nnhip_rope_kv_append_paged_q8: qkv and q_out must be aligned to 16 bytes, cos and sin to 8");
    REQ(ctx && T >= 0 && ((qkv && pos && slots && q_out) || T == 0),
        "nnhip_rope_kv_append_paged_q8: NULL argument or negative T");
    if (T == 0) return;
    set_device(ctx);
    if (!cos_t) {
      const nnhip_ctx::Rope &rt = nnhip::ctx_rope(ctx, n_pos, D);
      cos_t = rt.c.p;
      sin_t = rt.s.p;
    }
    nnhip::launch_rope_append_paged(ctx->c.stream, qkv, T, H, p, pos, slots, cos_t, sin_t, n_pos,
                                    q_out, codes, scales);
  });
}

int nnhip_attention_paged_q8(nnhip_ctx *ctx, const float *q, int T, const int8_t *codes,
                             const float *scales, int block_size, int num_blocks,
                             const int32_t *tables, int max_blocks, const int32_t *row_start,
                             const int32_t *lens, int B, int H, int Hkv, int D, float *out) {
  return guard([&] {
    const char *what = "nnhip_attention_paged_q8";
    const nnhip::PagedPool p = pool_of(block_size, num_blocks, Hkv, D, codes, scales, what);
    check_heads(H, Hkv, what);
    REQ(B > 0 && B <= nnhip::kMaxRequests, "nnhip_attention_paged_q8: B must be in [1, 4096]");
    REQ(max_blocks > 0 && (int64_t)max_blocks * block_size <= 1 << 30,
        "nnhip_attention_paged_q8: max_blocks must be positive, with at most 2^30 tokens a request");
    REQ(aligned(q, 16) && aligned(out, 16),
        "nnhip_attention_paged_q8: q and out must be aligned to 16 bytes");
    REQ(ctx && tables && row_start && lens && T >= 0 && ((q && out) || T == 0),
        "nnhip_attention_paged_q8: NULL argument or negative T");
    if (T == 0) return;
    REQ((int64_t)T * H <= INT32_MAX, "nnhip_attention_paged_q8: more than 2^31 - 1 rows of heads");
    set_device(ctx);
    hipStream_t st = ctx->c.stream;
    if (!ctx->paged_tickets.p) zeroed(ctx->paged_tickets, nnhip::attention_paged_tickets(), st);
    const size_t need = (size_t)nnhip::attention_paged_part_elems(D);
    if (need > ctx->paged_part.n) {
      NNHIP_CHECK(hipStreamSynchronize(st));   // earlier calls may read it
      ctx->paged_part.ensure(need);
    }
    nnhip::launch_attention_paged(st, q, T, codes, scales, p, tables, max_blocks, row_start, lens, B,
                                  H, out, ctx->paged_part.p, ctx->paged_tickets.p);
  });
}

int nnhip_kv_read_paged_q8(nnhip_ctx *ctx, const int8_t *codes, const float *scales,
                           int block_size, int num_blocks, const int32_t *slots, int T, int Hkv,
                           int D, float *k, float *v) {
  return guard([&] {
    const char *what = "nnhip_kv_read_paged_q8";
    const nnhip::PagedPool p = pool_of(block_size, num_blocks, Hkv, D, codes, scales, what);
    REQ(aligned(k, 16) && aligned(v, 16),
        "nnhip_kv_read_paged_q8: k and v must be aligned to 16 bytes");
    REQ(ctx && T >= 0 && ((slots && k && v) || T == 0),
        "nnhip_kv_read_paged_q8: NULL argument or negative T");
    if (T == 0) return;
    set_device(ctx);
    nnhip::launch_kv_read_paged(ctx->c.stream, codes, scales, p, slots, T, k, v);
  });
}

}  // extern "C"
