// The paged int8 KV cache: block tables and slot maps from request lengths,
// RoPE + append into blocks, and reading rows back (attention over them:
// paged_attention.hip).
#include "nnhip_internal.hpp"

#include <algorithm>
#include <climits>

namespace nnhip {

namespace {

constexpr int kWave = 64;
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Block tables and slot maps.
//
// need_b = ceil((cached_b + added_b) / bs).  A request that holds more returns
// table entries [need, held), one that holds fewer takes [held, need).  With
// exclusive sums over the requests, returned block r (in the order of requests
// and entries) belongs on the stack at count + R - 1 - r and taken block t
// comes from there, count + R - 1 - t: rank t < R is the returned block of the
// same rank, the others come off the old stack.  So nothing that one thread
// reads is written by another (returned entries stay in the table behind the
// request's blocks, the stack is written at and above the old count only), and
// every workgroup can form the sums itself: one launch without a wait between
// workgroups.  held and free_count alone are read by all and changed: the last
// workgroup to have read them (a ticket) writes them.
//
// Bound by latency: a scan over the requests, a search of each row's request among
// their sums in LDS, and the table's entry.  Decode step of 256 requests, with its
// rollback: 5.0 us a call; 64 prompts of up to 2000 tokens: 8.4, and back: 5.4.

// Sums over a wave, up to and including each lane.
__device__ inline int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// The last b of [0, n) with off[b] <= x; off ascending, off[0] = 0 <= x.
__device__ inline int last_at_most(const int *off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Rows, returned and taken blocks of some requests.  A call that asks for more than
// 2^31 of them is refused, so the sums are kept as 16 bits and the rest: neither
// part of 4096 requests' (at most 2^30 tokens each) passes 2^28.
struct TabSum {
  int lo, hi;
  __device__ int64_t all() const { return ((int64_t)hi << 16) + lo; }
  __device__ void add(int x) { lo += x & 0xffff; hi += x >> 16; }
  __device__ void add(const TabSum &x) { lo += x.lo; hi += x.hi; }
};

template <int THREADS>
__global__ __launch_bounds__(THREADS) void block_tables_kernel(
    int B, const int32_t *__restrict__ cached, const int32_t *__restrict__ added, int lbs,
    int max_blocks, int32_t *tables, int32_t *held, int blocks, int32_t *free_list,
    int32_t *free_count, int T, int32_t *__restrict__ row_start, int32_t *__restrict__ lens,
    int32_t *__restrict__ pos, int32_t *__restrict__ slots, int32_t *__restrict__ status,
    unsigned *ticket) {
  constexpr int kMost = THREADS * 4 < kMaxRequests ? THREADS * 4 : kMaxRequests, kPer = 4;
  constexpr int kWaves = THREADS / kWave;
  __shared__ int s_rows[kMost + 1], s_back[kMost + 1], s_take[kMost + 1];
  __shared__ int s_need[kMost], s_pos[kMost];     // blocks; position of row 0
  __shared__ TabSum s_wave[3][kWaves];
  __shared__ int s_worst, s_last, s_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) {
    s_worst = INT_MAX;
    s_count = *free_count;
  }
  // consecutive requests, as few a thread as there are
  const int per = (B + THREADS - 1) / THREADS, b0 = tid * per;
  BlockNeed nd[kPer];
  int add[kPer], len[kPer];
  TabSum mine[3] = {};
  int worst = INT_MAX;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = b0 + i;
    nd[i] = BlockNeed{0, 0, 0, 0};
    add[i] = len[i] = 0;
    if (i < per && b < B) {
      const int c = cached[b];
      add[i] = added[b];
      nd[i] = block_need(c, add[i], held[b], lbs, max_blocks);
      if (nd[i].status) worst = min(worst, nd[i].status);
      else len[i] = c + add[i];
      mine[0].add(add[i]);
      mine[1].add(nd[i].back);
      mine[2].add(nd[i].take);
    }
  }
  TabSum at[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    at[k] = TabSum{wave_scan(mine[k].lo), wave_scan(mine[k].hi)};
    if (lane == 63) s_wave[k][wave] = at[k];
  }
  __syncthreads();                                // held and free_count have been read
  const int64_t count = s_count;
  if (worst != INT_MAX) atomicMin(&s_worst, worst);
  const unsigned before = tid == 0 ? atomicAdd(ticket, 1u) : 0;  // looked at when all is done
  TabSum all[3] = {};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    at[k].lo -= mine[k].lo;
    at[k].hi -= mine[k].hi;
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) at[k].add(all[k]);
      all[k].add(s_wave[k][w]);
    }
  }
  __syncthreads();
  const int st = tables_status(s_worst == INT_MAX ? 0 : s_worst, all[0].all(), T, all[1].all(),
                               all[2].all(), count, blocks);
  const int64_t gt = (int64_t)blockIdx.x * THREADS + tid, gn = (int64_t)gridDim.x * THREADS;
  const int total = st ? 0 : (int)all[0].all(), R = (int)all[1].all(), K = (int)all[2].all();
  if (blockIdx.x == 0 && tid == 0) {
    *status = st;
    row_start[B] = total;
  }
  int rows = (int)at[0].all(), back = (int)at[1].all(), take = (int)at[2].all();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = b0 + i;
    if (i < per && b < B) {
      s_rows[b] = rows;
      s_back[b] = back;
      s_take[b] = take;
      s_need[b] = nd[i].need;
      s_pos[b] = len[i] - add[i] - rows;
      if (blockIdx.x == 0) {
        row_start[b] = st ? 0 : rows;
        lens[b] = st ? 0 : len[i];
      }
    }
    rows += add[i];
    back += nd[i].back;
    take += nd[i].take;
  }
  if (tid == 0) {
    s_rows[B] = total;
    s_back[B] = R;
    s_take[B] = K;
  }
  __syncthreads();
  auto returned = [&](int r) {
    const int b = last_at_most(s_back, B, r);
    return tables[(int64_t)b * max_blocks + s_need[b] + r - s_back[b]];
  };
  auto taken = [&](int t) { return t < R ? returned(t) : free_list[count + R - 1 - t]; };
  for (int64_t t = gt; t < T; t += gn) {
    int p = -1, s = -1;
    if (t < total) {
      const int b = last_at_most(s_rows, B, (int)t);
      p = s_pos[b] + (int)t;
      const int j = p >> lbs, first = s_need[b] - (s_take[b + 1] - s_take[b]);
      const int blk = j < first ? tables[(int64_t)b * max_blocks + j] : taken(s_take[b] + j - first);
      s = block_ok(blk, blocks) ? (blk << lbs) + (p & ((1 << lbs) - 1)) : -1;
    }
    pos[t] = p;
    slots[t] = s;
  }
  if (!st) {
    for (int64_t t = gt; t < K; t += gn) {
      const int b = last_at_most(s_take, B, (int)t);
      tables[(int64_t)b * max_blocks + s_need[b] - (s_take[b + 1] - (int)t)] = taken((int)t);
    }
    for (int64_t r = K + gt; r < R; r += gn) free_list[count + R - 1 - r] = returned((int)r);
  }
  if (tid == 0) s_last = before == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  for (int b = tid; b < B && !st; b += THREADS) held[b] = s_need[b];
  if (tid == 0) {
    *ticket = 0;
    if (!st) *free_count = (int)count + R - K;
  }
}

// ---------------------------------------------------------------------------
// RoPE + append.
//
// The rows of one block lie within bs rows of one another; the first of them leads:
// where it stands, the block is stored whole, its rows gathered from the bs rows that
// follow.  Which row each token takes is noted in LDS (the last row where several
// name a token), so rows that are skipped, or out of order, do not divide a block
// between two workgroups.  The rotation and the rounding to codes are in 64 bits
// (the sines, cosines and rows are fp32 inputs, so a product is exact and a code
// does not depend on how a sum of two was rounded): the launch is bound by its
// memory traffic all the same.
//
// A workgroup takes the leaders among some 16 rows (4, where that leaves the card
// idle) for one head.  A prompt has one or two, of up to bs tokens: the workgroup's
// threads share it.  A decode step has a leader a row, of one token: a wave takes
// one after another.  The first quads that a thread has looked at for the scale stay
// in registers until their codes are stored (more of them cost workgroups a unit:
// two 22 us, four 27, one 20, where the rest is read from L2 again).  The queries are
// rotated by workgroups behind those, with stores that do not stay in the caches: on
// the other dies, which read most of them, they would not be found (with the rows
// read back 28 us for 32, with attention behind it the same to 1%).
//
// 9 prompts of up to 1000 tokens (7835 rows, 16 heads over 4 of 64 dims): 20 us,
// 4.3 TB/s; bound by memory at that size.  A step of 27 requests: 5 us, latency.

struct AppendRows {
  const float *qkv;
  int T, H;
  const int32_t *pos, *slots;
  const float *cosb, *sinb;
  int n_pos;
};

// Slot of row t, or -1 where the row is skipped.
__device__ inline int append_slot(const AppendRows &a, const PagedPool &p, int x, int s) {
  return x >= 0 && x < a.n_pos && slot_ok(p, s) ? s : -1;
}

// Four elements of a head and the cosines and sines of their two pairs.
struct Quad {
  float4 x;
  float2 c, s;
};
__device__ inline Quad quad(const AppendRows &a, int pos, int64_t at, int c, int D) {
  const int64_t r = (int64_t)pos * (D / 2) + 2 * c;
  return Quad{*reinterpret_cast<const float4 *>(a.qkv + at + 4 * c),
              *reinterpret_cast<const float2 *>(a.cosb + r),
              *reinterpret_cast<const float2 *>(a.sinb + r)};
}
__device__ inline void rotate(const Quad &q, double x[4]) {
  x[0] = (double)q.x.x * q.c.x - (double)q.x.y * q.s.x;
  x[1] = (double)q.x.x * q.s.x + (double)q.x.y * q.c.x;
  x[2] = (double)q.x.z * q.c.y - (double)q.x.w * q.s.y;
  x[3] = (double)q.x.z * q.s.y + (double)q.x.w * q.c.y;
}

__device__ inline int requant4(int word, double ratio) {
  int out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out |= ((int)rint((double)(int8_t)(word >> (8 * i)) * ratio) & 255) << (8 * i);
  return out;
}

constexpr int kLeadRows = 16, kLeadFew = 4, kLeadMany = 480, kQuads = 1024;

// LDS between the lanes of a wave: its accesses are in order.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A block's scale before and after this call.
struct Rescale {
  double inv, ratio;                              // powers of two; inv 0: the block is zeros
  bool none, grown;                               // none: not a number
  float now;
  __device__ Rescale(double amax, double old) {
    none = !(amax < 1e300) || !(fabs(old) < 1e300);
    const double s = none ? __builtin_nan("") : fmax(old, block_scale(amax));
    inv = !none && s > 0 ? 1.0 / s : 0.0;
    grown = !none && s > old;
    ratio = grown ? old * inv : 1.0;
    now = (float)s;
  }
};

// Four codes: value * inv, which is exact and at most 127, rounded to nearest by the
// sum with 1.5 times the power of two whose last bit is 1, and its low byte.
__device__ inline int pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400),
                               __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
}
__device__ inline uint32_t code(double x, double inv) {
  return (uint32_t)__double_as_longlong(fma(x, inv, 0x1.8p52));
}

// Larger of m and |x|, as bits without the sign: in the order of the values, and
// infinities and NaN from 0xff000000.
__device__ inline uint32_t max_bits(uint32_t m, float x) { return max(m, __float_as_uint(x) << 1); }

// Head h of the block that row w0 + lead leads, k and v, stored by a wave or by the
// whole workgroup.  Window entry i is row w0 + i: s_slot its slot, s_pos its position.
template <bool ALL>
__device__ void append_block(const AppendRows &a, const PagedPool &p, const int *s_slot,
                             const int *s_pos, int w0, int n, int lead, int *row,
                             double (*s_amax)[2], int h, int8_t *codes, float *scales) {
  constexpr int kThreads = ALL ? 256 : kWave, kKeep = 1;  // quads that stay in registers
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = ALL ? threadIdx.x : lane;
  const int blk = s_slot[lead] >> p.lbs, D = p.D, D4 = D / 4, ld4 = 31 - __builtin_clz(D4);
  float *sc[2] = {scales + scale_offset(p, blk, 0, h), scales + scale_offset(p, blk, 1, h)};
  const float had[2] = {*sc[0], *sc[1]};
  for (int i = tid; i < p.bs; i += kThreads) row[i] = -1;  // the window entry of each token
  if (ALL) __syncthreads(); else wave_sync();
  for (int i = tid; i < p.bs; i += kThreads)
    if (lead + i < n) {
      const int s = s_slot[lead + i];
      if (s >= 0 && s >> p.lbs == blk) atomicMax(&row[s & (p.bs - 1)], lead + i);
    }
  if (ALL) __syncthreads(); else wave_sync();
  int off = p.bs, end = 0;                        // the block's tokens of this call
  for (int i = 0; i < p.bs; i += kWave) {
    const uint64_t m = __ballot(i + lane < p.bs && row[(i + lane) & 127] >= 0);
    if (!m) continue;
    off = min(off, i + __builtin_ctzll(m));
    end = i + 64 - __builtin_clzll(m);
  }
  const int64_t stride = (int64_t)(a.H + 2 * p.Hkv) * D;
  const int64_t k_at = w0 * stride + (int64_t)(a.H + h) * D, v_at = k_at + (int64_t)p.Hkv * D;
  int *kd = reinterpret_cast<int *>(codes + head_offset(p, blk, 0, h));
  int *vd = reinterpret_cast<int *>(codes + head_offset(p, blk, 1, h));
  // k: a quad is four dims of a token.  v: four tokens of a dim, as the codes lie; 4
  // lanes have the 16 tokens that are 16 bytes, where there are as many.  What is no
  // row reads the leader.
  const int sub = end - (off & ~3) > 8 ? 2 : 0, w0_v = off >> 2 >> sub << sub;
  const int k_end = end << ld4, v_end = ((end + 3 >> 2) + (1 << sub) - 1 >> sub << sub) * D;
  const int k0 = (off << ld4) + tid, v0 = w0_v * D + tid;
  auto k_quad = [&](int i) {
    const int r = i < k_end ? row[i >> ld4] : -1, e = r < 0 ? lead : r;
    return quad(a, s_pos[e], k_at + e * stride, i & (D4 - 1), D);
  };
  auto v_word = [&](int i) { return (i >> (ld4 + 2 + sub) << sub) + (i & ((1 << sub) - 1)); };
  auto v_dim = [&](int i) { return (i >> sub) & (D - 1); };
  auto v_rows = [&](int i) {
    return i < v_end ? *reinterpret_cast<const int4 *>(row + 4 * v_word(i)) : make_int4(-1, -1, -1, -1);
  };
  auto v_quad = [&](int i) {
    const int4 r = v_rows(i);
    const float *x = a.qkv + v_at + v_dim(i);
    return make_float4(x[(r.x < 0 ? lead : r.x) * stride], x[(r.y < 0 ? lead : r.y) * stride],
                       x[(r.z < 0 ? lead : r.z) * stride], x[(r.w < 0 ? lead : r.w) * stride]);
  };
  auto v_old = [&](int i) {                       // the word as it is, where part of it stays
    const int4 r = v_rows(i);
    return i < v_end && (r.x | r.y | r.z | r.w) < 0 ? vd[v_dim(i) * (p.bs / 4) + v_word(i)]
                                                    : 0;
  };
  double k_max = 0;
  uint32_t k_bits = 0, v_bits = 0;
  auto k_look = [&](const Quad &q, double x[4], int i) {
    rotate(q, x);
    if (i >= k_end || row[i >> ld4] < 0) return;
    k_max = fmax(k_max, fmax(fmax(fabs(x[0]), fabs(x[1])), fmax(fabs(x[2]), fabs(x[3]))));
    k_bits = max_bits(max_bits(max_bits(max_bits(k_bits, q.x.x), q.x.y), q.x.z), q.x.w);
    k_bits = max_bits(max_bits(max_bits(max_bits(k_bits, q.c.x), q.c.y), q.s.x), q.s.y);
  };
  auto v_look = [&](const float4 &q, int i) {
    const int4 r = v_rows(i);
    if (r.x >= 0) v_bits = max_bits(v_bits, q.x);
    if (r.y >= 0) v_bits = max_bits(v_bits, q.y);
    if (r.z >= 0) v_bits = max_bits(v_bits, q.z);
    if (r.w >= 0) v_bits = max_bits(v_bits, q.w);
  };
  double kx[kKeep][4];
  float4 vq[kKeep];
  int vw[kKeep];
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    const Quad q = k_quad(k0 + j * kThreads);
    vq[j] = v_quad(v0 + j * kThreads);
    vw[j] = v_old(v0 + j * kThreads);
    k_look(q, kx[j], k0 + j * kThreads);
  }
#pragma unroll
  for (int j = 0; j < kKeep; ++j) v_look(vq[j], v0 + j * kThreads);
  double x[4];
#pragma unroll 2
  for (int i = k0 + kKeep * kThreads; i < k_end; i += kThreads) k_look(k_quad(i), x, i);
#pragma unroll 2
  for (int i = v0 + kKeep * kThreads; i < v_end; i += kThreads) v_look(v_quad(i), i);
  if (k_bits >= 0xff000000u) k_max = __builtin_inf();
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    k_max = fmax(k_max, __shfl_xor(k_max, o, kWave));
    v_bits = max(v_bits, (uint32_t)__shfl_xor((int)v_bits, o, kWave));
  }
  double amax[2] = {k_max, v_bits >= 0xff000000u ? __builtin_inf() : __uint_as_float(v_bits >> 1)};
  if (ALL) {
    if (lane == 0) { s_amax[wave][0] = amax[0]; s_amax[wave][1] = amax[1]; }
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
      amax[0] = fmax(amax[0], s_amax[w][0]);
      amax[1] = fmax(amax[1], s_amax[w][1]);
    }
  }
  // a block that begins anew (its token 0 is in this call) has no scale yet
  const Rescale ks(amax[0], off ? (double)had[0] : 0.0), vs(amax[1], off ? (double)had[1] : 0.0);
  if (tid == 0) {
    *sc[0] = ks.now;
    *sc[1] = vs.now;
  }
  auto k_store = [&](const double x[4], int i) {
    if (i >= k_end || row[i >> ld4] < 0) return;
    kd[i] = ks.none ? 0 : pack4(code(x[0], ks.inv), code(x[1], ks.inv), code(x[2], ks.inv),
                                code(x[3], ks.inv));
  };
  auto v_store = [&](const float4 &q, int word, int i) {
    if (i >= v_end) return;
    const int4 r = v_rows(i);
    const int w = v_word(i);
    if (vs.grown && 4 * w < off) {
      const int moved = requant4(word, vs.ratio);
      const int m = off - 4 * w >= 4 ? -1 : (1 << (8 * (off - 4 * w))) - 1;
      word = (moved & m) | (word & ~m);
    } else if ((r.x & r.y & r.z & r.w) < 0) {
      return;
    }
    const int now = vs.none ? 0 : pack4(code(q.x, vs.inv), code(q.y, vs.inv), code(q.z, vs.inv),
                                        code(q.w, vs.inv));
    const int m = (r.x < 0 ? 0 : 255) | (r.y < 0 ? 0 : 255 << 8) | (r.z < 0 ? 0 : 255 << 16) |
                  (r.w < 0 ? 0 : 255 << 24);
    vd[v_dim(i) * (p.bs / 4) + w] = (now & m) | (word & ~m);
  };
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    k_store(kx[j], k0 + j * kThreads);
    v_store(vq[j], vw[j], v0 + j * kThreads);
  }
#pragma unroll 2
  for (int i = k0 + kKeep * kThreads; i < k_end; i += kThreads) {
    rotate(k_quad(i), x);
    k_store(x, i);
  }
#pragma unroll 2
  for (int i = v0 + kKeep * kThreads; i < v_end; i += kThreads) v_store(v_quad(i), v_old(i), i);
  // what the block held before
  if (ks.grown)
    for (int i = tid; i < off << ld4; i += kThreads) kd[i] = requant4(kd[i], ks.ratio);
  if (vs.grown)
    for (int i = tid; i < w0_v * D; i += kThreads) {
      int &word = vd[v_dim(i) * (p.bs / 4) + v_word(i)];
      word = requant4(word, vs.ratio);
    }
}

template <int ROWS>
__global__ __launch_bounds__(256, 6) void rope_append_paged_kernel(
    AppendRows a, PagedPool p, int leads, int q_rows, float *__restrict__ q_out, int8_t *codes,
    float *scales) {
  const int D = p.D, D4 = D / 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t stride = (int64_t)(a.H + 2 * p.Hkv) * D;
  if ((int)blockIdx.x >= leads) {
    const int64_t t0 = (int64_t)(blockIdx.x - leads) * q_rows;
    const int per = a.H * D4, n = (int)min((int64_t)q_rows, a.T - t0) * per;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) {
      const int r = i / per, c = i - r * per, t = (int)t0 + r, pos = a.pos[t];
      if (append_slot(a, p, pos, a.slots[t]) < 0) continue;
      double x[4];
      rotate(quad(a, pos, t * stride + (int64_t)(c / D4) * D, c & (D4 - 1), D), x);
      const f32x4 out = {(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
      __builtin_nontemporal_store(out, reinterpret_cast<f32x4 *>(q_out + ((int64_t)t * per + c) * 4));
    }
    return;
  }
  __shared__ int s_slot[2 * 128 + kLeadRows], s_pos[2 * 128 + kLeadRows];  // the rows around
  __shared__ __align__(16) int s_row[4][128];
  __shared__ double s_amax[4][2];
  __shared__ unsigned s_leads;
  const int h = blockIdx.x % p.Hkv;
  const int w0 = (int)(blockIdx.x / p.Hkv) * ROWS - (p.bs - 1);  // row of window entry 0
  const int n = 2 * p.bs + ROWS - 2;
  if (threadIdx.x == 0) s_leads = 0;
  for (int i = threadIdx.x; i < n; i += 256) {
    int s = -1, pos = 0;
    if (w0 + i >= 0 && w0 + i < a.T) {
      pos = a.pos[w0 + i];
      s = append_slot(a, p, pos, a.slots[w0 + i]);
    }
    s_slot[i] = s;
    s_pos[i] = pos;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROWS / 4; ++k) {
    const int r = 4 * k + wave, s = s_slot[p.bs - 1 + r];
    bool lead = s >= 0;
    for (int i = lane; i < p.bs - 1; i += kWave) {
      const int e = s_slot[r + i];
      lead &= e < 0 || e >> p.lbs != s >> p.lbs;
    }
    if (__all(lead) && lane == 0) atomicOr(&s_leads, 1u << r);
  }
  __syncthreads();
  unsigned m = s_leads;
  if (__builtin_popcount(m) <= 2) {
    for (; m; m &= m - 1) {
      append_block<true>(a, p, s_slot, s_pos, w0, n, p.bs - 1 + __builtin_ctz(m), s_row[0], s_amax,
                         h, codes, scales);
      __syncthreads();                            // row and s_amax are free again
    }
    return;
  }
  for (int i = 0; m; m &= m - 1, ++i)
    if ((i & 3) == wave) {
      append_block<false>(a, p, s_slot, s_pos, w0, n, p.bs - 1 + __builtin_ctz(m), s_row[wave],
                          s_amax, h, codes, scales);
      wave_sync();
    }
}

// ---------------------------------------------------------------------------
// Cached rows as fp32: a wave per 16 rows and head.  Rows whose slots follow one
// another within 16 tokens of a block are read together: of k a lane takes four
// codes of a token and writes 16 bytes, of v it takes the 16 tokens of a dim in one
// load and writes each token's dim beside its neighbours'.  A workgroup's waves take
// neighbouring rows of one head, whose tokens of a dim share lines: 24 requests of up
// to 1000 tokens, 8 heads of 128 dims in blocks of 64, 34 us, 6.0 TB/s, bound by the
// writes, four times the codes (49 us with the waves on neighbouring heads, and 61
// with stores that stay in the caches besides).
constexpr int kReadRows = 16;

template <int D>
__global__ __launch_bounds__(256) void kv_read_paged_kernel(
    const int8_t *__restrict__ codes, const float *__restrict__ scales, PagedPool p,
    const int32_t *__restrict__ slots, int T, float *__restrict__ k, float *__restrict__ v) {
  // neighbouring rows in a workgroup: their 16 bytes of a dim of v lie side by side
  const int lane = threadIdx.x & 63, h = blockIdx.x % p.Hkv;
  const int64_t t0 = ((int64_t)(blockIdx.x / p.Hkv) * 4 + (threadIdx.x >> 6)) * kReadRows;
  if (t0 >= T) return;
  const int mine = lane < kReadRows && t0 + lane < T ? slots[t0 + lane] : -1;
  const int before = __shfl_up(mine, 1, kWave);
  const uint64_t ok = __ballot(slot_ok(p, mine));
  const uint64_t on = __ballot(lane > 0 && slot_ok(p, mine) && before >= 0 && mine == before + 1 &&
                               (mine & 15) != 0);
  for (int s = 0; s < kReadRows; ++s) {
    if (!(ok >> s & 1)) continue;
    const int n = 1 + __builtin_ctzll(~(on >> (s + 1)));
    const int slot = __builtin_amdgcn_readlane(mine, s);
    const int blk = slot >> p.lbs, off = slot & (p.bs - 1), sub = off & ~15;
    const float ks = scales[scale_offset(p, blk, 0, h)], vs = scales[scale_offset(p, blk, 1, h)];
    const int8_t *kc = codes + head_offset(p, blk, 0, h) + (int64_t)off * D;
    const int8_t *vc = codes + head_offset(p, blk, 1, h) + sub;
    float *ko = k + ((t0 + s) * p.Hkv + h) * D, *vo = v + ((t0 + s) * p.Hkv + h) * D;
    const int64_t step = (int64_t)p.Hkv * D;
    uint4 vw[(D + 63) / 64];
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i)
      if (lane + 64 * i < D)
        vw[i] = *reinterpret_cast<const uint4 *>(vc + ((lane + 64 * i) << p.lbs));
#pragma unroll 4
    for (int i = lane; i < n * (D / 4); i += kWave) {
      const int r = i / (D / 4), c = i % (D / 4);
      const int w = *reinterpret_cast<const int *>(kc + 4 * i);
      const f32x4 x = {(float)(int8_t)w * ks, (float)(int8_t)(w >> 8) * ks,
                       (float)(int8_t)(w >> 16) * ks, (float)(w >> 24) * ks};
      __builtin_nontemporal_store(x, reinterpret_cast<f32x4 *>(ko + r * step + 4 * c));
    }
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) continue;
      const uint32_t w[4] = {vw[i].x, vw[i].y, vw[i].z, vw[i].w};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = e - (off & 15);
        const float x = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * vs;
        if (r >= 0 && r < n) __builtin_nontemporal_store(x, vo + r * step + d);
      }
    }
    s += n - 1;
  }
}

}  // namespace

void launch_block_tables(hipStream_t st, int B, const int32_t *cached, const int32_t *added,
                         int lbs, int max_blocks, int32_t *tables, int32_t *held, int blocks,
                         int32_t *free_list, int32_t *free_count, int T, int32_t *row_start,
                         int32_t *lens, int32_t *pos, int32_t *slots, int32_t *status,
                         unsigned *ticket) {
  const bool few = B <= 1024;
  const int threads = few ? 256 : 1024;
  // rows, and blocks that move, of which the host only knows that requests have some
  const int64_t work = std::max<int64_t>(T, (int64_t)B * 64);
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(256, (work + threads - 1) / threads));
  if (few)
    hipLaunchKernelGGL(block_tables_kernel<256>, dim3(grid), dim3(256), 0, st, B, cached, added, lbs,
                       max_blocks, tables, held, blocks, free_list, free_count, T, row_start, lens,
                       pos, slots, status, ticket);
  else
    hipLaunchKernelGGL(block_tables_kernel<1024>, dim3(grid), dim3(1024), 0, st, B, cached, added,
                       lbs, max_blocks, tables, held, blocks, free_list, free_count, T, row_start,
                       lens, pos, slots, status, ticket);
  NNHIP_CHECK(hipGetLastError());
}

void launch_rope_append_paged(hipStream_t st, const float *qkv, int T, int H, const PagedPool &p,
                              const int32_t *pos, const int32_t *slots, const float *cosb,
                              const float *sinb, int n_pos, float *q_out, int8_t *codes,
                              float *scales) {
  const AppendRows a{qkv, T, H, pos, slots, cosb, sinb, n_pos};
  // Few rows a workgroup where there are few workgroups: 439 requests' tokens for
  // 16 heads 11 us with 4 rows, 15.5 with 16; 2000 rows of a prompt for 4 heads 12
  // and 7.
  const bool few = (T + kLeadRows - 1) / kLeadRows * (int64_t)p.Hkv < kLeadMany;
  const int rows = few ? kLeadFew : kLeadRows;
  const int q_rows = std::max(1, kQuads / (H * p.D / 4));
  const int64_t leads = ((int64_t)T + rows - 1) / rows * p.Hkv;
  const dim3 grid((unsigned)(leads + (T + q_rows - 1) / q_rows));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a, p, (int)leads, q_rows, q_out, codes,
                       scales);
  };
  if (few) launch(rope_append_paged_kernel<kLeadFew>);
  else launch(rope_append_paged_kernel<kLeadRows>);
  NNHIP_CHECK(hipGetLastError());
}

void launch_kv_read_paged(hipStream_t st, const int8_t *codes, const float *scales,
                          const PagedPool &p, const int32_t *slots, int T, float *k, float *v) {
  const dim3 grid((unsigned)(((int64_t)T + 4 * kReadRows - 1) / (4 * kReadRows) * p.Hkv));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, codes, scales, p, slots, T, k, v);
  };
  if (p.D == 32) launch(kv_read_paged_kernel<32>);
  else if (p.D == 64) launch(kv_read_paged_kernel<64>);
  else launch(kv_read_paged_kernel<128>);
  NNHIP_CHECK(hipGetLastError());
}

}  // namespace nnhip
