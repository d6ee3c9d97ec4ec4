// The paged int8 KV cache: block tables and slot maps from request lengths,
// RoPE + append into blocks, and reading rows back (attention over them:
// paged_attention.hip).
#include "nnhip_internal.hpp"

#include <algorithm>
#include <climits>

namespace nnhip {

namespace {

constexpr int kWave = 64;

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
// rollback: @@; 64 prompts of up to 2000 tokens: @@.

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
// idle) for k or v of one head.  A decode step has a leader a row, of one token: a
// wave takes one.  A prompt has one or two, of up to bs tokens: the workgroup's
// threads share it.  The rows are read twice, for the scale and for the codes, the
// second time from L2.  The queries are rotated by workgroups behind those.
// @@
struct AppendRows {
  const float *qkv;
  int T, H;
  const int32_t *pos, *slots;
  const float *cosb, *sinb;
  int n_pos;
};

// Slot of row t, or -1 where the row is skipped.
__device__ inline int append_slot(const AppendRows &a, const PagedPool &p, int t) {
  const int x = a.pos[t], s = a.slots[t];
  return x >= 0 && x < a.n_pos && slot_ok(p, s) ? s : -1;
}

// Elements 4c .. 4c+3 of a head of row t (at `at`) after RoPE.
__device__ inline void rotate4(const AppendRows &a, int t, int64_t at, int c, int D, double x[4]) {
  const float4 v = *reinterpret_cast<const float4 *>(a.qkv + at + 4 * c);
  const int64_t r = (int64_t)a.pos[t] * (D / 2) + 2 * c;
  const float2 cs = *reinterpret_cast<const float2 *>(a.cosb + r);
  const float2 sn = *reinterpret_cast<const float2 *>(a.sinb + r);
  x[0] = (double)v.x * cs.x - (double)v.y * sn.x;
  x[1] = (double)v.x * sn.x + (double)v.y * cs.x;
  x[2] = (double)v.z * cs.y - (double)v.w * sn.y;
  x[3] = (double)v.z * sn.y + (double)v.w * cs.y;
}

__device__ inline int requant4(int word, double ratio) {
  int out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out |= ((int)rint((double)(int8_t)(word >> (8 * i)) * ratio) & 255) << (8 * i);
  return out;
}

constexpr int kLeadRows = 16, kLeadFew = 4, kLeadMany = 768, kQuads = 1024;

// LDS between the lanes of a wave: its accesses are in order.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// k or v (kv) of head h of the block that row `lead` of the window s_slot leads,
// stored by a wave or by the whole workgroup.  Window entry i is row w0 + i.
template <bool ALL>
__device__ void append_block(const AppendRows &a, const PagedPool &p, const int *s_slot, int w0,
                             int n, int lead, int *row, double *s_amax, int kv, int h,
                             int8_t *codes, float *scales) {
  constexpr int kThreads = ALL ? 256 : kWave;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = ALL ? threadIdx.x : lane;
  const int blk = s_slot[lead] >> p.lbs, D = p.D, D4 = D / 4, ld4 = 31 - __builtin_clz(D4);
  float *sc = scales + scale_offset(p, blk, kv, h);
  const float had = *sc;
  for (int i = tid; i < p.bs; i += kThreads) row[i] = -1;  // the row of each token
  if (ALL) __syncthreads(); else wave_sync();
  for (int i = tid; i < p.bs; i += kThreads)
    if (lead + i < n) {
      const int s = s_slot[lead + i];
      if (s >= 0 && s >> p.lbs == blk) atomicMax(&row[s & (p.bs - 1)], w0 + lead + i);
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
  const int64_t head = (int64_t)(a.H + kv * p.Hkv + h) * D;
  double amax = 0;
  bool bad = false;
#pragma unroll 4
  for (int i = (off << ld4) + tid; i < end << ld4; i += kThreads) {
    const int r = row[i >> ld4], c = i & (D4 - 1);
    if (r < 0) continue;
    double x[4];
    if (kv == 0) {
      rotate4(a, r, head + r * stride, c, D, x);
    } else {
      const float4 v = *reinterpret_cast<const float4 *>(a.qkv + head + r * stride + 4 * c);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      bad |= !(fabs(x[k]) < 1e300);
      amax = fmax(amax, fabs(x[k]));
    }
  }
  if (__any(bad)) amax = __builtin_inf();
#pragma unroll
  for (int o = 32; o; o >>= 1) amax = fmax(amax, __shfl_xor(amax, o, kWave));
  if (ALL) {
    if (lane == 0) s_amax[wave] = amax;
    __syncthreads();
    for (int w = 0; w < 4; ++w) amax = fmax(amax, s_amax[w]);
  }
  const double old = off ? (double)had : 0.0;
  const bool none = !(amax < 1e300) || !(fabs(old) < 1e300);  // not a number: the block has no scale
  const double now = none ? __builtin_nan("") : fmax(old, block_scale(amax));
  const double inv = !none && now > 0 ? 1.0 / now : 0.0;
  const bool grown = !none && now > old;
  const double ratio = grown ? old * inv : 1.0;
  if (tid == 0) *sc = (float)now;
  int *dst = reinterpret_cast<int *>(codes + head_offset(p, blk, kv, h));
  const int first = grown ? 0 : off;
  if (kv == 0) {
#pragma unroll 4
    for (int i = (first << ld4) + tid; i < end << ld4; i += kThreads) {
      const int tok = i >> ld4, c = i & (D4 - 1), r = row[tok];
      if (tok < off) {
        dst[i] = requant4(dst[i], ratio);
      } else if (r >= 0) {
        double x[4];
        rotate4(a, r, head + r * stride, c, D, x);
        int w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) w |= (none ? 0 : (int)rint(x[k] * inv) & 255) << (8 * k);
        dst[i] = w;
      }
    }
  } else {
    // a lane takes 4 tokens of a dim, 4 lanes the 16 tokens that are 16 bytes
    const int lo = first >> 4, hi = (end + 15) >> 4;
#pragma unroll 2
    for (int i = lo * 4 * D + tid; i < hi * 4 * D; i += kThreads) {
      const int w = (i >> (ld4 + 4) << 2) + (i & 3), d = (i >> 2) & (D - 1);
      const int at = d * (p.bs / 4) + w;
      const int4 rw = *reinterpret_cast<const int4 *>(row + 4 * w);
      const int rows[4] = {rw.x, rw.y, rw.z, rw.w};
      const bool kept = (rw.x | rw.y | rw.z | rw.w) < 0;  // a token that stays as it was
      if (kept && (rw.x & rw.y & rw.z & rw.w) < 0 && !(grown && 4 * w < off)) continue;
      int word = kept ? dst[at] : 0;
      if (grown && 4 * w < off) {
        const int moved = requant4(word, ratio);
        const int m = off - 4 * w >= 4 ? -1 : (1 << (8 * (off - 4 * w))) - 1;
        word = (moved & m) | (word & ~m);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (rows[k] >= 0) {
          const double x = a.qkv[head + rows[k] * stride + d];
          word = (word & ~(255 << (8 * k))) | (none ? 0 : (int)rint(x * inv) & 255) << (8 * k);
        }
      dst[at] = word;
    }
  }
}

template <int ROWS>
__global__ __launch_bounds__(256) void rope_append_paged_kernel(
    AppendRows a, PagedPool p, int leads, int q_rows, float *__restrict__ q_out, int8_t *codes,
    float *scales) {
  const int D = p.D, D4 = D / 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t stride = (int64_t)(a.H + 2 * p.Hkv) * D;
  if ((int)blockIdx.x >= leads) {
    const int64_t t0 = (int64_t)(blockIdx.x - leads) * q_rows;
    const int per = a.H * D4, n = (int)min((int64_t)q_rows, a.T - t0) * per;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) {
      const int r = i / per, c = i - r * per, t = (int)t0 + r;
      if (append_slot(a, p, t) < 0) continue;
      double x[4];
      rotate4(a, t, t * stride + (int64_t)(c / D4) * D, c & (D4 - 1), D, x);
      *reinterpret_cast<float4 *>(q_out + ((int64_t)t * per + c) * 4) =
          make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
    }
    return;
  }
  __shared__ int s_slot[2 * 128 + kLeadRows];     // the rows around, their slots
  __shared__ __align__(16) int s_row[4][128];
  __shared__ double s_amax[4];
  __shared__ unsigned s_leads;
  const int unit = blockIdx.x % (2 * p.Hkv), kv = unit / p.Hkv, h = unit % p.Hkv;
  const int w0 = (int)(blockIdx.x / (2 * p.Hkv)) * ROWS - (p.bs - 1);  // row of window entry 0
  const int n = 2 * p.bs + ROWS - 2;
  if (threadIdx.x == 0) s_leads = 0;
  for (int i = threadIdx.x; i < n; i += 256)
    s_slot[i] = w0 + i >= 0 && w0 + i < a.T ? append_slot(a, p, w0 + i) : -1;
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
      append_block<true>(a, p, s_slot, w0, n, p.bs - 1 + __builtin_ctz(m), s_row[0], s_amax, kv, h,
                         codes, scales);
      __syncthreads();                            // row and s_amax are free again
    }
    return;
  }
  for (int i = 0; m; m &= m - 1, ++i)
    if ((i & 3) == wave) {
      append_block<false>(a, p, s_slot, w0, n, p.bs - 1 + __builtin_ctz(m), s_row[wave], s_amax, kv,
                          h, codes, scales);
      wave_sync();
    }
}

// ---------------------------------------------------------------------------
// Cached rows as fp32: a wave per 16 rows and head.  Rows whose slots follow one
// another within 16 tokens of a block are read together: of k a lane takes four
// codes of a token and writes 16 bytes, of v it takes the 16 tokens of a dim in one
// load and writes each token's dim beside its neighbours'.  Bound by the writes, four
// times the codes: @@.
constexpr int kReadRows = 16;
template <int D>
__global__ __launch_bounds__(256) void kv_read_paged_kernel(
    const int8_t *__restrict__ codes, const float *__restrict__ scales, PagedPool p,
    const int32_t *__restrict__ slots, int T, float *__restrict__ k, float *__restrict__ v) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, h = unit % p.Hkv;
  const int64_t t0 = unit / p.Hkv * kReadRows;
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
    for (int i = lane; i < n * (D / 4); i += kWave) {
      const int r = i / (D / 4), c = i % (D / 4);
      const int w = *reinterpret_cast<const int *>(kc + 4 * i);
      *reinterpret_cast<float4 *>(ko + r * step + 4 * c) =
          make_float4((float)(int8_t)w * ks, (float)(int8_t)(w >> 8) * ks,
                      (float)(int8_t)(w >> 16) * ks, (float)(w >> 24) * ks);
    }
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) continue;
      const uint32_t w[4] = {vw[i].x, vw[i].y, vw[i].z, vw[i].w};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = e - (off & 15);
        if (r >= 0 && r < n) vo[r * step + d] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * vs;
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
  const int64_t units = 2 * (int64_t)p.Hkv;
  const bool few = (T + kLeadRows - 1) / kLeadRows * units < kLeadMany;
  const int rows = few ? kLeadFew : kLeadRows;
  const int q_rows = std::max(1, kQuads / (H * p.D / 4));
  const int64_t leads = ((int64_t)T + rows - 1) / rows * units;
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
  const int64_t units = ((int64_t)T + kReadRows - 1) / kReadRows * p.Hkv;
  const dim3 grid((unsigned)((units + 3) / 4));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, codes, scales, p, slots, T, k, v);
  };
  if (p.D == 32) launch(kv_read_paged_kernel<32>);
  else if (p.D == 64) launch(kv_read_paged_kernel<64>);
  else launch(kv_read_paged_kernel<128>);
  NNHIP_CHECK(hipGetLastError());
}

}  // namespace nnhip
