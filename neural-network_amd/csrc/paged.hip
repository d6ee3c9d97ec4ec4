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
constexpr int kTabThreads = 1024, kTabPer = kMaxRequests / kTabThreads;

struct TabSums { int64_t added, back, take; };

__device__ inline int64_t wave_scan(int64_t x, int lane) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
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

__global__ __launch_bounds__(kTabThreads) void block_tables_kernel(
    int B, const int32_t *__restrict__ cached, const int32_t *__restrict__ added, int lbs,
    int max_blocks, int32_t *tables, int32_t *held, int blocks, int32_t *free_list,
    int32_t *free_count, int T, int32_t *__restrict__ row_start, int32_t *__restrict__ lens,
    int32_t *__restrict__ pos, int32_t *__restrict__ slots, int32_t *__restrict__ status,
    unsigned *ticket) {
  __shared__ int s_rows[kMaxRequests + 1], s_back[kMaxRequests + 1], s_take[kMaxRequests + 1];
  __shared__ int64_t s_wave[3][kTabThreads / kWave];
  __shared__ int s_worst, s_last, s_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) {
    s_worst = INT_MAX;
    s_count = *free_count;
  }
  BlockNeed nd[kTabPer];
  int add[kTabPer];
  TabSums mine{0, 0, 0};
  int worst = INT_MAX;
#pragma unroll
  for (int i = 0; i < kTabPer; ++i) {
    const int b = tid * kTabPer + i;
    nd[i] = BlockNeed{0, 0, 0, 0};
    add[i] = 0;
    if (b < B) {
      add[i] = added[b];
      nd[i] = block_need(cached[b], add[i], held[b], lbs, max_blocks);
      if (nd[i].status) worst = min(worst, nd[i].status);
      mine.added += add[i];
      mine.back += nd[i].back;
      mine.take += nd[i].take;
    }
  }
  TabSums sc{wave_scan(mine.added, lane), wave_scan(mine.back, lane), wave_scan(mine.take, lane)};
  if (lane == 63) {
    s_wave[0][wave] = sc.added;
    s_wave[1][wave] = sc.back;
    s_wave[2][wave] = sc.take;
  }
  __syncthreads();                                // held and free_count have been read
  const int64_t count = s_count;
  if (worst != INT_MAX) atomicMin(&s_worst, worst);
  if (tid == 0) s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  TabSums all{0, 0, 0}, at{sc.added - mine.added, sc.back - mine.back, sc.take - mine.take};
  for (int w = 0; w < kTabThreads / kWave; ++w) {
    if (w == wave) { at.added += all.added; at.back += all.back; at.take += all.take; }
    all.added += s_wave[0][w];
    all.back += s_wave[1][w];
    all.take += s_wave[2][w];
  }
  __syncthreads();
  const bool last = s_last != 0;
  if (last && tid == 0) *ticket = 0;
  const int st = tables_status(s_worst == INT_MAX ? 0 : s_worst, all.added, T, all.back, all.take,
                               count, blocks);
  const int64_t gt = (int64_t)blockIdx.x * kTabThreads + tid, gn = (int64_t)gridDim.x * kTabThreads;
  if (last && tid == 0) *status = st;
  if (st) {                                       // nothing changes, and the step has no rows
    for (int64_t t = gt; t < T; t += gn) { pos[t] = -1; slots[t] = -1; }
    if (last) {
      for (int b = tid; b < B; b += kTabThreads) lens[b] = 0;
      for (int b = tid; b <= B; b += kTabThreads) row_start[b] = 0;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kTabPer; ++i) {
    const int b = tid * kTabPer + i;
    if (b < B) {
      s_rows[b] = (int)at.added;
      s_back[b] = (int)at.back;
      s_take[b] = (int)at.take;
      if (last) {
        row_start[b] = (int)at.added;
        lens[b] = cached[b] + add[i];
        held[b] = nd[i].need;
      }
    }
    at.added += add[i];
    at.back += nd[i].back;
    at.take += nd[i].take;
  }
  const int rows = (int)all.added, R = (int)all.back, K = (int)all.take;
  if (tid == 0) {
    s_rows[B] = rows;
    s_back[B] = R;
    s_take[B] = K;
    if (last) {
      row_start[B] = rows;
      *free_count = (int)count + R - K;
    }
  }
  __syncthreads();
  auto needs = [&](int b) { return (cached[b] + added[b] + (1 << lbs) - 1) >> lbs; };
  auto returned = [&](int r) {
    const int b = last_at_most(s_back, B, r);
    return tables[(int64_t)b * max_blocks + needs(b) + r - s_back[b]];
  };
  auto taken = [&](int t) { return t < R ? returned(t) : free_list[count + R - 1 - t]; };
  for (int64_t t = gt; t < K; t += gn) {
    const int b = last_at_most(s_take, B, (int)t);
    tables[(int64_t)b * max_blocks + needs(b) - (s_take[b + 1] - (int)t)] = taken((int)t);
  }
  for (int64_t r = K + gt; r < R; r += gn) free_list[count + R - 1 - r] = returned((int)r);
  for (int64_t t = gt; t < T; t += gn) {
    int p = -1, s = -1;
    if (t < rows) {
      const int b = last_at_most(s_rows, B, (int)t);
      p = cached[b] + (int)t - s_rows[b];
      const int j = p >> lbs, first = needs(b) - (s_take[b + 1] - s_take[b]);
      const int blk = j < first ? tables[(int64_t)b * max_blocks + j] : taken(s_take[b] + j - first);
      s = block_ok(blk, blocks) ? (blk << lbs) + (p & ((1 << lbs) - 1)) : -1;
    }
    pos[t] = p;
    slots[t] = s;
  }
}

// ---------------------------------------------------------------------------
// RoPE + append.
//
// The rows of one block lie within bs rows of one another; the wave of the first
// of them stores the block's k or v of one head.  Which row each token takes is
// gathered in LDS (the last row where several name a token), so rows that are
// skipped, or out of order, do not divide a block between two waves.  The
// rotation and the rounding to codes are in 64 bits (the sines, cosines and rows
// are fp32 inputs, so a product is exact and a code does not depend on how a sum
// of two was rounded): the launch is bound by its memory traffic all the same.
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

__global__ __launch_bounds__(256) void rope_append_paged_kernel(
    AppendRows a, PagedPool p, float *__restrict__ q_out, int8_t *codes, float *scales) {
  const int t = blockIdx.x, D = p.D, H = a.H, Hkv = p.Hkv;
  const int slot = append_slot(a, p, t);
  if (slot < 0) return;
  const int64_t stride = (int64_t)(H + 2 * Hkv) * D;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < H * D / 4; i += 256) {
      double x[4];
      rotate4(a, t, t * stride + (int64_t)(i / (D / 4)) * D, i % (D / 4), D, x);
      *reinterpret_cast<float4 *>(q_out + (int64_t)t * H * D + 4 * i) =
          make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
    }
    return;
  }
  const int blk = slot >> p.lbs;
  // an earlier row of the same block stores it
  bool later = false;
  for (int i = 1 + (int)(threadIdx.x & 63); i < p.bs; i += kWave)
    if (t - i >= 0) {
      const int s = append_slot(a, p, t - i);
      later |= s >= 0 && s >> p.lbs == blk;
    }
  if (__any(later)) return;
  __shared__ int s_row[4][128];                   // the row of each token, -1: none
  int *row = s_row[wave];
  for (int i = lane; i < p.bs; i += kWave) row[i] = -1;
  __syncthreads();
  for (int i = lane; i < p.bs; i += kWave)
    if (t + i < a.T) {
      const int s = append_slot(a, p, t + i);
      if (s >= 0 && s >> p.lbs == blk) atomicMax(&row[s & (p.bs - 1)], t + i);
    }
  __syncthreads();
  const int unit = (blockIdx.y - 1) * 4 + wave;
  if (unit >= 2 * Hkv) return;
  const int kv = unit / Hkv, h = unit % Hkv, D4 = D / 4;
  int off = p.bs, end = 0;                        // the block's tokens of this call
  for (int i = 0; i < p.bs; i += kWave) {
    const uint64_t m = __ballot(i + lane < p.bs && row[(i + lane) & 127] >= 0);
    if (!m) continue;
    off = min(off, i + __builtin_ctzll(m));
    end = i + 64 - __builtin_clzll(m);
  }
  const int64_t head = (int64_t)(H + kv * Hkv + h) * D;
  double amax = 0;
  bool bad = false;
  for (int i = off * D4 + lane; i < end * D4; i += kWave) {
    const int r = row[i / D4], c = i % D4;
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
#pragma unroll
  for (int o = 32; o; o >>= 1) amax = fmax(amax, __shfl_xor(amax, o, kWave));
  float *sc = scales + scale_offset(p, blk, kv, h);
  const double old = off ? (double)*sc : 0.0, want = block_scale(amax);
  const bool none = __any(bad) || !(fabs(old) < 1e300);  // not a number: the block has no scale
  const double now = none ? __builtin_nan("") : fmax(old, want);
  const double inv = !none && now > 0 ? 1.0 / now : 0.0;
  const bool grown = !none && now > old;
  const double ratio = grown ? old * inv : 1.0;
  if (lane == 0) *sc = (float)now;
  int *dst = reinterpret_cast<int *>(codes + head_offset(p, blk, kv, h));
  const int first = grown ? 0 : off;
  if (kv == 0) {
    for (int i = first * D4 + lane; i < end * D4; i += kWave) {
      const int tok = i / D4, c = i % D4, r = row[tok];
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
    for (int i = first / 4 * D + lane; i < (end + 3) / 4 * D; i += kWave) {
      const int w = i / D, d = i % D, at = d * (p.bs / 4) + w;
      int word = dst[at];
      const int moved = grown ? requant4(word, ratio) : word;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = 4 * w + k, r = row[tok], m = 255 << (8 * k);
        int code = tok < off ? moved & m : word & m;
        if (r >= 0)
          code = (none ? 0 : (int)rint((double)a.qkv[head + r * stride + d] * inv) & 255) << (8 * k);
        word = (word & ~m) | code;
      }
      dst[at] = word;
    }
  }
}

// ---------------------------------------------------------------------------
// Cached rows as fp32: a wave per (row, head).
__global__ __launch_bounds__(256) void kv_read_paged_kernel(
    const int8_t *__restrict__ codes, const float *__restrict__ scales, PagedPool p,
    const int32_t *__restrict__ slots, int T, float *__restrict__ k, float *__restrict__ v) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (int64_t)T * p.Hkv) return;
  const int t = unit / p.Hkv, h = unit % p.Hkv, lane = threadIdx.x & 63;
  const int slot = slots[t];
  if (!slot_ok(p, slot)) return;
  const int blk = slot >> p.lbs, off = slot & (p.bs - 1);
  const int8_t *kc = codes + head_offset(p, blk, 0, h) + off * p.D;
  const int8_t *vc = codes + head_offset(p, blk, 1, h) + off;
  const float ks = scales[scale_offset(p, blk, 0, h)], vs = scales[scale_offset(p, blk, 1, h)];
  for (int d = lane; d < p.D; d += kWave) {
    k[unit * p.D + d] = (float)kc[d] * ks;
    v[unit * p.D + d] = (float)vc[d << p.lbs] * vs;
  }
}

}  // namespace

void launch_block_tables(hipStream_t st, int B, const int32_t *cached, const int32_t *added,
                         int lbs, int max_blocks, int32_t *tables, int32_t *held, int blocks,
                         int32_t *free_list, int32_t *free_count, int T, int32_t *row_start,
                         int32_t *lens, int32_t *pos, int32_t *slots, int32_t *status,
                         unsigned *ticket) {
  const int grid = (int)std::min<int64_t>(64, ((int64_t)T + kTabThreads - 1) / kTabThreads);
  hipLaunchKernelGGL(block_tables_kernel, dim3(std::max(grid, 1)), dim3(kTabThreads), 0, st, B,
                     cached, added, lbs, max_blocks, tables, held, blocks, free_list, free_count, T,
                     row_start, lens, pos, slots, status, ticket);
  NNHIP_CHECK(hipGetLastError());
}

void launch_rope_append_paged(hipStream_t st, const float *qkv, int T, int H, const PagedPool &p,
                              const int32_t *pos, const int32_t *slots, const float *cosb,
                              const float *sinb, int n_pos, float *q_out, int8_t *codes,
                              float *scales) {
  const AppendRows a{qkv, T, H, pos, slots, cosb, sinb, n_pos};
  hipLaunchKernelGGL(rope_append_paged_kernel, dim3(T, 1 + (2 * p.Hkv + 3) / 4), dim3(256), 0, st,
                     a, p, q_out, codes, scales);
  NNHIP_CHECK(hipGetLastError());
}

void launch_kv_read_paged(hipStream_t st, const int8_t *codes, const float *scales,
                          const PagedPool &p, const int32_t *slots, int T, float *k, float *v) {
  const int64_t units = (int64_t)T * p.Hkv;
  hipLaunchKernelGGL(kv_read_paged_kernel, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st,
                     codes, scales, p, slots, T, k, v);
  NNHIP_CHECK(hipGetLastError());
}

}  // namespace nnhip
