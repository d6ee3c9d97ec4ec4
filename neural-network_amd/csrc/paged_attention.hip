// Causal attention of ragged rows over the paged int8 KV cache (paged.hpp).
//
// Every product runs on the fp16 matrix cores with fp32 results.  Codes are
// whole numbers of at most 8 bits, exact in fp16.  The other factor is fp32 and
// enters as two halves x = hi + lo of 11 bits each: hi the nearest (or, for the
// weights, the next smaller) half, lo the rest, so a product of two matrix
// instructions is off by 2^-22 (2^-20) of x where one half alone would be off by
// 2^-11.  An element far below the largest is carried to half a step of the
// smallest half, so q is scaled by a power of two for each row (its largest
// element to [2^13, 2^14)) and the weights by one for each row and tile of keys.
//
// Softmax over tiles, in base 2: with x_j = q . k_j log2(e) / sqrt(D) the kernels
// keep, for each row, m >= x_j (a whole number), l = sum 2^(x_j - m), and the sums
// O_d = 2^(m + 15 - E) sum 2^(x_j - m) vs_j v_jd, where vs is the block's scale and
// E >= x_j + log2(vs_j) the largest contribution's exponent: a weight times its
// block's scale is at most 2^15, and over 2^14 for the largest, however the
// scales differ.  m and E are whole numbers, so that changing them rounds
// nothing.  out = O 2^(E - m - 15) / l.
#include "nnhip_internal.hpp"

#include <algorithm>
#include <cfloat>

namespace nnhip {

namespace {

constexpr int kWave = 64;
constexpr int kCols = 16;        // (row, head) columns of a tile of rows
constexpr int kKeys = 64;        // keys of a tile
constexpr int kNone = -(1 << 20);  // E before the first contribution

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

__device__ inline half2_t as_half2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ inline uint32_t as_u32(half2_t x) { return __builtin_bit_cast(uint32_t, x); }
__device__ inline half8_t as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 x = {a, b, c, d};
  return __builtin_bit_cast(half8_t, x);
}

// 8 codes as halves: 0x6400 | (code + 128) is the half 1024 + 128 + code.
__device__ inline half8_t codes8(uint32_t lo, uint32_t hi) {
  const half2_t off = {(_Float16)1152.f, (_Float16)1152.f};
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  const uint32_t x = 0x64646464u;
  return as_half8(as_u32(as_half2(__builtin_amdgcn_perm(x, lo, 0x04010400u)) - off),
                  as_u32(as_half2(__builtin_amdgcn_perm(x, lo, 0x04030402u)) - off),
                  as_u32(as_half2(__builtin_amdgcn_perm(x, hi, 0x04010400u)) - off),
                  as_u32(as_half2(__builtin_amdgcn_perm(x, hi, 0x04030402u)) - off));
}

// max and sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ inline float max_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float sum_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Where the codes and scales of 16 tokens lie: their block, and the first one's
// place in it.  Tokens behind the request's last are read from block 0 (and
// masked), tokens of a block outside the pool too, with `bad`.
struct Sub { int blk, off; bool bad; };
__device__ inline Sub sub_of(const int32_t *table, int64_t tok, int64_t len, const PagedPool &p) {
  Sub s{0, (int)tok & (p.bs - 1), false};
  if (tok < len) {
    const int blk = table[tok >> p.lbs];
    s.bad = !block_ok(blk, p.blocks);
    s.blk = s.bad ? 0 : blk;
  }
  return s;
}

// A scale as it is used: NaN unless it is a number >= 0; 0 below 2^-126, where a
// logarithm and the products lose it.
__device__ inline float scale_ok(float s, bool bad) {
  return bad || !(s >= 0.f && s <= FLT_MAX) ? __builtin_nanf("") : s < FLT_MIN ? 0.f : s;
}

// 2^(m - M) for a share of a sum whose largest exponent is M; both may be
// -infinity, of a share that saw nothing.
__device__ inline float share(float m, float M) {
  return m == M ? 1.f : __builtin_amdgcn_exp2f(m - M);
}

struct AttnArgs {
  const float *q;
  int T;
  const int8_t *codes;
  const float *scales;
  PagedPool p;
  const int32_t *tables;
  int max_blocks;
  const int32_t *row_start, *lens;
  int B, H, G;                   // G: heads of q for one of k and v
  float *out;
};

// 16 columns of a request: column c is row first + c / G, head hk * G + c % G.
struct Columns {
  int first, n, base;            // the request's rows, the tile's first column
  int64_t len;
};

// The q of a lane's column, and what its scores are multiplied by.
template <int D>
struct Query {
  half8_t hi[D / 32], lo[D / 32];
  float mul;
  int64_t see;                   // tokens that the column's row sees; 0: no row
};

template <int D>
__device__ inline Query<D> load_query(const AttnArgs &a, const Columns &c, int hk, int lane) {
  Query<D> r;
  const int col = c.base + (lane & 15), g = lane >> 4;
  const bool live = col < c.n * a.G;
  const int row = live ? col / a.G : 0, h = hk * a.G + (live ? col % a.G : 0);
  const float *src = a.q + ((int64_t)(c.first + row) * a.H + h) * D + g * (D == 32 ? 8 : 16);
  float x[D / 4];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const float4 v = *reinterpret_cast<const float4 *>(src + 64 * (i / 4) + 4 * (i % 4));
    x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < D / 4; ++i) {
    if (!live) x[i] = 0.f;
    top = fmaxf(top, fabsf(x[i]));
  }
  top = max_groups(top);
  const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;   // 2^e <= top < 2^(e + 1)
  const int up = min(13 - e, 120);
#pragma unroll
  for (int k = 0; k < D / 32; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = ldexpf(x[8 * k + j], up);
      r.hi[k][j] = (_Float16)y;
      r.lo[k][j] = (_Float16)(y - (float)r.hi[k][j]);
    }
  r.mul = ldexpf(1.4426950408889634f / sqrtf((float)D), -up);
  r.see = live ? max((int64_t)0, c.len - c.n + row + 1) : 0;
  return r;
}

// The running state of a lane's column: m and E as above (the same in the four
// lanes of a column), l the sum over the lane's own tokens.
template <int D>
struct State {
  float m = -INFINITY, l = 0.f, E = (float)kNone;
  float4_t o[D / 16] = {};
};

// Softmax of one tile: acc[t][i] is the unscaled score of token tok + 4 t + i of
// the lane's column, `ks` / `vs` the scales of these 16 tokens.  Gives the
// weights' halves, as the right operand of the products with v.
template <int D, bool MASK>
__device__ inline void softmax_tile(State<D> &s, const float4_t (&acc)[4], float ks, float vs,
                                    float mul, int visible, half8_t (&hi)[2], half8_t (&lo)[2]) {
  const float mult = ks * mul;
  float top = -FLT_MAX;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = fmaxf(top, !MASK || 4 * t + i < visible ? acc[t][i] : -FLT_MAX);
  const bool none = MASK && visible <= 0;
  const float x = none ? -INFINITY : top * mult;
  const float xm = max_groups(x), am = max_groups(x + __builtin_amdgcn_logf(vs));
  const float m = fmaxf(s.m, ceilf(xm));
  if (__any(m != s.m)) {
    s.l *= share(s.m, m);
    s.m = m;
  }
  if (__any(am > s.E)) {
    const float E = am > s.E ? ceilf(am) : s.E;
    const float f = __builtin_amdgcn_exp2f(s.E - E);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s.o[i] *= f;
    s.E = E;
  }
  const float base = m == -INFINITY ? 0.f : m;
  const float factor = fminf(ldexpf(vs, (int)(base - s.E) + 15), FLT_MAX);
  float w[16];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float e = __builtin_amdgcn_exp2f(fmaf(acc[t][i], mult, -base));
      if (MASK && 4 * t + i >= visible) e = 0.f;
      s.l += e;
      w[4 * t + i] = e * factor;
    }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = w[8 * c + 2 * j], b = w[8 * c + 2 * j + 1];
      const auto x2 = __builtin_amdgcn_cvt_pkrtz(a, b);
      h[j] = __builtin_bit_cast(uint32_t, x2);
      l[j] = __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_pkrtz(a - (float)x2[0], b - (float)x2[1]));
    }
    hi[c] = as_half8(h[0], h[1], h[2], h[3]);
    lo[c] = as_half8(l[0], l[1], l[2], l[3]);
  }
}

// ---------------------------------------------------------------------------
// Short requests: the keys split over waves and workgroups.
//
// A unit is 16 columns of one request and kv head over a range of key tiles; the
// four waves of a workgroup take its tiles in turn and join in LDS.  The range is
// chosen so that all units together fill the chip, whatever the lengths are:
// they are on the device, so every workgroup forms the sums over the requests
// itself.  Where a request's keys go to several units, each leaves its state in
// the scratch, and the last to arrive (a counter per group, left zero) joins them.
//
// S^T = K Q^T and O^T = V^T P^T: the codes are the left operand, as they lie in
// memory, and the weights that the first product leaves in a lane are what the
// second one wants there.  Lane (r = lane & 15, g = lane >> 4): the left operand of
// score product t holds, in row r, token 16 (r >> 2) + 4 t + (r & 3), dims 16 g ..
// 16 g + 15 of each 64 (the order of the dims is free: four lanes load 64
// neighbouring bytes), so that lane (column, g) gets the scores of tokens 16 g +
// 4 t + i, all of one block; the left operand of the products with v holds dim
// 16 d + r, the 16 tokens of block g.
constexpr int kSplitWaves = 4, kSplitThreads = kWave * kSplitWaves;
constexpr int kSplitUnits = 512;    // units that a launch is split into, if it has the tiles
constexpr int kSplitMin = 4;        // least tiles of a split

struct Part {                        // a request's share of the work
  int first, n, len;                 // its rows, its tokens
  int tiles, groups;                 // tiles of keys, tiles of columns
};
__device__ inline Part part_of(const AttnArgs &a, int b) {
  const RowRange r = request_rows(a.row_start, b, a.T);
  const int len = (int)request_len(a.lens[b], a.max_blocks, a.p.lbs);
  Part p{r.first, r.last - r.first, len, 0, 0};
  if (p.n) {
    p.tiles = (int)(((int64_t)len + kKeys - 1) / kKeys);
    p.groups = (int)(((int64_t)p.n * a.G + kCols - 1) / kCols);
  }
  return p;
}
// Units of one group and kv head.
__device__ inline int splits_of(const Part &p, int64_t chunk) {
  return max(1, (int)((p.tiles + chunk - 1) / chunk));
}

// Sums over the 256 threads before and including `tid`; the last entry is all.
__device__ inline int block_scan(int x, int tid, int *s_sum) {
  const int lane = tid & 63, w = tid >> 6;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  if (lane == 63) s_sum[w] = x;
  __syncthreads();
  for (int i = 0; i < w; ++i) x += s_sum[i];
  __syncthreads();
  return x;
}

template <int D>
__device__ inline void load_k(const AttnArgs &a, const Sub &s, int hk, int lane,
                              uint32_t (&r)[4][D / 16]) {
  const int m = lane & 15, g = lane >> 4;
  const int8_t *src = a.codes + head_offset(a.p, s.blk, 0, hk) +
                      (int64_t)(s.off + (m & 3)) * D + g * (D == 32 ? 8 : 16);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (D == 32) {
      const uint2 v = *reinterpret_cast<const uint2 *>(src + 4 * t * D);
      r[t][0] = v.x; r[t][1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 v = *reinterpret_cast<const uint4 *>(src + 4 * t * D + 64 * i);
        r[t][4 * i] = v.x; r[t][4 * i + 1] = v.y; r[t][4 * i + 2] = v.z; r[t][4 * i + 3] = v.w;
      }
    }
  }
}

template <int D>
__device__ inline void load_v(const AttnArgs &a, const Sub &s, int hk, int lane,
                              uint32_t (&r)[D / 16][4]) {
  const int8_t *src =
      a.codes + head_offset(a.p, s.blk, 1, hk) + s.off + ((lane & 15) << a.p.lbs);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const uint4 v = *reinterpret_cast<const uint4 *>(src + (d << (4 + a.p.lbs)));
    r[d][0] = v.x; r[d][1] = v.y; r[d][2] = v.z; r[d][3] = v.w;
  }
}

// Joins the shares of a group's units, `step` floats apart: a wave at a time takes
// a column's exponents (a lane a unit), then the threads the sums, eight units'
// loads in flight.  lds: at least 16 x 64 floats.
template <int D>
__device__ inline void join(const AttnArgs &a, const Columns &c, int hk, int cols, const float *src,
                            int64_t step, int splits, float *lds, float *s_m, float *s_l) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int col = wave; col < cols; col += kSplitWaves) {
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < splits; s += kWave) M = fmaxf(M, src[s * step + col * (D + 2) + D]);
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, kWave));
    for (int s = lane; s < splits; s += kWave) {
      const float *p = src + s * step + col * (D + 2) + D;
      L = fmaf(p[1], share(p[0], M), L);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o, kWave);
    if (lane == 0) {
      s_m[col] = M;
      s_l[col] = L == 0.f ? 1.f : L;
    }
  }
  __syncthreads();
  constexpr int kTasks = kCols * D / 4, kPer = (kTasks + kSplitThreads - 1) / kSplitThreads;
  const int tasks = cols * (D / 4);
  float4_t o[kPer] = {};
  for (int s0 = 0; s0 < splits; s0 += kWave) {
    const int n = min(kWave, splits - s0);
    for (int i = tid; i < cols * kWave; i += kSplitThreads) {
      const int col = i / kWave, s = i % kWave;
      lds[i] = s < n ? share(src[(s0 + s) * step + col * (D + 2) + D], s_m[col]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = tid + k * kSplitThreads, col = i / (D / 4);
      if (i >= tasks) continue;
      const float *at = src + s0 * step + col * (D + 2) + 4 * (i % (D / 4));
      for (int s = 0; s < n; s += 8) {
        float2 x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float *q = at + min(s + e, n - 1) * step;
          x[e] = *reinterpret_cast<const float2 *>(q);
          y[e] = *reinterpret_cast<const float2 *>(q + 2);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (s + e < n) {
            const float f = lds[col * kWave + s + e];
            o[k][0] = fmaf(x[e].x, f, o[k][0]);
            o[k][1] = fmaf(x[e].y, f, o[k][1]);
            o[k][2] = fmaf(y[e].x, f, o[k][2]);
            o[k][3] = fmaf(y[e].y, f, o[k][3]);
          }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = tid + k * kSplitThreads, col = i / (D / 4), x = c.base + col;
    if (i < tasks)
      *reinterpret_cast<float4_t *>(
          a.out + ((int64_t)(c.first + x / a.G) * a.H + hk * a.G + x % a.G) * D +
          4 * (i % (D / 4))) = o[k] / s_l[col];
  }
}

__device__ inline void put2(float *p, float x, float y) {
  const uint64_t bits = ((uint64_t)__float_as_uint(y) << 32) | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), bits, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
template <int D>
__global__ __launch_bounds__(kSplitThreads, 2) void attn_paged_split_kernel(
    AttnArgs a, float *__restrict__ part, unsigned *__restrict__ tickets) {
  constexpr int kOut = D + 4;        // a column's sums in LDS
  __shared__ float s_o[kSplitWaves][kCols][kOut];
  __shared__ float s_m[kSplitWaves][kCols], s_l[kSplitWaves][kCols], s_e[kSplitWaves][kCols];
  __shared__ int s_pick[12], s_sum[kSplitWaves];
  __shared__ int64_t s_tiles[2][kSplitWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int Hkv = a.p.Hkv, per = (a.B + kSplitThreads - 1) / kSplitThreads;
  const int b0 = tid * per, b1 = min(a.B, b0 + per);
  // up to 256 requests: one a thread, read once
  const Part only = b0 < b1 ? part_of(a, b0) : Part{0, 0, 0, 0, 0};
  auto part_at = [&](int b) { return b == b0 ? only : part_of(a, b); };
  int64_t work = 0, groups = 0;
  for (int b = b0; b < b1; ++b) {
    const Part p = part_at(b);
    work += (int64_t)p.tiles * p.groups;
    groups += p.groups;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    work += __shfl_xor(work, o, kWave);
    groups += __shfl_xor(groups, o, kWave);
  }
  if (lane == 0) {
    s_tiles[0][wave] = work;
    s_tiles[1][wave] = groups;
  }
  __syncthreads();
  work = groups = 0;
  for (int w = 0; w < kSplitWaves; ++w) {
    work += s_tiles[0][w];
    groups += s_tiles[1][w];
  }
  // a group of tiles / chunk + 1 units at most: all units run at once
  const int64_t room = max((int64_t)kSplitUnits / 4, kSplitUnits - groups * Hkv);
  const int64_t chunk = max((int64_t)kSplitMin, (work * Hkv + room - 1) / room);
  int mine = 0, shared = 0, sgroups = 0;     // units of a kv head; those and groups that are split
  for (int b = b0; b < b1; ++b) {
    const Part p = part_at(b);
    const int splits = splits_of(p, chunk);
    mine += p.groups * splits;
    if (splits > 1) {
      shared += p.groups * splits;
      sgroups += p.groups;
    }
  }
  const int upto = block_scan(mine, tid, s_sum);
  const int sat = block_scan(shared, tid, s_sum) - shared;
  const int gat = block_scan(sgroups, tid, s_sum) - sgroups;
  if (tid == kSplitThreads - 1) s_pick[11] = upto;
  __syncthreads();
  const int units = s_pick[11] * Hkv;

  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = u / Hkv, hk = u % Hkv;
    // the thread whose requests hold the item looks it up
    if (item < upto && item >= upto - mine) {
      int at = upto - mine, sb = sat, gb = gat;
      for (int b = b0; b < b1; ++b) {
        const Part p = part_at(b);
        const int splits = splits_of(p, chunk), k = p.groups * splits;
        if (item < at + k) {
          const int x = item - at, grp = x / splits;
          s_pick[0] = b;
          s_pick[1] = grp;
          s_pick[2] = x % splits;
          s_pick[3] = splits;
          s_pick[4] = p.tiles;
          s_pick[5] = sb + x;
          s_pick[6] = gb + grp;
          s_pick[8] = p.first;
          s_pick[9] = p.n;
          s_pick[10] = p.len;
          break;
        }
        at += k;
        if (splits > 1) {
          sb += k;
          gb += p.groups;
        }
      }
    }
    __syncthreads();
    const int b = s_pick[0], grp = s_pick[1], split = s_pick[2], splits = s_pick[3];
    const int tiles = s_pick[4], slot = s_pick[5] * Hkv + hk, group = s_pick[6] * Hkv + hk;
    const Columns c{s_pick[8], s_pick[9], grp * kCols, s_pick[10]};
    // key tiles of the unit: of the last row's tokens at most
    const int cols = min(kCols, c.n * a.G - c.base);
    const int64_t most = max((int64_t)0, c.len - c.n + (c.base + cols - 1) / a.G + 1);
    const int64_t least = c.len - c.n + c.base / a.G + 1;   // seen by every column
    const int t0 = (int)min((int64_t)tiles, split * chunk);
    const int t1 = (int)min(min((int64_t)tiles, (split + 1) * chunk), (most + kKeys - 1) / kKeys);
    const int32_t *table = a.tables + (int64_t)b * a.max_blocks;
    const int g = lane >> 4, m4 = (lane & 15) >> 2;
    State<D> st;
    int t = t0 + wave;
    if (t < t1) {
      uint32_t kr[4][D / 16], vr[D / 16][4];
      Sub ks = sub_of(table, (int64_t)t * kKeys + 16 * m4, c.len, a.p);
      Sub vs = sub_of(table, (int64_t)t * kKeys + 16 * g, c.len, a.p);
      load_k<D>(a, ks, hk, lane, kr);
      float ksc = a.scales[scale_offset(a.p, vs.blk, 0, hk)];
      float vsc = a.scales[scale_offset(a.p, vs.blk, 1, hk)];
      load_v<D>(a, vs, hk, lane, vr);
      const Query<D> q = load_query<D>(a, c, hk, lane);
      bool bad = vs.bad;
      for (; t < t1; t += kSplitWaves) {
        const int64_t next = (int64_t)(t + kSplitWaves) * kKeys;
        const bool more = t + kSplitWaves < t1;
        if (more) {
          ks = sub_of(table, next + 16 * m4, c.len, a.p);
          vs = sub_of(table, next + 16 * g, c.len, a.p);
        }
        float4_t acc[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            const half8_t x = codes8(kr[i][2 * k], kr[i][2 * k + 1]);
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.hi[k], acc[i], 0, 0, 0);
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.lo[k], acc[i], 0, 0, 0);
          }
        const float kf = scale_ok(ksc, bad), vf = scale_ok(vsc, bad);
        if (more) {
          load_k<D>(a, ks, hk, lane, kr);
          ksc = a.scales[scale_offset(a.p, vs.blk, 0, hk)];
          vsc = a.scales[scale_offset(a.p, vs.blk, 1, hk)];
          bad = vs.bad;
        }
        half8_t hi[2], lo[2];
        // a v scale that is no number makes the scores NaN too
        const float kn = vf == vf ? kf : vf;
        if ((int64_t)(t + 1) * kKeys <= least && cols == kCols)
          softmax_tile<D, false>(st, acc, kn, vf, q.mul, 16, hi, lo);
        else
          softmax_tile<D, true>(st, acc, kn, vf, q.mul,
                                (int)min(q.see - (int64_t)t * kKeys, (int64_t)kKeys) - 16 * g, hi,
                                lo);
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const half8_t x = codes8(vr[d][2 * k], vr[d][2 * k + 1]);
            st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi[k], st.o[d], 0, 0, 0);
            st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo[k], st.o[d], 0, 0, 0);
          }
        if (more) load_v<D>(a, vs, hk, lane, vr);
      }
    }
    // the four waves' states, then the column's result or the unit's share of it
    const int col = lane & 15;
    st.l = sum_groups(st.l);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      *reinterpret_cast<float4_t *>(&s_o[wave][col][16 * d + 4 * g]) = st.o[d];
    if (g == 0) {
      s_m[wave][col] = st.m;
      s_l[wave][col] = st.l;
      s_e[wave][col] = st.E;
    }
    __syncthreads();
    float *mine_part = part + (int64_t)slot * kCols * (D + 2);
    for (int i = tid; i < cols * (D / 4); i += kSplitThreads) {
      const int cc = i / (D / 4), d4 = i % (D / 4);
      float M = s_m[0][cc];
#pragma unroll
      for (int w = 1; w < kSplitWaves; ++w) M = fmaxf(M, s_m[w][cc]);
      float L = 0.f;
      float4_t o = {};
#pragma unroll
      for (int w = 0; w < kSplitWaves; ++w) {
        L += s_l[w][cc] * share(s_m[w][cc], M);
        const float4_t x = *reinterpret_cast<const float4_t *>(&s_o[w][cc][4 * d4]);
        const int e = (int)(s_e[w][cc] - M) - 15;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] += ldexpf(x[k], e);
      }
      if (splits > 1) {
        float *dst = mine_part + cc * (D + 2);
        put2(dst + 4 * d4, o[0], o[1]);
        put2(dst + 4 * d4 + 2, o[2], o[3]);
        if (d4 == 0) put2(dst + D, M, L);
      } else {
        const int x = c.base + cc;
        if (L == 0.f) L = 1.f;       // no token is seen: the sums are 0
        *reinterpret_cast<float4_t *>(
            a.out + ((int64_t)(c.first + x / a.G) * a.H + hk * a.G + x % a.G) * D + 4 * d4) = o / L;
      }
    }
    if (splits > 1) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (tid == 0) s_pick[7] = atomicAdd(tickets + group, 1u) == (unsigned)splits - 1;
      __syncthreads();
      if (s_pick[7]) {
        // what the others stored is read past this die's caches
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        join<D>(a, c, hk, cols, mine_part - (int64_t)split * Hkv * kCols * (D + 2),
                (int64_t)Hkv * kCols * (D + 2), splits, &s_o[0][0][0], s_m[0], s_l[0]);
        if (tid == 0) atomicExch(tickets + group, 0u);
      }
    }
    __syncthreads();                 // s_pick and the states are free
  }
}

template <int D>
void launch_split(hipStream_t st, const AttnArgs &a, float *part, unsigned *tickets) {
  // as many workgroups as there can be units, up to two a CU; the rest in turn
  const int64_t bound = (int64_t)kSplitUnits +
      (((int64_t)a.T * a.G + kCols - 1) / kCols + std::min(a.B, a.T)) * a.p.Hkv;
  const int grid = (int)std::min<int64_t>(bound, kSplitUnits);
  hipLaunchKernelGGL(attn_paged_split_kernel<D>, dim3(grid), dim3(kSplitThreads), 0, st, a, part,
                     tickets);
}

}  // namespace

// A launch's units that share their columns with another: fewer than 2 units for
// kSplitUnits (a split of `tiles` over chunk has tiles / chunk + 1 < 2 tiles /
// chunk of them), in half as many groups at most.
int64_t attention_paged_part_elems(int D) { return (int64_t)2 * kSplitUnits * kCols * (D + 2); }
int attention_paged_tickets() { return kSplitUnits; }

void launch_attention_paged(hipStream_t st, const float *q, int T, const int8_t *codes,
                            const float *scales, const PagedPool &p, const int32_t *tables,
                            int max_blocks, const int32_t *row_start, const int32_t *lens, int B,
                            int H, float *out, float *part, unsigned *tickets) {
  const AttnArgs a{q, T, codes, scales, p, tables, max_blocks, row_start, lens, B, H, H / p.Hkv,
                   out};
  if (p.D == 32) launch_split<32>(st, a, part, tickets);
  else if (p.D == 64) launch_split<64>(st, a, part, tickets);
  else launch_split<128>(st, a, part, tickets);
  NNHIP_CHECK(hipGetLastError());
}

}  // namespace nnhip
