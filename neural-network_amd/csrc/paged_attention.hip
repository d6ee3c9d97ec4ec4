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
#include <climits>

namespace nnhip {

namespace {

constexpr int kWave = 64;
constexpr int kCols = 16;        // (row, head) columns of a tile of rows
constexpr int kKeys = 64;        // keys of a tile
constexpr int kNone = -(1 << 20);  // E before the first contribution

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

// threadIdx.x for one stretch of code: what is formed from it is formed there, and
// not kept in registers over the loops around.
__device__ inline int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

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

// Blocks and scales of 16 key tiles, `step` tiles apart, a lane for each of a tile's
// four times 16 tokens: read once and passed between the lanes, so that no tile's
// loads wait for the table.  Tokens behind the request's last (len > 0) take its
// block, and are masked; a block outside the pool is read as block 0, with scales
// that make what sees it NaN, as a scale that is no number does.
constexpr int kHeld = 16;
struct Held {
  uint32_t head;                                 // index of the block's k among all heads
  float ks, vs, lvs;                             // lvs: log2(vs)
};
// The first code of a head.
template <int D>
__device__ inline const int8_t *head_at(const AttnArgs &a, uint32_t head) {
  return a.codes + ((uint64_t)head << (a.p.lbs + (D == 128 ? 7 : D == 64 ? 6 : 5)));
}
__device__ inline Held held_tiles(const AttnArgs &a, const int32_t *table, int tile, int step, int len,
                                  int hk) {
  const int lane = threadIdx.x & 63;
  const int tok = (tile + (lane >> 2) * step) * kKeys + 16 * (lane & 3);
  const int blk = table[min(tok, len - 1) >> a.p.lbs];
  const bool bad = !block_ok(blk, a.p.blocks);
  Held r;
  r.head = (uint32_t)scale_offset(a.p, bad ? 0 : blk, 0, hk);
  r.ks = scale_ok(a.scales[r.head], bad);
  r.vs = scale_ok(a.scales[r.head + a.p.Hkv], bad);
  if (r.vs != r.vs) r.ks = r.vs;
  r.lvs = __builtin_amdgcn_logf(r.vs);
  return r;
}

// Columns of a request: column c is row first + c / G, head hk * G + c % G.
struct Columns {
  int first, n, base;            // the request's rows, the unit's first column
  int len;
  const int32_t *table;
};
__device__ inline float *out_row(const AttnArgs &a, const Columns &c, int hk, int col, int D) {
  const int x = c.base + col;
  return a.out + ((int64_t)(c.first + x / a.G) * a.H + hk * a.G + x % a.G) * D;
}

// Two floats that a workgroup of another die reads: written through and read past
// the die's cache.  (A fence in their place would empty the cache for the other
// workgroups, whose keys and values lie in it: 4 x 1000 rows of 16 heads over 4 of 64
// dims in ranges of 10 tiles, 63 us with a fence after the counter, 60 without.)
__device__ inline float2 get2(const float *p) {
  const uint64_t bits = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)bits), __uint_as_float((uint32_t)(bits >> 32)));
}
__device__ inline void put2(float *p, float x, float y) {
  const uint64_t bits = ((uint64_t)__float_as_uint(y) << 32) | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), bits, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

// The power of two that takes a row's largest element to [2^13, 2^14).
__device__ inline int query_shift(float top) {
  return min(13 + 127 - (int)((__float_as_uint(top) >> 23) & 255), 120);
}
// Two weights as halves and what these leave.
__device__ inline void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.f, x),
                                                               fmaf((float)h[1], -1.f, y)));
}

// ---------------------------------------------------------------------------
// Units.
//
// A unit is a tile of columns of one request and kv head over a range of `chunk`
// key tiles: 128 columns where the requests fill them (attn_paged_tall_kernel), else
// 16 (attn_paged_short_kernel, and attn_paged_solo_kernel for many of them).  The
// lengths are on the device, so every workgroup forms the sums over the requests
// itself and takes its units from them; the ranges are chosen so that the units of a
// launch fill the chip, whatever the lengths are.  Where a group of columns has
// several ranges, each unit leaves its state in the scratch, and the last to arrive
// (a counter a group, left zero) joins them, in their order.
constexpr int kShortWaves = 4, kTallWaves = 8;
constexpr int kTallCols = kCols * kTallWaves;
constexpr int kSlots = 512;              // workgroups that run at once: two a CU
// Workgroups of the tall kernel that run at once: its registers allow one a CU for
// 128 dims.
__device__ inline int tall_slots(int D) { return D == 128 ? kSlots / 2 : kSlots; }
constexpr int kShortRoom = kSlots / 4;   // least slots that are shared out by tiles
constexpr int kSoloSlots = kSlots * kShortWaves;
constexpr int kTickets = kSoloSlots;     // counters of groups, then the queues'
// Queues of units, of which a workgroup uses the one of its index, and so mostly of
// its die: takes of one counter are 12 ns apart.  Their counters lie in lines of
// their own, and behind them the one of the workgroups that have ended.
constexpr int kQueues = 8, kLine = 32;
static_assert(kSlots % kQueues == 0, "the queues share out all units");
enum { kShort, kSolo, kTall };
// Least tiles of a unit of several.  Short: 32 requests of up to 1024 tokens 11.3 us
// with 4, 10.3 with 8, 10.4 with 16; one of 4000 tokens (8 heads of 128 dims) 14.2,
// 13.0 and 16.0.  Tall: 4 x 1000 rows of 64 dims 55 us with 6 to 11, 51 with 16; 800
// rows 27 with 8, 29 with 16.
constexpr int kShortMin = 8, kTallMin = 16;

struct Part {                            // a request's share of the work
  int first, n, len;                     // its rows, its tokens
  int groups;                            // tiles of columns
};
template <bool TALL>
__device__ inline Part part_of(const AttnArgs &a, int b) {
  const RowRange r = request_rows(a.row_start, b, a.T);
  const int len = (int)request_len(a.lens[b], a.max_blocks, a.p.lbs);
  Part p{r.first, r.last - r.first, len, 0};
  const int64_t cols = (int64_t)p.n * a.G;
  constexpr int kWide = TALL ? kTallCols : kCols;
  p.groups = (int)((cols + kWide - 1) / kWide);
  return p;
}
__device__ inline int tiles_of(const Part &p) { return (p.len + kKeys - 1) / kKeys; }
// Tokens that column x of a request sees.
__device__ inline int seen_by(int len, int n, int x, int G) { return max(0, len - n + x / G + 1); }

// The ranges of a request.  Short: every group has all of them.  Tall: a group has
// those that its last row sees something of, so range s has groups first_group(s)
// and on: the groups of a row i with len - n + i >= s chunk 64.
template <bool TALL>
struct Ranges {
  int count;                             // of the last group
  int shared;                            // first group that has several
  int chunk, groups;
  int64_t past, G;

  __device__ Ranges(const Part &p, int chunk_, int G_)
      : chunk(chunk_), groups(p.groups), past((int64_t)p.len - p.n), G(G_) {
    count = groups ? max(1, (tiles_of(p) + chunk - 1) / chunk) : 1;
    shared = count > 1 ? first_group(1) : groups;
  }
  __device__ int first_group(int s) const {
    if (!TALL || s == 0) return 0;
    const int64_t row = max((int64_t)0, (int64_t)s * chunk * kKeys - past);
    return (int)min((int64_t)groups, row * G / kTallCols);
  }
  __device__ int units() const {
    if (!TALL) return groups * count;
    int u = 0;
    for (int s = 0; s < count; ++s) u += groups - first_group(s);
    return u;
  }
  // units that share their group
  __device__ int shares() const { return shared < groups ? units() - shared : 0; }
  // ranges of group g
  __device__ int of_group(int g) const {
    if (!TALL) return count;
    int s = 1;
    while (s < count && first_group(s) <= g) ++s;
    return s;
  }
  // place of (group g, range s) among the request's shares, range by range
  __device__ int place(int g, int s) const {
    if (!TALL) return s * groups + g;
    int at = 0;
    for (int i = 0; i < s; ++i) at += groups - max(shared, first_group(i));
    return at + g - max(shared, first_group(s));
  }
};

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

struct Pick {                            // a unit
  int b, group, range, ranges;
  Part part;
  int slot, ticket;                      // of its shares' first, its counter; for kv head 0
};

template <int WAVES>
struct PlanMem {
  // of each thread's requests: units up to them, the first one's place in the
  // scratch and among the counters
  int upto[WAVES * kWave], slot[WAVES * kWave], ticket[WAVES * kWave];
  int sum[WAVES][3];
  float work[WAVES], groups[WAVES];
  int next, last;
};

struct Plan {
  int units, chunk;                        // of a kv head; tiles of a unit
  float work;                              // tiles of all groups of a kv head
};
// FEW: as many requests as a wave has lanes, or fewer.  A lane has one, every wave
// forms all the sums, nothing waits, and a workgroup's first unit is found with the
// lanes' values, `m`: the kernel of 32 requests of up to 1024 tokens takes 9.2 us in
// place of 9.7, of one request of 100 tokens 6.2 in place of 6.8.
constexpr int kFewRequests = kWave;
struct Mine {
  int upto, slot, ticket;
  Part part;
};
template <int KIND, int WAVES, bool FEW>
__device__ inline Plan make_plan(const AttnArgs &a, PlanMem<WAVES> &s, Mine &m) {
  constexpr int kThreads = WAVES * kWave;
  constexpr bool TALL = KIND == kTall;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, Hkv = a.p.Hkv;
  // a few consecutive requests a thread (one, up to as many as there are threads)
  const int per = FEW ? 1 : (a.B + kThreads - 1) / kThreads, b0 = FEW ? lane : tid * per;
  const int b1 = min(a.B, b0 + per);
  const Part only = b0 < b1 ? part_of<TALL>(a, b0) : Part{0, 0, 0, 0};
  auto part_at = [&](int b) { return b == b0 ? only : part_of<TALL>(a, b); };
  // tiles of all groups, from above, and groups: fp32 sums are off by 2^-14 at most
  float work = 0.f, groups = 0.f;
  for (int b = b0; b < b1; ++b) {
    const Part p = part_at(b);
    const float g = (float)p.groups;
    work += TALL ? g * (max(0, p.len - p.n) + 1) / kKeys + g * (g + 1.f) * kTallCols / 2 /
                           (kKeys * (float)a.G) + g
                 : g * (float)tiles_of(p);
    groups += g;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    work += __shfl_xor(work, o, kWave);
    groups += __shfl_xor(groups, o, kWave);
  }
  if (!FEW) {
    if (lane == 0) {
      s.work[wave] = work;
      s.groups[wave] = groups;
    }
    __syncthreads();
    work = groups = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      work += s.work[w];
      groups += s.groups[w];
    }
    __syncthreads();
  }
  // requests that have more rows than there are: counts beyond 32 bits, and no units
  constexpr int kWide = TALL ? kTallCols : kCols;
  if (groups > (float)a.T * a.G / kWide * (1.f + 1.f / 1024) + a.B + 1) return Plan{0, 1, 0.f};
  // Short: work / chunk + groups units, all at once.  Tall, solo: no unit longer than
  // a slot's part of the work (the rows of a prompt see more and more tokens).
  const int room = KIND == kSolo ? kSoloSlots
                   : TALL        ? tall_slots(a.p.D)
                   : groups < kSlots ? max(kShortRoom, kSlots - (int)groups * Hkv)
                                     : kShortRoom;
  const float target = work * (1.f + 1.f / 8192) * Hkv / room;
  // Few long requests: a range costs its own tiles and the join all the ranges'
  // shares, so neither is much longer than the other (one request of 100000 tokens
  // and one head of 64 dims: 30 us in ranges of 8 tiles, 21 in ranges of 29).
  const int least = KIND == kShort ? max(kShortMin, (int)(0.75f * sqrtf(work / fmaxf(groups, 1.f))))
                                   : kTallMin;
  const int chunk = max(least, (int)fminf(target, 1e6f) + 1);
  int mine = 0, shares = 0, shared = 0;      // units, those that share a group, such groups
  for (int b = b0; b < b1; ++b) {
    const Part p = part_at(b);
    const Ranges<TALL> r(p, chunk, a.G);
    mine += r.units();
    shares += r.shares();
    shared += p.groups - r.shared;
  }
  int upto = wave_scan(mine), sat = wave_scan(shares), gat = wave_scan(shared);
  int all = 0;
  if (FEW) {
    all = __builtin_amdgcn_readlane(upto, 63);
  } else {
    if (lane == 63) {
      s.sum[wave][0] = upto;
      s.sum[wave][1] = sat;
      s.sum[wave][2] = gat;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      all += s.sum[w][0];
      if (w < wave) {
        upto += s.sum[w][0];
        sat += s.sum[w][1];
        gat += s.sum[w][2];
      }
    }
  }
  m = Mine{upto, sat - shares, gat - shared, only};
  s.upto[tid] = FEW && wave ? all : m.upto;
  s.slot[tid] = m.slot;
  s.ticket[tid] = m.ticket;
  if (!FEW) __syncthreads();           // FEW: read behind a unit's barriers only
  return Plan{all, chunk, work};
}

// Unit x of a request; slot, ticket: of its first shares and counter.
template <bool TALL>
__device__ inline Pick pick_unit(const AttnArgs &a, const Part &p, int b, int x, int slot, int ticket,
                                 int chunk) {
  const Ranges<TALL> r(p, chunk, a.G);
  // range by range, a prompt's last rows, which see the most, first; short groups
  // one by one
  int g, range = 0;
  if (TALL) {
    while (x >= p.groups - r.first_group(range)) x -= p.groups - r.first_group(range++);
    g = p.groups - 1 - x;
  } else {
    g = x / r.count;
    range = x % r.count;
  }
  auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return Pick{one(b), one(g), one(range), one(r.of_group(g)),
              Part{one(p.first), one(p.n), one(p.len), one(p.groups)}, one(slot),
              one(ticket + g - r.shared)};
}
// Unit `item` (of a kv head) of few requests; item < units.
template <bool TALL>
__device__ inline Pick first_unit(const AttnArgs &a, const Mine &m, int chunk, int item) {
  const int b = __builtin_ctzll(__ballot(m.upto > item));
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, b); };
  const int before = b ? __builtin_amdgcn_readlane(m.upto, b - 1) : 0;
  return pick_unit<TALL>(a, Part{of(m.part.first), of(m.part.n), of(m.part.len), of(m.part.groups)}, b,
                         item - before, of(m.slot), of(m.ticket), chunk);
}

// Unit `item` (of a kv head), the same for the whole wave.
template <bool TALL, int WAVES>
__device__ inline Pick find_unit(const AttnArgs &a, const PlanMem<WAVES> &s, int chunk, int item) {
  constexpr int kThreads = WAVES * kWave;
  const int lane = thread_here() & 63;
  // the first thread whose requests reach beyond it
  const uint64_t beyond = __ballot(s.upto[lane * WAVES + WAVES - 1] > item);
  int tid = beyond ? __builtin_ctzll(beyond) * WAVES : 0;
  while (s.upto[tid] <= item && tid < kThreads - 1) ++tid;
  tid = __builtin_amdgcn_readfirstlane(tid);
  const int per = (a.B + kThreads - 1) / kThreads, b1 = min(a.B, tid * per + per);
  int x = item - (tid ? s.upto[tid - 1] : 0), slot = s.slot[tid], ticket = s.ticket[tid];
  for (int b = tid * per; b < b1; ++b) {
    const Part p = part_of<TALL>(a, b);
    const Ranges<TALL> r(p, chunk, a.G);
    const int units = r.units();
    if (x >= units) {
      x -= units;
      slot += r.shares();
      ticket += p.groups - r.shared;
      continue;
    }
    return pick_unit<TALL>(a, p, b, x, slot, ticket, chunk);
  }
  return Pick{0, 0, 0, 0, Part{0, 0, 0, 0}, 0, 0};   // not reached: item < units
}

// A group's units have left their shares and arrive here; whether this is the
// last of them, which joins.
__device__ inline bool last_of(unsigned *ticket, int ranges, int *s_last) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) *s_last = atomicAdd(ticket, 1u) == (unsigned)ranges - 1;
  __syncthreads();
  if (!*s_last) return false;
  if (threadIdx.x == 0) atomicExch(ticket, 0u);
  return true;
}

// Joins the shares of a group's units: a column's exponents and weights first, a
// lane a unit, then the sums, a thread for four of a column, eight units' loads in
// flight.  at(s): the unit's share.
struct JoinMem { float w[kCols][kWave], m[kCols], l[kCols]; };
template <int D, int WAVES, typename At>
__device__ inline void join(const AttnArgs &a, const Columns &c, int hk, int cols, int ranges,
                            JoinMem &s, At at) {
  constexpr int kThreads = WAVES * kWave;
  const int tid = thread_here(), lane = tid & 63, wave = tid >> 6;
  for (int col0 = 0; col0 < cols; col0 += kCols) {
    const int here = min(kCols, cols - col0);
    for (int col = wave; col < here; col += WAVES) {
      float M = -INFINITY, L = 0.f;
      for (int r = lane; r < ranges; r += kWave) M = fmaxf(M, get2(at(r) + (col0 + col) * (D + 2) + D).x);
#pragma unroll
      for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, kWave));
      for (int r = lane; r < ranges; r += kWave) {
        const float2 ml = get2(at(r) + (col0 + col) * (D + 2) + D);
        L = fmaf(ml.y, share(ml.x, M), L);
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o, kWave);
      if (lane == 0) {
        s.m[col] = M;
        s.l[col] = L == 0.f ? 1.f : L;       // no token is seen: the sums are 0
      }
    }
    __syncthreads();
    constexpr int kPer = (kCols * D / 4 + kThreads - 1) / kThreads;
    float4_t o[kPer] = {};
    for (int r0 = 0; r0 < ranges; r0 += kWave) {
      const int n = min(kWave, ranges - r0);
      for (int i = tid; i < here * kWave; i += kThreads) {
        const int col = i / kWave, r = i % kWave;
        s.w[col][r] = r < n ? share(get2(at(r0 + r) + (col0 + col) * (D + 2) + D).x, s.m[col]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int i = tid + k * kThreads, col = i / (D / 4);
        if (col >= here) continue;
        const int off = (col0 + col) * (D + 2) + 4 * (i % (D / 4));
        for (int r = 0; r < n; r += 8) {
          float2 x[8], y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float *q = at(r0 + min(r + e, n - 1)) + off;
            x[e] = get2(q);
            y[e] = get2(q + 2);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (r + e < n) {
              const float f = s.w[col][r + e];
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
      const int i = tid + k * kThreads, col = i / (D / 4);
      if (col < here)
        *reinterpret_cast<float4_t *>(out_row(a, c, hk, col0 + col, D) + 4 * (i % (D / 4))) =
            o[k] / s.l[col];
    }
    __syncthreads();
  }
}
// The same for a few units, nothing shared between the threads.
constexpr int kFew = 8;
template <int D, int WAVES, typename At>
__device__ inline void join_few(const AttnArgs &a, const Columns &c, int hk, int cols, int ranges,
                                At at) {
  for (int i = thread_here(); i < cols * (D / 4); i += WAVES * kWave) {
    const int col = i / (D / 4), d4 = i % (D / 4);
    float2 ml[kFew], x[kFew], y[kFew];
#pragma unroll
    for (int r = 0; r < kFew; ++r) {
      const float *q = at(min(r, ranges - 1)) + col * (D + 2);
      ml[r] = get2(q + D);
      x[r] = get2(q + 4 * d4);
      y[r] = get2(q + 4 * d4 + 2);
    }
    float M = ml[0].x, L = 0.f;
#pragma unroll
    for (int r = 1; r < kFew; ++r) M = fmaxf(M, ml[r].x);
    float4_t o = {};
#pragma unroll
    for (int r = 0; r < kFew; ++r)
      if (r < ranges) {
        const float f = share(ml[r].x, M);
        L = fmaf(ml[r].y, f, L);
        o[0] = fmaf(x[r].x, f, o[0]);
        o[1] = fmaf(x[r].y, f, o[1]);
        o[2] = fmaf(y[r].x, f, o[2]);
        o[3] = fmaf(y[r].y, f, o[3]);
      }
    if (L == 0.f) L = 1.f;
    *reinterpret_cast<float4_t *>(out_row(a, c, hk, col, D) + 4 * d4) = o / L;
  }
}

// ---------------------------------------------------------------------------
// Short units: 16 columns, the four waves taking the key tiles in turn and joining
// in LDS.
//
// S^T = K Q^T and O^T = V^T P^T: the codes are the left operand, as they lie in
// memory, and the weights that the first product leaves in a lane are what the
// second one wants there.  Lane (r = lane & 15, g = lane >> 4): the left operand of
// score product t holds, in row r, token 16 (r >> 2) + 4 t + (r & 3), dims 16 g ..
// 16 g + 15 of each 64 (the order of the dims is free: four lanes load 64
// neighbouring bytes), so that lane (column, g) gets the scores of tokens 16 g +
// 4 t + i, all of one block; the left operand of the products with v holds dim
// 16 d + r, the 16 tokens of block g.
//
// 4 requests of up to 131072 tokens, 32 heads on 8 of 128 dims: 105 us, 5.3 TB/s, bound
// by memory.  2 chunks of 500 rows beside 31 requests that decode, 16 heads on 4 of
// 128: 62 us, bound by VALU, two fifths of it the codes to halves, which every wave
// forms for its own 16 columns.  32 requests of up to 1024 tokens: 9.5 us, latency.
// The q of a lane's column, and what its scores are multiplied by.  A column
// without a row has q 0 and is written nowhere: it sees all, so that whole tiles
// need no mask.
template <int D>
struct Query {
  half8_t hi[D / 32], lo[D / 32];
  float mul;
  int see;                       // tokens that the column's row sees
};

// The dims of lane group g are `piece` of each `step`, from piece g on (constants).
template <int D>
__device__ inline Query<D> load_query(const AttnArgs &a, const Columns &c, int hk, int ucol,
                                      int step, int piece) {
  Query<D> r;
  const int col = c.base + ucol, g = (threadIdx.x & 63) >> 4;
  const bool live = col < c.n * a.G;
  const int row = live ? col / a.G : 0, h = hk * a.G + (live ? col % a.G : 0);
  const float *src = a.q + ((int64_t)(c.first + row) * a.H + h) * D + g * piece;
  float x[D / 4];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int at = 4 * i / piece * step + 4 * i % piece;
    const float4 v = *reinterpret_cast<const float4 *>(src + at);
    x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < D / 4; ++i) {
    if (!live) x[i] = 0.f;
    top = fmaxf(top, fabsf(x[i]));
  }
  const int up = query_shift(max_groups(top));
#pragma unroll
  for (int k = 0; k < D / 32; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = ldexpf(x[8 * k + j], up);
      r.hi[k][j] = (_Float16)y;
      r.lo[k][j] = (_Float16)(y - (float)r.hi[k][j]);
    }
  r.mul = ldexpf(1.4426950408889634f / sqrtf((float)D), -up);
  r.see = live ? max(0, c.len - c.n + row + 1) : INT_MAX;
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
                                    float lvs, float mul, int visible, half8_t (&hi)[2], half8_t (&lo)[2]) {
  const float mult = ks * mul;
  float top = -FLT_MAX;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = fmaxf(top, !MASK || 4 * t + i < visible ? acc[t][i] : -FLT_MAX);
  const bool none = MASK && visible <= 0;
  const float x = none ? -INFINITY : top * mult;
  const float xm = max_groups(x), am = max_groups(x + lvs);
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
    for (int j = 0; j < 4; ++j) split2(w[8 * c + 2 * j], w[8 * c + 2 * j + 1], h[j], l[j]);
    hi[c] = as_half8(h[0], h[1], h[2], h[3]);
    lo[c] = as_half8(l[0], l[1], l[2], l[3]);
  }
}

// A wave's 16 columns: their results, or the unit's share of them, as the registers
// lie (16 bytes a lane; the wave's part of a share of `width` columns).
template <int D>
__device__ inline void wave_out(const AttnArgs &a, const Columns &c, int hk, int col, int g,
                                const float4_t (&o)[D / 16], float l) {
  float *dst = out_row(a, c, hk, col, D) + 4 * g;
  const float L = l == 0.f ? 1.f : l;             // no token is seen: the sums are 0
#pragma unroll
  for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float4_t *>(dst + 16 * i) = o[i] / L;
}
template <int D>
__device__ inline void wave_end(const AttnArgs &a, const Columns &c, int hk, int col, int cols,
                                int ranges, float *share_at, int part, int width, State<D> &st) {
  const int lane = thread_here() & 63, g = lane >> 4;
  st.l = sum_groups(st.l);
  const int e = (int)(st.E - st.m) - 15;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) st.o[i][k] = ldexpf(st.o[i][k], e);
  if (ranges > 1) {
    float *dst = share_at + (part * (D / 16) * kWave + lane) * 4;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      put2(dst + i * kWave * 4, st.o[i][0], st.o[i][1]);
      put2(dst + i * kWave * 4 + 2, st.o[i][2], st.o[i][3]);
    }
    if (g == 0) put2(share_at + width * D + 2 * col, st.m, st.l);
  } else if (col < cols) {
    wave_out<D>(a, c, hk, col, g, st.o, st.l);
  }
}
// The shares of a group, in the order of the ranges.
template <int D, typename At>
__device__ inline void wave_join(const AttnArgs &a, const Columns &c, int hk, int col, int cols,
                                 int ranges, int part, int width, At at) {
  const int lane = thread_here() & 63, g = lane >> 4;
  float M = -INFINITY, L = 0.f;
  for (int r = g; r < ranges; r += 4) M = fmaxf(M, get2(at(r) + width * D + 2 * col).x);
  M = max_groups(M);
  float4_t o[D / 16] = {};
  constexpr int kAhead = D == 128 ? 2 : 4;       // shares whose loads are in flight
  for (int r0 = 0; r0 < ranges; r0 += kAhead) {
    float2 ml[kAhead], x[kAhead][D / 8];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const float *src = at(min(r0 + e, ranges - 1));
      ml[e] = get2(src + width * D + 2 * col);
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        x[e][i] = get2(src + ((part * (D / 16) + i / 2) * kWave + lane) * 4 + 2 * (i % 2));
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (r0 + e >= ranges) break;
      const float f = share(ml[e].x, M);
      L = fmaf(ml[e].y, f, L);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i / 2][2 * (i % 2)] = fmaf(x[e][i].x, f, o[i / 2][2 * (i % 2)]);
        o[i / 2][2 * (i % 2) + 1] = fmaf(x[e][i].y, f, o[i / 2][2 * (i % 2) + 1]);
      }
    }
  }
  if (col < cols) wave_out<D>(a, c, hk, col, g, o, L);
}

// 16 codes; ONCE: which no other unit reads, and which are not kept in the caches.
template <bool ONCE>
__device__ inline uint4 load16(const int8_t *p) {
  if constexpr (ONCE) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 x = __builtin_nontemporal_load(reinterpret_cast<const u4 *>(p));
    return make_uint4(x.x, x.y, x.z, x.w);
  }
  return *reinterpret_cast<const uint4 *>(p);
}
template <int D, bool ONCE>
__device__ inline void load_k(const AttnArgs &a, uint32_t head, int off, int lane,
                              uint32_t (&r)[4][D / 16]) {
  const int m = lane & 15, g = lane >> 4;
  const int8_t *src = head_at<D>(a, head) + (off + (m & 3)) * D + g * (D == 32 ? 8 : 16);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (D == 32) {
      const uint2 v = *reinterpret_cast<const uint2 *>(src + 4 * t * D);
      r[t][0] = v.x; r[t][1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 v = load16<ONCE>(src + 4 * t * D + 64 * i);
        r[t][4 * i] = v.x; r[t][4 * i + 1] = v.y; r[t][4 * i + 2] = v.z; r[t][4 * i + 3] = v.w;
      }
    }
  }
}

template <int D, bool ONCE>
__device__ inline void load_v(const AttnArgs &a, uint32_t head, int off, int lane,
                              uint32_t (&r)[D / 16][4]) {
  const int8_t *src = head_at<D>(a, head + a.p.Hkv) + off + ((lane & 15) << a.p.lbs);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const uint4 v = load16<ONCE>(src + (d << (4 + a.p.lbs)));
    r[d][0] = v.x; r[d][1] = v.y; r[d][2] = v.z; r[d][3] = v.w;
  }
}

template <int D>
struct ShortMem {
  float o[kShortWaves][kCols][D + 4], m[kShortWaves][kCols], l[kShortWaves][kCols], e[kShortWaves][kCols];
};

template <int D>
__device__ inline void short_scores(const uint32_t (&kr)[4][D / 16], const Query<D> &q,
                                    float4_t (&acc)[4]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half8_t x = codes8(kr[i][2 * j], kr[i][2 * j + 1]);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.hi[j], acc[i], 0, 0, 0);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.lo[j], acc[i], 0, 0, 0);
    }
}
template <int D>
__device__ inline void short_sums(const uint32_t (&vr)[D / 16][4], const half8_t (&hi)[2],
                                  const half8_t (&lo)[2], State<D> &st) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const half8_t x = codes8(vr[i][2 * j], vr[i][2 * j + 1]);
      st.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi[j], st.o[i], 0, 0, 0);
      st.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo[j], st.o[i], 0, 0, 0);
    }
}

// The state of a wave after key tiles t, t + STEP, .. below `end`, of 16 columns.
template <int D, int STEP, bool ONCE>
__device__ inline void short_tiles(const AttnArgs &a, const Columns &c, int hk, int t, int end,
                                   State<D> &st) {
  const int lane = thread_here() & 63, g = lane >> 4, m4 = (lane & 15) >> 2;
  const int least =                  // seen by every column
      __builtin_amdgcn_readfirstlane(seen_by(c.len, c.n, c.base, a.G));
  if (t >= end) return;
  uint32_t kr[4][D / 16], vr[D / 16][4];
  // places of the tile's tokens 16 m4 (k) and 16 g (v, scales) in their blocks
  auto place = [&](int tile, int sub) { return (tile * kKeys + 16 * sub) & (a.p.bs - 1); };
  Held held = held_tiles(a, c.table, t, STEP, c.len, hk);
  int at = 0;
  auto head = [&](int sub) { return (uint32_t)__shfl((int)held.head, 4 * at + sub, kWave); };
  load_k<D, ONCE>(a, head(m4), place(t, m4), lane, kr);
  load_v<D, ONCE>(a, head(g), place(t, g), lane, vr);
  const Query<D> q = load_query<D>(a, c, hk, lane & 15, D == 32 ? 32 : 64, D == 32 ? 8 : 16);
  for (; t + STEP < end; t += STEP) {
    const float ks = __shfl(held.ks, 4 * at + g, kWave), vs = __shfl(held.vs, 4 * at + g, kWave);
    const float lvs = __shfl(held.lvs, 4 * at + g, kWave);
    if (++at == kHeld) {
      held = held_tiles(a, c.table, t + STEP, STEP, c.len, hk);
      at = 0;
    }
    const uint32_t k_head = head(m4), v_head = head(g);
    float4_t acc[4] = {};
    short_scores<D>(kr, q, acc);
    load_k<D, ONCE>(a, k_head, place(t + STEP, m4), lane, kr);
    half8_t hi[2], lo[2];
    if ((t + 1) * kKeys <= least)
      softmax_tile<D, false>(st, acc, ks, vs, lvs, q.mul, 16, hi, lo);
    else
      softmax_tile<D, true>(st, acc, ks, vs, lvs, q.mul, min(q.see - t * kKeys, kKeys) - 16 * g, hi,
                            lo);
    short_sums<D>(vr, hi, lo, st);
    load_v<D, ONCE>(a, v_head, place(t + STEP, g), lane, vr);
  }
  // the last tile on its own: a condition on the loads within the loop would have
  // them all waited for
  float4_t acc[4] = {};
  half8_t hi[2], lo[2];
  short_scores<D>(kr, q, acc);
  softmax_tile<D, true>(st, acc, __shfl(held.ks, 4 * at + g, kWave),
                        __shfl(held.vs, 4 * at + g, kWave), __shfl(held.lvs, 4 * at + g, kWave),
                        q.mul, min(q.see - t * kKeys, kKeys) - 16 * g, hi, lo);
  short_sums<D>(vr, hi, lo, st);
}
// Key tiles of a unit: up to the last row's tokens.
__device__ inline int end_of(const AttnArgs &a, const Columns &c, int start, int chunk, int cols) {
  // (through a division, which leaves it in a vector register)
  return __builtin_amdgcn_readfirstlane(
      min(start + chunk, (seen_by(c.len, c.n, c.base + cols - 1, a.G) + kKeys - 1) / kKeys));
}

template <int D, bool ONCE>
__device__ inline void short_unit(const AttnArgs &a, const Columns &c, const Pick &u, int hk,
                                  int chunk, float *share_at, ShortMem<D> &s) {
  const int tid = thread_here(), lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cols = min(kCols, c.n * a.G - c.base), start = u.range * chunk;
  State<D> st;
  short_tiles<D, kShortWaves, ONCE>(a, c, hk, start + wave, end_of(a, c, start, chunk, cols), st);
  // the four waves' states, then the columns' results or the unit's share of them
  const int col = lane & 15;
  st.l = sum_groups(st.l);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    *reinterpret_cast<float4_t *>(&s.o[wave][col][16 * i + 4 * g]) = st.o[i];
  if (g == 0) {
    s.m[wave][col] = st.m;
    s.l[wave][col] = st.l;
    s.e[wave][col] = st.E;
  }
  __syncthreads();
  for (int i = tid; i < cols * (D / 4); i += (kShortWaves * kWave)) {
    const int cc = i / (D / 4), d4 = i % (D / 4);
    float M = s.m[0][cc];
#pragma unroll
    for (int w = 1; w < kShortWaves; ++w) M = fmaxf(M, s.m[w][cc]);
    float L = 0.f;
    float4_t o = {};
#pragma unroll
    for (int w = 0; w < kShortWaves; ++w) {
      L += s.l[w][cc] * share(s.m[w][cc], M);
      const float4_t x = *reinterpret_cast<const float4_t *>(&s.o[w][cc][4 * d4]);
      const int e = (int)(s.e[w][cc] - M) - 15;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += ldexpf(x[k], e);
    }
    if (u.ranges > 1) {
      float *dst = share_at + cc * (D + 2);
      put2(dst + 4 * d4, o[0], o[1]);
      put2(dst + 4 * d4 + 2, o[2], o[3]);
      if (d4 == 0) put2(dst + D, M, L);
    } else {
      if (L == 0.f) L = 1.f;           // no token is seen: the sums are 0
      *reinterpret_cast<float4_t *>(out_row(a, c, hk, cc, D) + 4 * d4) = o / L;
    }
  }
}

// ---------------------------------------------------------------------------
// Tall units: 128 columns, 16 a wave, over key tiles in LDS.
//
// The workgroup turns a tile's codes into halves once (two buffers: the next tile's
// codes are loaded while a tile is worked on) and its waves read them as left
// operands.  Row r of score product t is token 16 t + r, so lane (column, g) gets
// the scores of tokens 16 t + 4 g + i, and the products with v take 32 tokens a step
// in the order 4 g + i, 16 + 4 g + i, in which v is laid out.  A row has 16 bytes
// more than its halves: 16 rows' pieces lie in different banks, at offsets that are
// constants.  All columns see the same blocks: a scale is the same for the wave.
//
// 8000 rows of 32 heads on 8: 650 us with 64 dims, 1.11 ms with 128, 400 and 475 TFLOP/s
// of the formula's own products, bound by VALU (the softmax, the weights' halves, the
// codes' conversion).  4 prompts of up to 1000 rows, 16 heads on 4 of 64 dims: 49 us, bound
// by the longest unit.  Side by side with it v's rows were laid out so that the stores
// miss each other's banks: no change.
template <int D>
struct TallMem {
  uint4 k[2][kKeys][D / 8 + 1];        // [token][8 dims]
  uint4 v[2][D][8 + 1];                // [dim][32 tokens: g]
};

__device__ inline uint4 as_u4(half8_t x) { return __builtin_bit_cast(uint4, x); }
__device__ inline half8_t as_half8(uint4 x) { return __builtin_bit_cast(half8_t, x); }
__device__ inline float lane_of(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// The codes of a tile that a thread brings, 16 of them: of k 16 dims of a token, of v
// 16 tokens of a dim.  Waves bring either (k: the waves behind v's), or, for 128 dims,
// both.  Every address is a head's and one of 32 bits.
template <int D>
struct TallLoad { uint4 k, v; };                 // D < 128: v alone, for both
template <int D>
constexpr int tall_first() { return D == 128 ? 0 : 4 * D; }  // k's first thread
__device__ inline int tall_thread() { return thread_here() & (kTallWaves * kWave - 1); }
template <int D>
__device__ inline void tall_load(const AttnArgs &a, const Held &h, int at, int tok, int wave,
                                 TallLoad<D> &r) {
  const int m = a.p.bs - 1;
  auto load = [](const int8_t *p) { return *reinterpret_cast<const uint4 *>(p); };
  auto head = [&](int sub) { return (uint32_t)__shfl((int)h.head, 4 * at + sub, kWave); };
  auto load_k = [&] {
    const int id = tall_thread() - tall_first<D>();
    if constexpr (D == 32) {
      const int sub = (id >> 5) & 3;
      return load(head_at<D>(a, head(sub)) + (((tok + 16 * sub) & m) * D + (id & (D - 1)) * 16));
    } else {
      const int sub = (wave - tall_first<D>() / kWave) / (D / kWave);
      const uint32_t k = __builtin_amdgcn_readlane(h.head, 4 * at + sub);
      return load(head_at<D>(a, k) + ((tok + 16 * sub) & m) * D + (id & (D - 1)) * 16);
    }
  };
  auto load_v = [&] {
    const int id = tall_thread(), sub = id & 3;
    return load(head_at<D>(a, head(sub) + a.p.Hkv) +
                (((tok + 16 * sub) & m) + ((id >> 2) << a.p.lbs)));
  };
  if constexpr (D == 128) {
    r.k = load_k();
    r.v = load_v();
  } else if (wave < 4 * D / kWave) {
    r.v = load_v();
  } else if (wave < 8 * D / kWave) {
    r.v = load_k();
  }
}
template <int D>
__device__ inline void tall_store(TallMem<D> &s, int buf, int wave, const TallLoad<D> &r) {
  auto store_k = [&](const uint4 &x) {
    const int id = tall_thread() - tall_first<D>();
    uint4 *row = &s.k[buf][0][0] + __umul24(id / (D / 16), D / 8 + 1) + 2 * (id & (D / 16 - 1));
    row[0] = as_u4(codes8(x.x, x.y));
    row[1] = as_u4(codes8(x.z, x.w));
  };
  auto store_v = [&](const uint4 &x) {
    // block b of the tile: tokens 4 g .. of it, at half b % 2 of piece 4 (b / 2) + g
    const int id = tall_thread(), b = id & 3;
    uint2 *row = reinterpret_cast<uint2 *>(&s.v[buf][0][0]) + __umul24(id >> 2, 18) + 8 * (b >> 1) +
                 (b & 1);
    const uint4 lo = as_u4(codes8(x.x, x.y)), hi = as_u4(codes8(x.z, x.w));
    row[0] = make_uint2(lo.x, lo.y);
    row[2] = make_uint2(lo.z, lo.w);
    row[4] = make_uint2(hi.x, hi.y);
    row[6] = make_uint2(hi.z, hi.w);
  };
  if constexpr (D == 128) {
    store_k(r.k);
    store_v(r.v);
  } else if (wave < 4 * D / kWave) {
    store_v(r.v);
  } else if (wave < 8 * D / kWave) {
    store_k(r.v);
  }
}

// A tile's scales, in scalar registers.
struct Scales { float ks[4], vs[4], lvs[4]; };
__device__ inline Scales scales_of(const Held &h, int at) {
  Scales s;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    s.ks[b] = lane_of(h.ks, 4 * at + b);
    s.vs[b] = lane_of(h.vs, 4 * at + b);
    s.lvs[b] = lane_of(h.lvs, 4 * at + b);
  }
  return s;
}

// Scores, softmax and products with v of a tile.  visible: tokens of the tile that
// the lane's column sees, counted from the lane's first one.
template <int D, bool MASK>
__device__ inline void tall_tile(const TallMem<D> &s, int buf, const Scales &sc, const Query<D> &q,
                                 State<D> &st, int visible) {
  const int lane = thread_here() & 63, r = lane & 15, g = lane >> 4;
  float4_t acc[4] = {};
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    half8_t x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = as_half8(s.k[buf][16 * t + r][4 * k + g]);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[t], q.hi[k], acc[t], 0, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[t], q.lo[k], acc[t], 0, 0, 0);
  }
  float ks[4], xm = -INFINITY, am = -INFINITY;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    ks[t] = sc.ks[t] * q.mul;
    float top = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = fmaxf(top, !MASK || 16 * t + i < visible ? acc[t][i] : -FLT_MAX);
    const float x = MASK && 16 * t >= visible ? -INFINITY : top * ks[t];
    xm = fmaxf(xm, x);
    am = fmaxf(am, x + sc.lvs[t]);
  }
  const float m = fmaxf(st.m, ceilf(max_groups(xm)));
  st.l *= share(st.m, m);
  st.m = m;
  const float E = fmaxf(st.E, ceilf(max_groups(am)));
  if (__any(st.E != E)) {              // seldom, after the first tiles
    const float f = __builtin_amdgcn_exp2f(st.E - E);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i] *= f;
  }
  st.E = E;
  const float base = m == -INFINITY ? 0.f : m;
  const int shift = (int)(base - E) + 15;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float factor = fminf(ldexpf(sc.vs[2 * c + t], shift), FLT_MAX);
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = __builtin_amdgcn_exp2f(fmaf(acc[2 * c + t][i], ks[2 * c + t], -base));
        if (MASK && 16 * (2 * c + t) + i >= visible) x = 0.f;
        st.l += x;
        w[i] = x * factor;
      }
      split2(w[0], w[1], h[2 * t], l[2 * t]);
      split2(w[2], w[3], h[2 * t + 1], l[2 * t + 1]);
    }
    const half8_t hi = as_half8(h[0], h[1], h[2], h[3]), lo = as_half8(l[0], l[1], l[2], l[3]);
    constexpr int kRun = D == 32 ? 2 : 4;
#pragma unroll
    for (int i0 = 0; i0 < D / 16; i0 += kRun) {
      half8_t x[kRun];
#pragma unroll
      for (int i = 0; i < kRun; ++i) x[i] = as_half8(s.v[buf][16 * (i0 + i) + r][4 * c + g]);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        st.o[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], hi, st.o[i0 + i], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        st.o[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], lo, st.o[i0 + i], 0, 0, 0);
    }
  }
}

template <int D>
__device__ inline void tall_unit(const AttnArgs &a, const Columns &c, const Pick &u, int hk,
                                 int chunk, float *share_at, TallMem<D> &s) {
  const int tid = thread_here(), lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cols = min(kTallCols, c.n * a.G - c.base);
  const int col = kCols * wave + (lane & 15);
  // tokens that the unit's last column, and the wave's last and first ones see
  const bool any = kCols * wave < cols;
  auto seen = [&](int x) { return seen_by(c.len, c.n, c.base + x, a.G); };
  const int start = u.range * chunk;
  const int end = end_of(a, c, start, chunk, cols);
  const int most = __builtin_amdgcn_readfirstlane(
      any ? seen(min(cols, kCols * wave + kCols) - 1) : 0);
  const int least = __builtin_amdgcn_readfirstlane(any ? seen(kCols * wave) : 0);
  State<D> st;
  if (start < end) {
    TallLoad<D> r;
    Held held = held_tiles(a, c.table, start, 1, c.len, hk);
    int at = 0, t = start;
    tall_load<D>(a, held, 0, start * kKeys, wave, r);
    const Query<D> q = load_query<D>(a, c, hk, col, 32, 8);
    tall_store<D>(s, 0, wave, r);
    __syncthreads();
    // a tile, while the next one's codes are on their way
    auto step = [&](auto tile) {
      const int buf = (t - start) & 1;
      const Scales sc = scales_of(held, at);
      if (t + 1 < end) {
        if (++at == kHeld) {
          held = held_tiles(a, c.table, t + 1, 1, c.len, hk);
          at = 0;
        }
        tall_load<D>(a, held, at, (t + 1) * kKeys, wave, r);
      }
      tile(buf, sc);
      if (t + 1 < end) tall_store<D>(s, buf ^ 1, wave, r);
      __syncthreads();
    };
    // tiles that the wave's columns see whole, then the others: two loops, whose sums
    // stay in the registers that they are in
    for (const int whole = min(end, least / kKeys); t < whole; ++t)
      step([&](int buf, const Scales &sc) { tall_tile<D, false>(s, buf, sc, q, st, kKeys); });
    for (; t < end; ++t)
      step([&](int buf, const Scales &sc) {
        if (t * kKeys < most)
          tall_tile<D, true>(s, buf, sc, q, st, min(q.see - t * kKeys, kKeys) - 4 * g);
      });
  }
  if (any) wave_end<D>(a, c, hk, col, cols, u.ranges, share_at, wave, kTallCols, st);
}

// What a unit works on.
template <int D, bool TALL>
struct Unit {
  static constexpr int kWide = TALL ? kTallCols : kCols;
  Pick u;
  int hk, cols;
  Columns c;
  Ranges<TALL> r;
  float *shares;
  int64_t step;
  __device__ Unit(const AttnArgs &a, const Pick &u_, int hk_, int chunk, float *scratch)
      : u(u_), hk(hk_),
        c{u.part.first, u.part.n, kWide * u.group, u.part.len, a.tables + (int64_t)u.b * a.max_blocks},
        r(u.part, chunk, a.G) {
    cols = min(kWide, c.n * a.G - c.base);
    step = (int64_t)a.p.Hkv * kWide * (D + 2);
    shares = scratch + u.slot * step + (int64_t)hk * kWide * (D + 2);
  }
  __device__ float *share_of(int range) const { return shares + r.place(u.group, range) * step; }
};

// Workgroups take the unit of their index first, then units from a queue; the last
// to end leaves the counters zero.
__device__ inline unsigned take_unit(unsigned *queues) {
  const unsigned q = blockIdx.x % kQueues;
  return gridDim.x + kQueues * atomicAdd(queues + kLine * q, 1u) + q;
}
__device__ inline void leave_queues(unsigned *queues) {
  if (atomicAdd(queues + kLine * kQueues, 1u) == gridDim.x - 1)
    for (int q = 0; q <= kQueues; ++q) atomicExch(queues + kLine * q, 0u);
}

template <int D, int KIND, int WAVES, bool FEW, typename Run>
__device__ inline void run_units(const AttnArgs &a, float *scratch, unsigned *tickets,
                                 PlanMem<WAVES> &s, JoinMem &jm, Run run) {
  constexpr bool TALL = KIND == kTall;
  unsigned *queues = tickets + kTickets;
  const int Hkv = a.p.Hkv;
  Mine mine;
  const Plan plan = make_plan<KIND, WAVES, FEW>(a, s, mine);
  const int chunk = __builtin_amdgcn_readfirstlane(plan.chunk);
  const unsigned units = __builtin_amdgcn_readfirstlane(plan.units * Hkv);
  unsigned at = blockIdx.x;
  Pick pick{};
  if (FEW && at < units) pick = first_unit<TALL>(a, mine, chunk, at / Hkv);
  while (at < units) {
    if (!FEW) pick = find_unit<TALL, WAVES>(a, s, chunk, at / Hkv);
    const Unit<D, TALL> w(a, pick, at % Hkv, chunk, scratch);
    if (threadIdx.x == 0) s.next = units > gridDim.x ? take_unit(queues) : units;
    run(plan, w.c, w.u, w.hk, chunk, w.u.ranges > 1 ? w.share_of(w.u.range) : nullptr);
    if (w.u.ranges > 1 && last_of(tickets + (int64_t)w.u.ticket * Hkv + w.hk, w.u.ranges, &s.last)) {
      auto share_of = [&](int range) { return w.share_of(range); };
      if constexpr (TALL) {
        const int wave = __builtin_amdgcn_readfirstlane(thread_here() >> 6);
        if (kCols * wave < w.cols)
          wave_join<D>(a, w.c, w.hk, kCols * wave + (thread_here() & 15), w.cols, w.u.ranges, wave,
                       kTallCols, share_of);
      } else if (w.u.ranges <= kFew) {
        join_few<D, WAVES>(a, w.c, w.hk, w.cols, w.u.ranges, share_of);
      } else {
        join<D, WAVES>(a, w.c, w.hk, w.cols, w.u.ranges, jm, share_of);
      }
    }
    __syncthreads();                   // s.next is there
    at = __builtin_amdgcn_readfirstlane(s.next);
    __syncthreads();                   // the LDS is free
    if (FEW && at < units) pick = find_unit<TALL, WAVES>(a, s, chunk, at / Hkv);
  }
  if (units > gridDim.x && threadIdx.x == 0) leave_queues(queues);
}

// Whether codes are read once: requests of a group of columns, and more codes than the
// caches would hold (kept / not kept: 4 requests of up to 131072 tokens, 8 heads of 128
// dims, 109 / 105 us, 128 of up to 1000 46 / 43, 64 of up to 8000 in blocks of 16 with
// 64 dims 74 / 68, with 128 dims, though, 136 / 142; with half as many codes 16 of up to
// 8000, 64 dims, 22.4 / 23.3).
template <int D>
__device__ inline bool once_pays(const AttnArgs &a, const Plan &plan) {
  return (int64_t)a.T * a.G <= (int64_t)kCols * a.B && plan.work * (2 * D * kKeys) * a.p.Hkv > 1e8f;
}

// Units of 16 columns with a wave each, where there are so many of them that four
// waves a unit would wait more than work: 512 requests of up to 300 tokens, 16 heads of
// 64 dims, 55 us, 2.9 TB/s.
template <int D>
__global__ __launch_bounds__(kShortWaves *kWave, 2) void attn_paged_solo_kernel(
    AttnArgs a, float *__restrict__ scratch, unsigned *__restrict__ tickets) {
  __shared__ PlanMem<kShortWaves> s;
  const int Hkv = a.p.Hkv;
  Mine mine;
  const Plan plan = make_plan<kSolo, kShortWaves, false>(a, s, mine);
  const int chunk = __builtin_amdgcn_readfirstlane(plan.chunk);
  const unsigned units = __builtin_amdgcn_readfirstlane(plan.units * Hkv);
  const unsigned takers = gridDim.x * kShortWaves;
  // neighbouring waves of different workgroups first: few units spread over the chip
  unsigned at = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * gridDim.x + blockIdx.x;
  for (; at < units; at += takers) {
    const Unit<D, false> w(a, find_unit<false, kShortWaves>(a, s, chunk, at / Hkv), at % Hkv, chunk,
                           scratch);
    const int col = thread_here() & 15, start = w.u.range * chunk;
    State<D> st;
    short_tiles<D, 1, false>(a, w.c, w.hk, start, end_of(a, w.c, start, chunk, w.cols), st);
    wave_end<D>(a, w.c, w.hk, col, w.cols, w.u.ranges,
                w.u.ranges > 1 ? w.share_of(w.u.range) : nullptr, 0, kCols, st);
    if (w.u.ranges > 1) {
      __builtin_amdgcn_s_waitcnt(0);
      unsigned *ticket = tickets + (int64_t)w.u.ticket * Hkv + w.hk;
      unsigned n = 0;
      if ((thread_here() & 63) == 0) n = atomicAdd(ticket, 1u);
      if (__builtin_amdgcn_readfirstlane(n) == (unsigned)w.u.ranges - 1) {
        if ((thread_here() & 63) == 0) atomicExch(ticket, 0u);
        wave_join<D>(a, w.c, w.hk, col, w.cols, w.u.ranges, 0, kCols,
                     [&](int range) { return w.share_of(range); });
      }
    }
  }
}

template <int D, bool FEW>
__global__ __launch_bounds__(kShortWaves *kWave, 2) void attn_paged_short_kernel(
    AttnArgs a, float *__restrict__ scratch, unsigned *__restrict__ tickets) {
  __shared__ PlanMem<kShortWaves> s_plan;
  __shared__ __align__(16) union { ShortMem<D> unit; JoinMem join; } s;
  run_units<D, kShort, kShortWaves, FEW>(a, scratch, tickets, s_plan, s.join,
                                   [&](const Plan &plan, const Columns &c, const Pick &u, int hk, int chunk, float *to) {
                                     if (once_pays<D>(a, plan)) short_unit<D, true>(a, c, u, hk, chunk, to, s.unit);
                                     else short_unit<D, false>(a, c, u, hk, chunk, to, s.unit);
                                   });
}

template <int D, bool FEW>
__global__ __launch_bounds__(kTallWaves *kWave, D == 128 ? 2 : 4) void attn_paged_tall_kernel(
    AttnArgs a, float *__restrict__ scratch, unsigned *__restrict__ tickets) {
  __shared__ PlanMem<kTallWaves> s_plan;
  __shared__ __align__(16) union { TallMem<D> unit; JoinMem join; } s;
  run_units<D, kTall, kTallWaves, FEW>(a, scratch, tickets, s_plan, s.join,
                                 [&](const Plan &plan, const Columns &c, const Pick &u, int hk, int chunk, float *to) {
                                   tall_unit<D>(a, c, u, hk, chunk, to, s.unit);
                                 });
}

template <int D>
void launch(hipStream_t st, const AttnArgs &a, float *scratch, unsigned *tickets) {
  auto run = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(kSlots), dim3(waves * kWave), 0, st, a, scratch, tickets);
  };
  const bool few = a.B <= kFewRequests;
  if (attention_paged_tall(a.T, a.B, a.G, a.p.Hkv)) {
    if (few) run(attn_paged_tall_kernel<D, true>, kTallWaves);
    else run(attn_paged_tall_kernel<D, false>, kTallWaves);
  } else if (attention_paged_solo(a.T, a.B, a.G, a.p.Hkv)) {
    run(attn_paged_solo_kernel<D>, kShortWaves);
  } else if (few) {
    run(attn_paged_short_kernel<D, true>, kShortWaves);
  } else {
    run(attn_paged_short_kernel<D, false>, kShortWaves);
  }
}

}  // namespace

// Units that share their group.  Short: with room = kSlots - groups, work / chunk +
// groups of them, kSlots; with room = kShortRoom, tiles / chunk + 1 < 2 tiles / chunk
// for each group that has several, 2 kShortRoom.  Likewise 2 kSoloSlots of 16 and
// 2 kSlots of 128 columns, and half as many groups.
int64_t attention_paged_part_elems(int D) {
  return std::max((int64_t)2 * kSoloSlots * kCols, (int64_t)2 * kSlots * kTallCols) * (D + 2);
}
int attention_paged_tickets() { return kTickets + kLine * kQueues + 1; }

void launch_attention_paged(hipStream_t st, const float *q, int T, const int8_t *codes,
                            const float *scales, const PagedPool &p, const int32_t *tables,
                            int max_blocks, const int32_t *row_start, const int32_t *lens, int B,
                            int H, float *out, float *part, unsigned *tickets) {
  const int G = H / p.Hkv;
  const AttnArgs a{q, T, codes, scales, p, tables, max_blocks, row_start, lens, B, H, G, out};
  if (p.D == 32) launch<32>(st, a, part, tickets);
  else if (p.D == 64) launch<64>(st, a, part, tickets);
  else launch<128>(st, a, part, tickets);
  NNHIP_CHECK(hipGetLastError());
}

}  // namespace nnhip
