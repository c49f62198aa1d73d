// One token per row of logits from a given uniform (the batched counterpart of
// Sampler::sample, sampler.rs:47-109, whose draw order and filters it keeps,
// with min-p added and no random state of its own).
//
// With w_i = exp((x_i - max x) / T) and the rank order (x descending, index
// ascending), the kept tokens are a prefix of the rank order, the shortest of
//   top-k   the first k,
//   top-p   up to the first token whose running sum of w reaches top_p * sum w
//           (over the whole row, as the reference's cutoff),
//   min-p   w_i >= min_p,
// and never less than the first token. The draw takes the first kept token
// whose running sum reaches u * (kept sum): in rank order when a filter is
// on, in index order otherwise. Tokens at -infinity (or NaN) have w = 0 and
// are never drawn, nor are others whose w is 0 in f64 (745 T below the maximum);
// a row without any other token gives token 0.
//
// Next to a border a draw is decided by digits that an f32 sum over a
// vocabulary does not hold (with 100,000 even tokens, borders moved by 1e-7 of
// the mass would change one draw in a hundred). So weights are integers and sums
// of integers: no result depends on an order of summation, and the roundings of
// 100,000 even tokens move a border by about 1e-6 of one token. What is rounded:
//   * a weight has 30 bits in its bucket's unit (within 2^-28 of itself; from
//     2^20 logits on 28 to 26 bits, cut, so that a CTA's sums fit 32);
//   * sums over buckets are in units of 2^-b of the maximum's weight, b = 62 -
//     ceil(log2 n), at most 47 (44 at 151936 logits, 40 at 4194304). A weight below
//     2^(28 - b) has fewer than 28 bits there, one below 2^-b none;
//   * the histogram cuts a bucket's sum once to that unit and a list each token, so
//     the two may differ by a unit a token: at most n units, 2^-26 of the maximum's
//     weight at 151936 logits and 2^-18 at 4194304.
// The exponent 256 log2 w comes from
// one f64 FMA whose addend leaves 24 fractional bits; 2^(a/256) is the
// table-driven exponential (Tang 1989), a table of 256 steps and a polynomial
// of degree 3 for the rest, in f32 and integers.
//
// A cluster of up to 8 CTAs holds a row in shared memory (one pass over HBM,
// bulk copies), so every further pass runs at shared-memory speed:
//   1. the maximum;
//   2. a histogram over 512 buckets of (max - x) / T, 1/32 wide: counts, and
//      the mass in two 32-bit parts, in units of the bucket (shared-memory
//      atomics are fast in 32 bits only). Each CTA adds up a slice of the buckets
//      over the cluster; the running sums give the bucket of the last kept token (by count and by
//      mass alike) and, for a given mass, that of the draw;
//   3. the tokens of that bucket are listed, sorted and summed, which settles the
//      border exactly. A crowded bucket is split again by the key's
//      bits; equal logits beyond the list's room are counted in index order.
// When the kept tokens fit the list as a whole, one list serves both borders
// and no mass histogram is needed. Every CTA of the cluster reads the others'
// sums and lists over distributed shared memory and decides alike, so there
// is no result to send round.
//
// Measured: 64 rows of 151936 62 us (39 MB: 6 us at the copy rate), 256 of 128257
// 205 us, one row 23 us. Bound by the chain of a row's passes and barriers over the
// cluster, not by bytes: a scheduler issues in 0.43 of its cycles. The sides of the
// choices, us at 64 x 151936 / 256 x 128257: 8 CTAs a row holding it in shared memory
// 62 / 205, 4 holding it 70 / 234, 8 reading it again from L2 96 / 314, 4 so
// 107 / 273; 384 threads a CTA 68 / 225, 512 79 / 258. A row that shared memory
// cannot hold (more than 8 x kRowsCached = 390784 tokens) is read again.
#include <cooperative_groups.h>
#include <math.h>

#include <string>

#include "common.cuh"
#include "kernels.h"
#include "pipeline.cuh"

namespace minq {

namespace {

namespace cg = cooperative_groups;

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsBuckets = 512;           // two per thread
constexpr float kRowsPerNat = 32.0f;        // buckets per unit of (max - x) / T
constexpr int kRowsList = 4 * kRowsThreads; // tokens a list holds: four per thread
constexpr int kRowsMaxCtas = 8;             // the portable cluster size
constexpr int kRowsTable = 256;
constexpr size_t kRowsSmem = 227 * 1024;    // shared memory of a CTA

struct RowsParams {
  const float* logits;
  size_t stride;
  uint32_t n, chunk;         // chunk: elements per CTA
  bool cached;
  int part_bits, drop;       // a weight's 30 bits less `drop`, in two parts of part_bits
  int mass_bits;             // of w = 1 in 64-bit sums
  const float* temperature;  // null: 1
  const int* top_k;          // null or <= 0: off
  const float* top_p;        // null or >= 1: off
  const float* min_p;        // null or <= 0: off
  const float* u;
  uint32_t* out;
  uint32_t stall;            // bytes the row's wait expects beyond its copies (tests)
};

// Whether a token can be drawn (a number above -infinity).
__device__ __forceinline__ bool rows_real(float v) { return v > -INFINITY; }

// The least logit that weighs anything: below it exp((x - max) / T) is 0 even in
// f64 (2^-1075 = e^-745.13). Only a uniform of 0 asks: any other target is reached
// by a weight that the sums hold, 0 by whatever comes first, a mask of -1e9 too.
// Rounded up, so that values next to a large maximum stay out.
__device__ __forceinline__ float rows_floor(float max, float t) {
  return fmaxf(__double2float_ru((double)max - 745.13 * (double)t), -3.402823466e+38f);
}

// Set when a bounded wait gave up (read and cleared by take_sample_rows_status).
__device__ int g_rows_status;

// Unsigned key in the order of the values; -0 and +0 are one value, NaN
// counts as -infinity.
__device__ __forceinline__ uint32_t rows_key(float x) {
  uint32_t b = __float_as_uint(x);
  const uint32_t a = b & 0x7fffffffu;
  b = a > 0x7f800000u ? 0xff800000u : a == 0u ? 0u : b;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rows_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kKeyNone = 0x007fffffu;  // key of -infinity

struct RowsShared {
  // hist (counts, then the parts of the mass) and sort are never live at once:
  // a list is only sorted after a cluster barrier that follows the last read
  // of the histogram
  union {
    uint32_t hist[3][kRowsBuckets];
    alignas(16) unsigned long long sort[kRowsList];
  };
  unsigned long long list[2][kRowsList];
  uint32_t place[kRowsList];
  // this CTA's slice of the cluster's buckets: running sums before each
  unsigned long long slice_m[kRowsBuckets + 1];
  uint32_t slice_c[kRowsBuckets + 2];
  uint2 table[kRowsTable];  // 2^(29 + j/256), and it as a float
  unsigned long long redu[kRowsWarps];
  unsigned long long best;   // this CTA's maximum
  unsigned long long total;  // this CTA's mass (unfiltered and small top-k rows)
  unsigned long long ties;  // this CTA's count of one key
  uint32_t count[2];        // entries of the lists
  uint32_t result, last;
  int pick[4];
  unsigned long long pickm;
  uint64_t bar;
};

// Floats of a row that a CTA can hold beside its static shared memory (eight
// more: up to three of padding at either end, for the row's alignment).
constexpr size_t rows_cached_smem(uint32_t chunk) { return ((size_t)chunk + 8) * sizeof(float); }
constexpr uint32_t kRowsCached = (uint32_t)((kRowsSmem - sizeof(RowsShared)) / sizeof(float)) - 8;
static_assert(sizeof(RowsShared) % 16 == 0, "the row is 16-byte aligned behind it");
static_assert(sizeof(RowsShared) + rows_cached_smem(kRowsCached) <= kRowsSmem,
              "static and dynamic shared memory of the longest row that is held");

__device__ __forceinline__ RowsShared& rows_shared() {
  __shared__ RowsShared s;
  return s;
}

__device__ __forceinline__ unsigned long long rows_warp_scan(unsigned long long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Exclusive prefix over the block; the total in every thread.
__device__ __forceinline__ unsigned long long rows_scan(unsigned long long v,
                                                        unsigned long long* red,
                                                        unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long incl = rows_warp_scan(v);
  __syncthreads();
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  unsigned long long base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kRowsThreads / 32; ++w) {
    const unsigned long long x = red[w];
    if (w < warp) base += x;
    total += x;
  }
  return base + (incl - v);
}

constexpr uint32_t kRowsPad = 0xffffffffu;  // a NaN below every number: no token

template <bool CACHED>
struct Row {
  // this CTA's part of the row, four at a time: element i is token first + i,
  // ends padded with kRowsPad (cached: 16-byte aligned shared memory; else
  // `count` floats in global memory, first == base)
  const float* x;
  uint32_t first, n4;
  uint32_t base, count;  // its tokens
  uint32_t top;          // key of the maximum
  float fmax, per, low;  // buckets: (fmax - x) * per; what is below low weighs nothing
  float drawn;           // the least logit of an unfiltered draw, see rows_floor
  double scale, shift;   // 256 log2(w) = x * scale + shift, plus kMagic
  int bits, drop;        // see RowsParams
  static constexpr double kMagic = 402653184.0;  // 1.5 * 2^28: 24 fractional bits
  bool inf;              // the maximum is infinite: it counts as 0, all else as -infinity

  __device__ __forceinline__ float4 load(uint32_t j) const {
    if constexpr (CACHED) {
      extern __shared__ __align__(16) float s_row[];
      return reinterpret_cast<const float4*>(s_row)[j];
    } else {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = 4 * j + i < count ? at(4 * j + i) : __uint_as_float(kRowsPad);
      return make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  // Token base + i.
  __device__ __forceinline__ float at(uint32_t i) const {
    const float v = x[base - first + i];
    return CACHED || !inf ? v : v == INFINITY ? 0.0f : -INFINITY;
  }
  // Every element of this CTA, four at a time: f(values, first token). The
  // bodies keep to straight-line code, so that four elements' chains overlap.
  template <class F>
  __device__ __forceinline__ void each4(F f) const {
#pragma unroll 2
    for (uint32_t j = threadIdx.x; j < n4; j += kRowsThreads) {
      const float4 q = load(j);
      const float v[4] = {q.x, q.y, q.z, q.w};
      f(v, first + 4 * j);
    }
  }
  // Bucket of a value, in order (the nearest of (fmax - v) * per).
  __device__ __forceinline__ int bucket(float v) const {
    const float b = fminf((fmax - v) * per, (float)(kRowsBuckets - 1));
    return __float_as_int(b + 12582912.0f) - 0x4b400000;  // 1.5 * 2^23: rounds to an integer
  }
  // Exponent of the bucket's unit: at least that of any weight in it
  // (1/32 nat = 0.04508 octaves > 46 / 1024).
  __device__ static __forceinline__ int unit(int bucket) { return -((bucket * 46) >> 10); }
  // exp((v - max) / T) in units of 2^(unit(b) - 29 + drop), b = bucket(v).
  __device__ __forceinline__ uint32_t weight(float v, int b) const {
    const double m = fma((double)fmaxf(v, low), scale, shift);
    // a = 256 log2 w, times 2^24, below kMagic's bits
    const uint32_t lo = (uint32_t)__double2loint(m), hi = (uint32_t)__double2hiint(m);
    const int k = (int)__funnelshift_r(lo, hi, 24) - kMagicK;
    const float f = __uint_as_float(0x3f800000u | ((lo & 0xffffffu) >> 1)) - 1.0f;  // [0, 1)
    // 2^(f/256) - 1 = sum (f ln2/256)^i / i!
    float y = 3.3083026e-09f;        // (ln2/256)^3 / 6
    y = fmaf(y, f, 3.6655656e-06f);  // (ln2/256)^2 / 2
    y = fmaf(y, f, 2.7076062e-03f);  // ln2/256
    const uint2 t = rows_shared().table[k & (kRowsTable - 1)];
    const float up = fmaf(y * f, __uint_as_float(t.y), 12582912.0f);  // rounded to an integer
    const uint32_t w = t.x + (uint32_t)(__float_as_int(up) - 0x4b400000);  // [2^29, 2^30]
    return w >> min(unit(b) - (k >> 8) + drop, 31);
  }
  // kMagic's bits, shifted like those of m.
  static constexpr int kMagicK = (int)((0x41b8000000000000ull >> 24) & 0xffffffffull);
  // A sum of weights of bucket b in 64-bit units (2^-bits).
  __device__ __forceinline__ unsigned long long wide(unsigned long long w, int b) const {
    const int up = bits - 29 + drop + unit(b);  // -22 .. 22
    return up >= 0 ? w << up : w >> -up;
  }
  __device__ __forceinline__ unsigned long long value_weight(float v) const {
    const int b = bucket(v);
    return wide(weight(v, b), b);
  }
  __device__ __forceinline__ unsigned long long key_weight(uint32_t key) const {
    return key > kKeyNone ? value_weight(rows_value(key)) : 0ull;
  }
};

// The value of lane i < n of `get(i)` in every thread that asks for it: remote
// words read side by side instead of one after the other.
template <class T, class F>
__device__ __forceinline__ T rows_lane(int n, F get) {
  const int lane = threadIdx.x & 31;
  return lane < n ? get(lane) : T(0);
}

// Where the kept prefix ends, or the draw falls.
struct Targets {
  double k;        // tokens (infinity: none)
  double mass;     // running sum to reach, in fixed-point units (infinity: none)
  uint32_t least;  // smallest key kept (0: any)
};

// What the search has narrowed the border down to: keys [lo, hi] (of bucket b,
// where it is split); `count` tokens and `mass` lie above.
struct Range {
  int b;
  uint32_t lo, hi;
  uint32_t count;
  unsigned long long mass;
};

struct Found {
  int b;               // bucket (kRowsBuckets: no border in any)
  uint32_t cnt;        // tokens in it
  uint32_t above_c;    // tokens and mass above it
  unsigned long long above_m;
};

template <bool CACHED>
struct Search {
  const Row<CACHED> row;
  cg::cluster_group cl;
  const int ctas, part_bits;

  // Adds up the cluster's histogram: entry(value, bucket) gives a token's entry,
  // -1 for none; unit(i): the bucket of entry i's units. Afterwards
  // every CTA's slice holds running sums.
  template <class F, class U>
  __device__ __forceinline__ void histogram(bool mass, F entry, U unit) {
    RowsShared& sh = rows_shared();
    const int tid = threadIdx.x;
    for (int i = tid; i < (mass ? 3 : 1) * kRowsBuckets; i += kRowsThreads) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << part_bits) - 1;
    // the last entry (everything far below the maximum) is often crowded, and
    // adds to one word run one after the other: it is summed in registers
    uint32_t last_c = 0;
    unsigned long long last_m = 0;
    constexpr int kLast = kRowsBuckets - 1;
    if (mass) {
      row.each4([&](const float* v, uint32_t) {
        int at[4];
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = row.bucket(v[i]);
          w[i] = row.weight(v[i], b);
          at[i] = rows_real(v[i]) ? entry(v[i], b) : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          last_c += at[i] == kLast ? 1u : 0u;
          last_m += at[i] == kLast ? w[i] : 0u;
          if ((uint32_t)at[i] < (uint32_t)kLast) {
            atomicAdd(&sh.hist[0][at[i]], 1u);
            atomicAdd(&sh.hist[1][at[i]], w[i] & mask);
            atomicAdd(&sh.hist[2][at[i]], w[i] >> part_bits);
          }
        }
      });
    } else {
      row.each4([&](const float* v, uint32_t) {
        int at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = rows_real(v[i]) ? entry(v[i], row.bucket(v[i])) : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          last_c += at[i] == kLast ? 1u : 0u;
          if ((uint32_t)at[i] < (uint32_t)kLast) atomicAdd(&sh.hist[0][at[i]], 1u);
        }
      });
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      last_c += __shfl_xor_sync(0xffffffffu, last_c, o);
      last_m += __shfl_xor_sync(0xffffffffu, last_m, o);
    }
    if ((tid & 31) == 0 && last_c) {
      atomicAdd(&sh.hist[0][kLast], last_c);
      if (mass) {  // (the high part takes what its 32 bits hold of the chunk's sum)
        atomicAdd(&sh.hist[1][kLast], (uint32_t)last_m & mask);
        atomicAdd(&sh.hist[2][kLast], (uint32_t)(last_m >> part_bits));
      }
    }
    cl.sync();
    // this CTA's slice: thread i sums entries 2i, 2i + 1 of it over the cluster
    const int per = kRowsBuckets / ctas, rank = (int)cl.block_rank();
    uint32_t c[2] = {0, 0};
    unsigned long long m[2] = {0, 0};
    if (2 * tid < per) {
      const int b = rank * per + 2 * tid;
      unsigned long long m0 = 0, m1 = 0;
#pragma unroll
      for (int q = 0; q < kRowsMaxCtas; ++q)
        if (q < ctas) {
          const uint32_t* h = cl.map_shared_rank(&sh.hist[0][0], q) + b;
          const uint2 n = *reinterpret_cast<const uint2*>(h);
          c[0] += n.x;
          c[1] += n.y;
          if (mass) {
            const uint2 l = *reinterpret_cast<const uint2*>(h + kRowsBuckets);
            const uint2 u = *reinterpret_cast<const uint2*>(h + 2 * kRowsBuckets);
            m0 += l.x + ((unsigned long long)u.x << part_bits);
            m1 += l.y + ((unsigned long long)u.y << part_bits);
          }
        }
      m[0] = row.wide(m0, unit(b));
      m[1] = row.wide(m1, unit(b + 1));
    }
    unsigned long long tc, tm = 0;
    const uint32_t ec = (uint32_t)rows_scan((unsigned long long)c[0] + c[1], sh.redu, tc);
    const unsigned long long em = mass ? rows_scan(m[0] + m[1], sh.redu, tm) : 0ull;
    if (2 * tid < per) {
      sh.slice_c[2 * tid] = ec;
      sh.slice_c[2 * tid + 1] = ec + c[0];
      sh.slice_m[2 * tid] = em;
      sh.slice_m[2 * tid + 1] = em + m[0];
    }
    if (tid == 0) {
      sh.slice_c[per] = (uint32_t)tc;
      sh.slice_m[per] = tm;
    }
    cl.sync();
  }

  // The row's (or range's) whole mass and count, from the slices.
  __device__ __forceinline__ void totals(unsigned long long& count, unsigned long long& mass) const {
    RowsShared& sh = rows_shared();
    const int per = kRowsBuckets / ctas;
    unsigned long long c = rows_lane<unsigned long long>(
        ctas, [&](int q) { return (unsigned long long)cl.map_shared_rank(sh.slice_c, q)[per]; });
    unsigned long long m = rows_lane<unsigned long long>(
        ctas, [&](int q) { return cl.map_shared_rank(sh.slice_m, q)[per]; });
#pragma unroll
    for (int o = 1; o < kRowsMaxCtas; o <<= 1) {
      c += __shfl_xor_sync(0xffffffffu, c, o);
      m += __shfl_xor_sync(0xffffffffu, m, o);
    }
    count = __shfl_sync(0xffffffffu, c, 0);
    mass = __shfl_sync(0xffffffffu, m, 0);
  }

  // The first bucket with tokens where a border is reached, or `most` if that
  // is not further; `c0`, `m0`: what lies above the histogram's range.
  // meets(bucket): a border by key.
  template <class F>
  __device__ __forceinline__ Found find(const Targets& want, uint32_t c0, unsigned long long m0, bool mass, int most,
                        F meets) {
    RowsShared& sh = rows_shared();
    const int per = kRowsBuckets / ctas, tid = threadIdx.x, lane = tid & 31;
    // running sums of the slices, one per lane
    uint32_t sc = rows_lane<uint32_t>(ctas, [&](int q) { return cl.map_shared_rank(sh.slice_c, q)[per]; });
    unsigned long long sm = rows_lane<unsigned long long>(
        ctas, [&](int q) { return cl.map_shared_rank(sh.slice_m, q)[per]; });
    uint32_t ic = sc;
    unsigned long long im = sm;
#pragma unroll
    for (int o = 1; o < kRowsMaxCtas; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, ic, o);
      const unsigned long long y = __shfl_up_sync(0xffffffffu, im, o);
      if (lane >= o) {
        ic += x;
        im += y;
      }
    }
    __syncthreads();
    if (tid == 0) sh.pick[0] = most;
    __syncthreads();
    // thread i looks at buckets 2i and 2i + 1, in one CTA's slice
    const int q = 2 * tid / per, i = 2 * tid - q * per;
    uint32_t base_c = 0;
    unsigned long long base_m = 0;
#pragma unroll
    for (int x = 0; x < kRowsMaxCtas; ++x) {
      const uint32_t a = __shfl_sync(0xffffffffu, ic - sc, x);
      const unsigned long long b = __shfl_sync(0xffffffffu, im - sm, x);
      if (x == q) {
        base_c = a;
        base_m = b;
      }
    }
    const uint32_t* pc = cl.map_shared_rank(sh.slice_c, q) + i;
    const unsigned long long* pm = cl.map_shared_rank(sh.slice_m, q) + i;
    const uint32_t ac[3] = {base_c + pc[0], base_c + pc[1], base_c + pc[2]};
    unsigned long long am[3] = {0, 0, 0};
    if (mass)
#pragma unroll
      for (int x = 0; x < 3; ++x) am[x] = base_m + pm[x];
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (ac[x + 1] > ac[x] && ((double)(c0 + ac[x + 1]) >= want.k ||
                                (mass && (double)(m0 + am[x + 1]) >= want.mass) || meets(2 * tid + x)))
        atomicMin(&sh.pick[0], 2 * tid + x);
    __syncthreads();
    Found f;
    f.b = sh.pick[0];
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (2 * tid + x == min(f.b, kRowsBuckets - 1)) {
        sh.pick[1] = (int)(ac[x + 1] - ac[x]);
        sh.pick[2] = (int)(c0 + ac[x]);
        sh.pickm = m0 + am[x];
      }
    __syncthreads();
    f.cnt = (uint32_t)sh.pick[1];
    f.above_c = (uint32_t)sh.pick[2];
    f.above_m = sh.pickm;
    return f;
  }

  // Smallest key above -infinity whose bucket is at most b (row.top's is 0): a
  // search with one key per lane.
  __device__ __forceinline__ uint32_t key_of(int b) const {
    const int lane = threadIdx.x & 31;
    uint32_t lo = kKeyNone, hi = row.top;  // bucket(lo) > b >= bucket(hi)
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo - 1) / 32 + 1;
      const uint32_t probe = min(lo + step * (lane + 1), hi);
      const uint32_t at =
          __ffs(__ballot_sync(0xffffffffu, probe == hi || row.bucket(rows_value(probe)) <= b)) - 1;
      hi = min(lo + step * (at + 1), hi);
      lo = lo + step * at;
    }
    return hi;
  }

  // Splits a range of keys and narrows it to the first part where a border is
  // reached (else the last with any token); returns the tokens in it.
  __device__ __forceinline__ uint32_t split(Range& g, const Targets& want) {
    RowsShared& sh = rows_shared();
    int shift = 0;
    while (((g.hi - g.lo) >> shift) >= (uint32_t)kRowsBuckets) ++shift;
    const uint32_t width = (1u << shift) - 1;
    cl.sync();  // the others have read the last slices
    const uint32_t lo = g.lo, hi = g.hi;
    const int inside = g.b;  // every key of the range is in this bucket
    histogram(
        true,
        [&](float v, int) {
          const uint32_t key = rows_key(v);
          return key >= lo && key <= hi ? (int)((hi - key) >> shift) : -1;
        },
        [&](int) { return inside; });
    // without a border: the last part with any token
    Targets all{INFINITY, INFINITY, 0};
    unsigned long long c, m;
    totals(c, m);
    all.k = (double)c;
    const int last = find(all, 0, 0, false, kRowsBuckets - 1, [](int) { return false; }).b;
    const Found f = find(want, g.count, g.mass, true, last, [&](int b) {
      return want.least && hi - ((uint32_t)b << shift) - width <= want.least;
    });
    g.count = f.above_c;
    g.mass = f.above_m;
    const uint32_t first_key = hi - ((uint32_t)f.b << shift);
    if (first_key - lo > width) g.lo = first_key - width;
    g.hi = first_key;
    return f.cnt;
  }

  // The cluster's tokens with keys in [lo, hi] (at most kRowsList), sorted in rank
  // order into sh.list[which ^ 1]; returns their number. `which`: the list to use.
  __device__ __forceinline__ uint32_t gather(const Range& g, int which) {
    RowsShared& sh = rows_shared();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sh.count[which] = 0;
    __syncthreads();
    const float lo = rows_value(g.lo), hi = rows_value(g.hi);
    row.each4([&](const float* v, uint32_t token) {
      uint32_t in = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) in |= (uint32_t)(v[i] >= lo && v[i] <= hi) << i;
      if (in) {
        uint32_t at = atomicAdd(&sh.count[which], (uint32_t)__popc(in));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((in >> i) & 1) {
            if (at < (uint32_t)kRowsList)
              sh.list[which][at] =
                  ((unsigned long long)rows_key(v[i]) << 32) | (uint32_t)~(token + i);
            ++at;
          }
      }
    });
    cl.sync();
    const uint32_t k = rows_lane<uint32_t>(ctas, [&](int q) {
      return min(*cl.map_shared_rank(&sh.count[which], q), (uint32_t)kRowsList);
    });
    uint32_t incl = k;
#pragma unroll
    for (int o = 1; o < kRowsMaxCtas; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const uint32_t m = min(__shfl_sync(0xffffffffu, incl, kRowsMaxCtas - 1), (uint32_t)kRowsList);
    // a warp copies each CTA's list
    static_assert(kRowsWarps == kRowsMaxCtas, "one warp per CTA");
    {
      const uint32_t n = __shfl_sync(0xffffffffu, k, warp);
      const uint32_t base = __shfl_sync(0xffffffffu, incl, warp) - n;
      if (warp < ctas) {
        const unsigned long long* src = cl.map_shared_rank(&sh.list[which][0], warp);
        for (uint32_t i = lane; i < n; i += 32)
          if (base + i < (uint32_t)kRowsList) sh.sort[base + i] = src[i];
      }
    }
    if (tid == 0 && (m & 1)) sh.sort[m] = 0ull;
    __syncthreads();
    // an entry's place is the number of larger ones (they all differ); a long
    // list's entries are dealt out over the cluster
    unsigned long long* sorted = sh.list[which ^ 1];
    const bool dealt = ctas > 1 && m > (uint32_t)kRowsThreads;
    const uint32_t share = dealt ? (m + ctas - 1) / ctas : m;
    const uint32_t e0 = dealt ? min(m, share * cl.block_rank()) : 0u, e1 = min(m, e0 + share);
    for (uint32_t e = tid; e < e1 - e0; e += kRowsThreads) sh.place[e] = 0;
    __syncthreads();
    // each warp compares with its part of the list, four entries per lane at a time
    const uint32_t part = ((m + kRowsWarps - 1) / kRowsWarps + 1) & ~1u;
    const uint32_t j0 = min(m, part * warp), j1 = min(m, j0 + part);
    for (uint32_t e = e0; e < e1; e += 128) {
      unsigned long long x[4];
      uint32_t place[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = e + 32 * i + lane < e1 ? sh.sort[e + 32 * i + lane] : ~0ull;
#pragma unroll 2
      for (uint32_t j = j0; j < j1; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.sort[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) place[i] += (o.x > x[i] ? 1u : 0u) + (o.y > x[i] ? 1u : 0u);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (place[i]) atomicAdd(&sh.place[e - e0 + 32 * i + lane], place[i]);
    }
    __syncthreads();
    for (uint32_t e = tid; e < e1 - e0; e += kRowsThreads) {
      const unsigned long long x = sh.sort[e0 + e];
      const uint32_t place = sh.place[e];
      if (dealt) {
        for (int q = 0; q < ctas; ++q) cl.map_shared_rank(sorted, q)[place] = x;
      } else {
        sorted[place] = x;
      }
    }
    if (dealt)
      cl.sync();
    else
      __syncthreads();
    return m;
  }

  // Token of the t-th (1-based) element in index order with this key; in the
  // CTA that holds it.
  __device__ __forceinline__ uint32_t nth_tie(uint32_t key, unsigned long long t) {
    RowsShared& sh = rows_shared();
    const int tid = threadIdx.x;
    if (tid == 0) sh.result = 0xffffffffu;
    const uint32_t per = (row.count + kRowsThreads - 1) / kRowsThreads;
    const uint32_t lo = min(row.count, tid * per), hi = min(row.count, lo + per);
    unsigned long long mine = 0;
    for (uint32_t i = lo; i < hi; ++i) mine += rows_key(row.at(i)) == key;
    unsigned long long total;
    unsigned long long before = rows_scan(mine, sh.redu, total);
    if (tid == 0) sh.ties = total;
    cl.sync();
    const int rank = (int)cl.block_rank();
    for (int c = 0; c < rank; ++c) before += *cl.map_shared_rank(&sh.ties, c);
    if (before < t && t <= before + mine)
      for (uint32_t i = lo; i < hi; ++i)
        if (rows_key(row.at(i)) == key && ++before == t) {
          sh.result = row.base + i;
          break;
        }
    __syncthreads();
    return sh.result;
  }

  // The draw of a filtered row; the token in the CTA that writes it.
  __device__ __forceinline__ uint32_t filtered(const Targets& borders, double top_p, double u) {
    RowsShared& sh = rows_shared();
    const int tid = threadIdx.x, rank = (int)cl.block_rank();
    const bool by_p = top_p < 1.0;
    Targets kept = borders;
    // a mass histogram unless top-k alone makes the kept tokens fit a list;
    // then top-p needs the row's whole mass only
    bool mass = by_p && kept.k > (double)kRowsList / 2;
    if (by_p && !mass) {
      unsigned long long mine = 0, total;
      row.each4([&](const float* v, uint32_t) {
        unsigned long long w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = row.value_weight(v[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += rows_real(v[i]) ? w[i] : 0ull;
      });
      rows_scan(mine, sh.redu, total);
      if (tid == 0) sh.total = total;  // read after the histogram's barrier
    }
    const auto whole = [](float, int b) { return b; };
    const auto itself = [](int b) { return b; };
    const auto never = [](int) { return false; };
    unsigned long long z = 0;  // the row's mass (by_p or mass)
    Found end;       // bucket of the last kept token; kRowsBuckets: every token is kept
    for (;;) {
      histogram(mass, whole, itself);
      unsigned long long tc, tm;
      totals(tc, tm);
      if (mass) {
        z = tm;
      } else if (by_p) {
        const unsigned long long x = rows_lane<unsigned long long>(
            ctas, [&](int q) { return *cl.map_shared_rank(&sh.total, q); });
        z = 0;
#pragma unroll
        for (int q = 0; q < kRowsMaxCtas; ++q) z += __shfl_sync(0xffffffffu, x, q);
      }
      if (by_p) kept.mass = top_p * (double)z;
      // (without a mass histogram the border by mass is found in the list)
      const int most = kept.least ? row.bucket(rows_value(kept.least)) : kRowsBuckets;
      end = find(kept, 0, 0, mass, most, never);
      const uint32_t n = end.b < kRowsBuckets ? end.above_c + end.cnt : (uint32_t)tc;
      if (n <= (uint32_t)kRowsList) {
        end.cnt = n;
        break;
      }
      if (mass) {
        end.cnt = n;
        break;
      }
      mass = true;  // too many for one list: their mass has to be known by bucket
      cl.sync();    // the others have read these slices
    }
    const bool one_list = end.cnt <= (uint32_t)kRowsList;
    unsigned long long kept_mass = z;
    uint32_t end_key = kKeyNone + 1;  // no key below it is kept
    double end_ties = INFINITY;       // and of it so many
    bool fresh = true;                // the slices are those of the whole row
    // phase 0: where the kept tokens end; phase 1: where the draw falls, if
    // not among the tokens that phase 0 listed
    for (int phase = 0; phase < 2; ++phase) {
      Targets want = kept;
      Range g{0, kKeyNone + 1, row.top, 0, 0};
      uint32_t members = end.cnt;
      if (one_list) {
        g.lo = key_of(min(end.b, kRowsBuckets - 1));
      } else {
        Found f = end;
        if (phase == 0) {
          if (end.b >= kRowsBuckets) continue;  // everything is kept
          f.cnt = end.cnt - end.above_c;
        } else {
          want = Targets{INFINITY, u * (double)kept_mass, 0};
          if (!fresh) {
            cl.sync();
            histogram(true, whole, itself);
          }
          f = find(want, 0, 0, true, min(end.b, kRowsBuckets - 1), never);
        }
        g.b = f.b;
        g.lo = key_of(f.b);
        g.hi = f.b > 0 ? key_of(f.b - 1) - 1 : row.top;
        g.count = f.above_c;
        g.mass = f.above_m;
        members = f.cnt;
        // a crowded bucket is split by the key's bits until it fits, or is one key
        while (members > (uint32_t)kRowsList && g.lo < g.hi) {
          members = split(g, want);
          fresh = false;
        }
      }
      // --- settle the border among the listed tokens (or equal keys)
      if (members > (uint32_t)kRowsList) {  // `members` equal logits
        const unsigned long long w = row.key_weight(g.lo);
        double n = want.k - (double)g.count;
        if (w) n = fmin(n, ceil((want.mass - (double)g.mass) / (double)w));
        n = fmax(1.0, fmin(n, (double)members));
        if (phase == 1) {
          if (g.lo == end_key) n = fmin(n, end_ties);
          return nth_tie(g.lo, (unsigned long long)n);
        }
        if (want.least > g.lo) n = 0.0;  // min-p ends above them
        end_key = n > 0.0 ? g.lo : g.lo + 1;
        end_ties = n > 0.0 ? n : INFINITY;
        kept_mass = g.mass + (unsigned long long)n * w;
        continue;
      }
      const uint32_t m = gather(g, phase);
      const unsigned long long* sorted = sh.list[phase ^ 1];
      constexpr int kOwn = kRowsList / kRowsThreads;  // consecutive entries of a thread
      const int at = kOwn * tid;
      uint32_t key[kOwn];
      unsigned long long run[kOwn], mine = 0, tw;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        key[i] = at + i < (int)m ? (uint32_t)(sorted[at + i] >> 32) : 0u;
        if (at + i < (int)m) mine += row.key_weight(key[i]);
        run[i] = mine;
      }
      const unsigned long long before = g.mass + rows_scan(mine, sh.redu, tw);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) run[i] += before;
      // entries that a border allows, and the first that reaches one
      if (tid == 0) sh.pick[0] = (int)m - 1, sh.pick[1] = 0;
      __syncthreads();
      const uint32_t floor_key = phase == 0 ? want.least : end_key;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (at + i < (int)m) {
          if ((double)(g.count + at + i + 1) >= want.k || (double)run[i] >= want.mass)
            atomicMin(&sh.pick[0], at + i);
          if (key[i] >= floor_key) atomicMax(&sh.pick[1], at + i + 1);
        }
      __syncthreads();
      int e = min(sh.pick[0], sh.pick[1] - 1);  // the last kept entry, or the draw; -1: above all
      if (phase == 0) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (at + i == e) sh.pickm = run[i];
        __syncthreads();
        kept_mass = e >= 0 ? sh.pickm : g.mass;
        if (!one_list && !(u * (double)kept_mass > (double)g.mass)) {
          // above this list: no key of it may be drawn
          end_key = g.hi + 1;
          continue;
        }
        // the draw is among these, too
        const double target = u * (double)kept_mass;
        if (tid == 0) sh.pick[0] = e;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (at + i < e && (double)run[i] >= target) atomicMin(&sh.pick[0], at + i);
        __syncthreads();
        e = sh.pick[0];
      }
      return rank == 0 ? ~(uint32_t)sorted[max(0, e)] : 0xffffffffu;
    }
    return 0xffffffffu;  // not reached: phase 1 returns
  }

  // The draw of an unfiltered row, by the running sum in index order; the
  // token in the CTA that holds it.
  __device__ __forceinline__ uint32_t unfiltered(double u) {
    RowsShared& sh = rows_shared();
    const int tid = threadIdx.x, rank = (int)cl.block_rank();
    if (tid == 0) sh.result = 0xffffffffu, sh.last = 0;
    const uint32_t per = (row.count + kRowsThreads - 1) / kRowsThreads | 1u;  // odd: no bank twice
    const uint32_t lo = min(row.count, tid * per), hi = min(row.count, lo + per);
    unsigned long long mine = 0;
    uint32_t last = 0xffffffffu;
    for (uint32_t i = lo; i < hi; ++i) {
      const float v = row.at(i);
      if (!(v >= row.drawn)) continue;
      mine += row.value_weight(v);
      last = i;
    }
    unsigned long long total;
    const unsigned long long before = rows_scan(mine, sh.redu, total);
    if (tid == 0) sh.total = total;
    // the last CTA with a token takes what no sum reaches (u = 1)
    if (last != 0xffffffffu) atomicMax(&sh.last, last + 1);
    cl.sync();
    const unsigned long long xs = rows_lane<unsigned long long>(
        ctas, [&](int q) { return *cl.map_shared_rank(&sh.total, q); });
    const uint32_t any = rows_lane<uint32_t>(
        ctas, [&](int q) { return *cl.map_shared_rank(&sh.last, q); });
    unsigned long long z = 0, base = 0, run = 0;
    int holder = 0;
    bool reached = false;
#pragma unroll
    for (int q = 0; q < kRowsMaxCtas; ++q) z += __shfl_sync(0xffffffffu, xs, q);
    const double target = u * (double)z;
#pragma unroll
    for (int q = 0; q < kRowsMaxCtas; ++q) {
      const unsigned long long v = __shfl_sync(0xffffffffu, xs, q);
      if (__shfl_sync(0xffffffffu, any, q) && !reached) {
        holder = q;
        base = run;
        reached = (double)(run + v) >= target;
      }
      run += v;
    }
    if (holder != rank) return 0xffffffffu;
    // the first chunk that reaches the draw holds the token
    if (last != 0xffffffffu && (double)(base + before + mine) >= target) {
      unsigned long long r = base + before;
      uint32_t hit = last;
      for (uint32_t i = lo; i < hi; ++i) {
        const float v = row.at(i);
        if (!(v >= row.drawn)) continue;
        r += row.value_weight(v);
        if ((double)r >= target) {
          hit = i;
          break;
        }
      }
      atomicMin(&sh.result, hit);
    }
    __syncthreads();
    return row.base + (sh.result != 0xffffffffu ? sh.result : sh.last - 1);
  }
};

template <bool CACHED>
__global__ void __launch_bounds__(kRowsThreads, 2)
    sample_rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(16) float s_row[];
  RowsShared& sh = rows_shared();
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t r = blockIdx.x / ctas;
  Row<CACHED> row;
  row.base = min(p.n, p.chunk * (uint32_t)rank);
  row.count = min(p.n, row.base + p.chunk) - row.base;
  const float* src = p.logits + r * p.stride + row.base;
  row.x = src;
  row.first = row.base;
  row.n4 = (row.count + 3) / 4;
  row.inf = false;
  if (tid == 0) mbar_init(&sh.bar, 1);
  mbar_fence_init();
  for (int i = tid; i < kRowsTable; i += kRowsThreads) {
    const double x = exp2(29.0 + (double)i / kRowsTable);
    sh.table[i] = make_uint2((uint32_t)(x + 0.5), __float_as_uint((float)x));
  }
  __syncthreads();
  pdl_wait();
  bool got = true;  // the row has come
  if (CACHED) {
    // the 16-byte aligned middle by bulk copies, the ragged ends by loads; the
    // copy keeps the row's misalignment, the ends are padded
    const uint32_t mis = (uint32_t)((reinterpret_cast<uintptr_t>(src) >> 2) & 3);
    float* dst = s_row + mis;
    const uint32_t head = min(row.count, (4 - mis) & 3), body = (row.count - head) / 4 * 4;
    if (tid == 0 && body) {
      mbar_arrive_expect_tx(&sh.bar, body * 4 + p.stall);
      for (uint32_t o = 0; o < body; o += 4096)
        bulk_g2s(dst + head + o, src + head + o, min(4096u, body - o) * 4, &sh.bar);
    }
    const uint32_t tail = head + body, end = mis + row.count;
    if ((uint32_t)tid < mis) s_row[tid] = __uint_as_float(kRowsPad);
    if ((uint32_t)tid < head) dst[tid] = src[tid];
    if (tid < 4 && tail + tid < row.count) dst[tail + tid] = src[tail + tid];
    if (tid < 4 && end + tid < (end + 3) / 4 * 4) s_row[end + tid] = __uint_as_float(kRowsPad);
    if (body) {
      got = mbar_wait_timed(&sh.bar, 0, &g_rows_status);
      if (!got) mbar_wait_timed(&sh.bar, 0, &g_rows_status);  // the copies still in flight
    }
    got = __syncthreads_and(got) != 0;
    row.x = s_row;
    row.first = row.base - mis;
    row.n4 = (end + 3) / 4;
  }
  const float t = p.temperature ? p.temperature[r] : 1.0f;
  const int k = p.top_k ? p.top_k[r] : 0;
  const double top_p = p.top_p ? (double)p.top_p[r] : 1.0;
  const double min_p = p.min_p ? (double)p.min_p[r] : 0.0;
  const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
  const bool greedy = !(t > 0.0f) || k == 1;

  // --- the maximum; greedy: with its lowest index, in the total order of
  // minq_argmax (the padding comes last in it)
  unsigned long long best = 0;
  if (greedy) {
    row.each4([&](const float* v, uint32_t token) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned long long x = argmax_pack(v[i], token + i);
        best = x > best ? x : best;
      }
    });
  } else {
    float top = -INFINITY;
    row.each4([&](const float* v, uint32_t) {  // NaN gives way
      top = fmaxf(top, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    });
    best = (unsigned long long)rows_key(top) << 32;
  }
  best = warp_max_u64(best);
  if (lane == 0) sh.redu[warp] = best;
  __syncthreads();
  best = warp_max_u64(lane < kRowsWarps ? sh.redu[lane] : 0ull);
  // a row that did not come in one CTA is none in all: the highest key stands for
  // it (with index 0; a greedy row's NaN of that key and index gives token 0 anyway)
  if (tid == 0) sh.best = got ? best : ~0ull;
  cl.sync();
  best = warp_max_u64(rows_lane<unsigned long long>(
      ctas, [&](int q) { return *cl.map_shared_rank(&sh.best, q); }));
  row.top = (uint32_t)(best >> 32);
  uint32_t token = 0xffffffffu;  // set in the CTA that writes it
  if (greedy || best == ~0ull) {
    if (rank == 0) token = ~(uint32_t)best;
  } else if (row.top <= kKeyNone) {
    if (rank == 0) token = 0;  // nothing to draw from
  } else {
    if (rows_value(row.top) == INFINITY) {
      // only infinite logits are drawn, evenly: they become 0, the others -infinity
      row.inf = true;
      row.top = rows_key(0.0f);
      if (CACHED) {
        for (uint32_t i = tid; i < 4 * row.n4; i += kRowsThreads)
          s_row[i] = s_row[i] == INFINITY ? 0.0f : -INFINITY;
        __syncthreads();
      }
    }
    row.fmax = rows_value(row.top);
    // below |max| 1e-12 every other logit's weight is 0 already
    const float tt = fmaxf(t, fmaxf(1e-30f, fabsf(row.fmax) * 1e-12f));
    row.per = kRowsPerNat / tt;
    row.low = row.fmax - 64.0f * tt;
    row.drawn = rows_floor(row.fmax, tt);
    row.bits = p.mass_bits;
    row.drop = p.drop;
    row.scale = (kRowsTable * 1.4426950408889634074) / (double)tt;
    // one rounding for the whole row: a common factor next to 1 on all weights
    row.shift = Row<CACHED>::kMagic - (double)row.fmax * row.scale;
    Search<CACHED> s{row, cl, ctas, p.part_bits};
    const bool by_k = k > 0 && (uint32_t)k < p.n;
    if (!by_k && !(top_p < 1.0) && !(min_p > 0.0)) {
      token = s.unfiltered(u);
    } else {
      Targets kept{by_k ? (double)k : INFINITY, INFINITY, 0};
      if (min_p > 1.0) {
        kept.k = 1.0;  // no token reaches it: the first
      } else if (min_p > 0.0) {
        // smallest key with w >= min_p (w grows with the key): a search with one
        // key per lane, at most seven rounds
        const double bar = log(min_p) * (double)tt;
        uint32_t lo = kKeyNone, hi = row.top;  // w(lo) < min_p <= w(hi)
        if (tt == INFINITY) hi = lo + 1;       // every weight is 1
        while (hi - lo > 1) {
          const uint32_t step = (hi - lo - 1) / 32 + 1;
          const uint32_t probe = min(lo + step * (lane + 1), hi);
          const uint32_t yes = __ballot_sync(
              0xffffffffu, probe == hi || (double)rows_value(probe) - (double)row.fmax >= bar);
          const uint32_t at = __ffs(yes) - 1;
          hi = min(lo + step * (at + 1), hi);
          lo = lo + step * at;
        }
        kept.least = hi;
      }
      token = s.filtered(kept, top_p, u);
    }
  }
  if (tid == 0 && token != 0xffffffffu) p.out[r] = token;
  pdl_launch_dependents();
  cl.sync();  // the others may still read this CTA's shared memory
}

}  // namespace

minq_status take_sample_rows_status() {
  int v = 0;
  MINQ_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_rows_status, sizeof(int)));
  if (v == 0) return MINQ_OK;
  const int zero = 0;
  MINQ_CUDA_TRY(cudaMemcpyToSymbol(g_rows_status, &zero, sizeof(int)));
  return fail(MINQ_ERR_TIMEOUT, "a bounded wait of sample_rows timed out");
}

}  // namespace minq

using namespace minq;

extern "C" {

minq_status minq_sample_rows(const float* logits, size_t row_stride, size_t n_rows, size_t n,
                             const float* temperature, const int32_t* top_k, const float* top_p,
                             const float* min_p, const float* uniforms, uint32_t* tokens,
                             void* stream) {
  if (n_rows > (1u << 20)) return fail(MINQ_ERR_SHAPE, "sample_rows: at most 2^20 rows");
  if (n == 0 || n > (1u << 22))
    return fail(MINQ_ERR_SHAPE, "sample_rows: rows of 1 to 4194304 logits, got " +
                                    std::to_string(n));
  if (n_rows > 1 && row_stride < n)
    return fail(MINQ_ERR_ARG, "sample_rows: row stride smaller than the row");
  if (n_rows == 0) return MINQ_OK;
  if (!logits || !uniforms || !tokens) return fail(MINQ_ERR_ARG, "null pointer");
  MINQ_TRY(require_device());
  RowsParams p{};
  p.logits = logits;
  p.stride = row_stride;
  p.n = (uint32_t)n;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.u = uniforms;
  p.out = tokens;
  // as many CTAs as let two of them share an SM with their parts of the rows,
  // and more for few rows
  int ctas = 1;
  while (ctas < kRowsMaxCtas &&
         (n > 19456u * ctas || (n_rows * ctas < (size_t)sm_count() && n > 4096u * ctas)))
    ctas *= 2;
  p.chunk = (uint32_t)((n + ctas - 1) / ctas);
  p.cached = p.chunk <= kRowsCached;
  int chunk_bits = 0, n_bits = 0;
  while ((1u << chunk_bits) < p.chunk) ++chunk_bits;
  while ((1u << n_bits) < p.n) ++n_bits;
  // sums of a chunk's parts fit 32 bits, those of the row 63
  p.part_bits = 32 - chunk_bits < 15 ? 32 - chunk_bits : 15;
  p.drop = 30 - 2 * p.part_bits;
  p.mass_bits = 62 - n_bits < 47 ? 62 - n_bits : 47;
  p.stall = take_stall(kStallSampleRows);
  const size_t smem = p.cached ? rows_cached_smem(p.chunk) : 0;
  auto kernel = p.cached ? sample_rows_kernel<true> : sample_rows_kernel<false>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  MINQ_TRY(ensure_dynamic_smem(fn, smem));
  prefer_max_shared(fn);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_rows * ctas));
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  MINQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return MINQ_OK;
}

}  // extern "C"
