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
// are never drawn; a row without any other token gives token 0.
//
// Weights and sums carry about f64: next to a border a draw is decided by
// digits that an f32 sum over a vocabulary does not hold (with 100,000 even
// tokens, borders moved by 1e-7 of the mass would change one draw in a
// hundred). The exponential is the table-driven one (Tang 1989): 2^(m/256) from
// a table times a polynomial of degree 3 on half a step, to 1e-13.
//
// A cluster of up to 8 CTAs holds a row in shared memory (one pass over HBM,
// bulk copies), so every further pass runs at shared-memory speed:
//   1. the maximum;
//   2. a histogram over 512 buckets of (max - x) / T, 1/32 wide: counts, and
//      the mass as fixed-point integers in three 32-bit parts (shared-memory
//      atomics are fast in 32 bits only; integer sums do not depend on their
//      order). Each CTA adds up a slice of the buckets over the cluster; the
//      running sums give the bucket of the last kept token (by count and by
//      mass alike) and, for a given mass, that of the draw;
//   3. the tokens of that bucket are listed, sorted and summed in f64, which
//      settles the border exactly. A crowded bucket is split again by the key's
//      bits; equal logits beyond the list's room are counted in index order.
// When the kept tokens fit the list as a whole, one list serves both borders
// and no mass histogram is needed. Every CTA of the cluster reads the others'
// sums and lists over distributed shared memory and decides alike, so there
// is no result to send round.
#include <cooperative_groups.h>
#include <math.h>

#include <string>

#include "common.cuh"
#include "kernels.h"
#include "pipeline.cuh"

namespace minq {

namespace {

namespace cg = cooperative_groups;

constexpr int kRowsThreads = 512;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsBuckets = 512;           // one per thread
constexpr float kRowsPerNat = 32.0f;        // buckets per unit of (max - x) / T
constexpr int kRowsList = 1024;             // tokens a list holds
constexpr int kRowsMaxCtas = 8;             // the portable cluster size
constexpr uint32_t kRowsCached = 48 * 1024; // floats of a row that a CTA can hold
constexpr int kRowsTable = 256;

struct RowsParams {
  const float* logits;
  size_t stride;
  uint32_t n, chunk;         // chunk: elements per CTA
  bool cached;
  int part_bits, mass_bits;  // the fixed-point mass: bits per part, of w = 1
  const float* temperature;  // null: 1
  const int* top_k;          // null or <= 0: off
  const float* top_p;        // null or >= 1: off
  const float* min_p;        // null or <= 0: off
  const float* u;
  uint32_t* out;
};

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
    uint32_t hist[4][kRowsBuckets];
    unsigned long long sort[kRowsList];
  };
  unsigned long long list[2][kRowsList];
  // this CTA's slice of the cluster's buckets: running sums before each
  unsigned long long slice_m[kRowsBuckets + 1];
  uint32_t slice_c[kRowsBuckets + 2];
  double table[kRowsTable];  // 2^(j/256)
  double red[kRowsWarps];
  unsigned long long redu[kRowsWarps];
  unsigned long long best;  // this CTA's maximum
  double total;             // this CTA's mass (unfiltered and small top-k rows)
  unsigned long long ties;  // this CTA's count of one key
  uint32_t count[2];        // entries of the lists
  uint32_t result, last;
  int pick[4];
  unsigned long long pickm;
  double pickd;
  uint64_t bar;
};

__device__ __forceinline__ unsigned long long rows_warp_scan(unsigned long long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
__device__ __forceinline__ double rows_warp_scan(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Exclusive prefix over the block; the total in every thread.
template <class T>
__device__ __forceinline__ T rows_scan(T v, T* red, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T incl = rows_warp_scan(v);
  __syncthreads();
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  T base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kRowsThreads / 32; ++w) {
    const T x = red[w];
    if (w < warp) base += x;
    total += x;
  }
  return base + (incl - v);
}

constexpr uint32_t kRowsPad = 0xffffffffu;  // a NaN below every number: no token

struct Row {
  // this CTA's part of the row, four at a time: element i is token first + i,
  // ends padded with kRowsPad (cached: 16-byte aligned shared memory; else
  // `count` floats in global memory, first == base)
  const float* x;
  bool cached;
  uint32_t first, n4;
  uint32_t base, count;  // its tokens
  uint32_t top;          // key of the maximum
  float fmax, per;       // buckets: (fmax - x) * per
  double dmax, scale;    // 256 log2(w) = (x - dmax) * scale
  const double* table;

  __device__ __forceinline__ float4 load(uint32_t j) const {
    if (cached) return reinterpret_cast<const float4*>(x)[j];
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = 4 * j + i < count ? x[4 * j + i] : __uint_as_float(kRowsPad);
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  // Every element of this CTA: f(value, token).
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
    for (uint32_t j = threadIdx.x; j < n4; j += kRowsThreads) {
      const float4 v = load(j);
      f(v.x, first + 4 * j);
      f(v.y, first + 4 * j + 1);
      f(v.z, first + 4 * j + 2);
      f(v.w, first + 4 * j + 3);
    }
  }
  // Whether a weight can be drawn (a number above -infinity).
  __device__ static __forceinline__ bool real(float v) { return v > -INFINITY; }
  // 2^bits exp((v - max) / T); 0 where it is below 2^(bits - 860), or the
  // maximum is infinite and v is not.
  __device__ __forceinline__ double weight(float v, int bits = 0) const {
    const double kMagic = 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    if (fmax == INFINITY) return v == INFINITY ? ldexp(1.0, bits) : 0.0;
    if (!((fmax - v) * per < kRowsPerNat * 600.0f)) return 0.0;
    const double a = ((double)v - dmax) * scale;
    const double m = a + kMagic;
    const int k = __double2loint(m);
    const double f = a - (m - kMagic);         // [-1/2, 1/2] of 1/256 octave
    // 2^(f/256) = sum (f ln2/256)^i / i!
    double y = 3.308302680541371e-09;          // (ln2/256)^3 / 6
    y = fma(y, f, 3.665565596910106e-06);      // (ln2/256)^2 / 2
    y = fma(y, f, 0.0027076061740622863);      // ln2/256
    y = fma(y, f, 1.0);
    y *= table[k & (kRowsTable - 1)];
    return __hiloint2double(__double2hiint(y) + (((k >> 8) + bits) << 20), __double2loint(y));
  }
  __device__ __forceinline__ double key_weight(uint32_t key) const {
    return key > kKeyNone ? weight(rows_value(key)) : 0.0;
  }
  __device__ __forceinline__ int bucket(float v) const {
    const float b = (fmax - v) * per;  // NaN (both infinite): 0
    return b >= (float)(kRowsBuckets - 1) ? kRowsBuckets - 1 : (int)b;
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
  double mass;     // running sum to reach (infinity: none)
  uint32_t least;  // smallest key kept (0: any)
};

// What the search has narrowed the border down to: buckets [b0, b1] of the
// row, or (keyed) keys [lo, hi]; `count` tokens and `mass` lie above.
struct Range {
  bool keyed;
  int b0, b1;
  uint32_t lo, hi;
  uint32_t count;
  double mass;
};

struct Found {
  int b;               // bucket (kRowsBuckets: no border in any)
  uint32_t cnt;        // tokens in it
  uint32_t above_c;    // tokens and mass above it
  unsigned long long above_m;
};

struct Search {
  const RowsParams& p;
  RowsShared& sh;
  const Row& row;
  cg::cluster_group cl;
  int ctas;
  double unit;  // mass of one fixed-point step

  // Adds up the cluster's histogram: f(value, add) calls add(bucket) for a
  // token that counts. Afterwards every CTA's slice holds running sums.
  template <class F>
  __device__ void histogram(bool mass, F f) {
    const int tid = threadIdx.x;
    const int arrays = mass ? 4 : 1;
    for (int i = tid; i < arrays * kRowsBuckets; i += kRowsThreads) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << p.part_bits) - 1;
    row.each([&](float v, uint32_t) {
      f(v, [&](int b) {
        atomicAdd(&sh.hist[0][b], 1u);
        if (mass) {
          // 2^52 + w rounds w to an integer in the low mantissa bits
          const unsigned long long w =
              (unsigned long long)__double_as_longlong(row.weight(v, p.mass_bits) + 4503599627370496.0) &
              0xfffffffffffffull;
          const uint32_t w0 = (uint32_t)w & mask, w1 = (uint32_t)(w >> p.part_bits) & mask,
                         w2 = (uint32_t)(w >> (2 * p.part_bits));
          if (w0) atomicAdd(&sh.hist[1][b], w0);
          if (w1) atomicAdd(&sh.hist[2][b], w1);
          if (w2) atomicAdd(&sh.hist[3][b], w2);
        }
      });
    });
    cl.sync();
    // this CTA's slice: thread i sums bucket i of it over the cluster
    const int per = kRowsBuckets / ctas, rank = (int)cl.block_rank();
    uint32_t c = 0;
    unsigned long long m = 0;
    if (tid < per) {
      const int b = rank * per + tid;
#pragma unroll
      for (int q = 0; q < kRowsMaxCtas; ++q)
        if (q < ctas) {
          const uint32_t* h = cl.map_shared_rank(&sh.hist[0][0], q) + b;
          c += h[0];
          if (mass)
            m += h[kRowsBuckets] + ((unsigned long long)h[2 * kRowsBuckets] << p.part_bits) +
                 ((unsigned long long)h[3 * kRowsBuckets] << (2 * p.part_bits));
        }
    }
    unsigned long long tc, tm = 0;
    const uint32_t ec = (uint32_t)rows_scan((unsigned long long)c, sh.redu, tc);
    const unsigned long long em = mass ? rows_scan(m, sh.redu, tm) : 0ull;
    if (tid < per) {
      sh.slice_c[tid] = ec;
      sh.slice_m[tid] = em;
    }
    if (tid == 0) {
      sh.slice_c[per] = (uint32_t)tc;
      sh.slice_m[per] = tm;
    }
    cl.sync();
  }

  // The row's (or range's) whole mass and count, from the slices.
  __device__ void totals(unsigned long long& count, unsigned long long& mass) const {
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
  __device__ Found find(const Targets& want, uint32_t c0, double m0, bool mass, int most, F meets) {
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
    // thread b looks at bucket b, in the slice of CTA b / per
    const int q = tid / per, i = tid - q * per;
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
    const uint32_t a0 = base_c + pc[0], cnt = base_c + pc[1] - a0;
    unsigned long long am = 0, mm = 0;
    if (mass) {
      am = base_m + pm[0];
      mm = base_m + pm[1] - am;
    }
    if (cnt && ((double)(c0 + a0 + cnt) >= want.k ||
                (mass && m0 + (double)(am + mm) * unit >= want.mass) || meets(tid)))
      atomicMin(&sh.pick[0], tid);
    __syncthreads();
    Found f;
    f.b = sh.pick[0];
    if (tid == min(f.b, kRowsBuckets - 1)) {
      sh.pick[1] = (int)cnt;
      sh.pick[2] = (int)(c0 + a0);
      sh.pickm = am;
    }
    __syncthreads();
    f.cnt = (uint32_t)sh.pick[1];
    f.above_c = (uint32_t)sh.pick[2];
    f.above_m = sh.pickm;
    return f;
  }

  // Keys of the bucket g.b0 == g.b1, from the monotone bucket().
  __device__ void to_keys(Range& g) const {
    const int b = g.b0;
    const uint32_t first = kKeyNone + 1;
    g.hi = row.top;
    g.lo = first;
    if (b > 0) {  // largest key with bucket >= b
      uint32_t x = first, y = row.top;  // bucket(x) >= b > bucket(y)
      while (y - x > 1) {
        const uint32_t m = x + (y - x) / 2;
        (row.bucket(rows_value(m)) >= b ? x : y) = m;
      }
      g.hi = x;
    }
    if (row.bucket(rows_value(first)) > b) {  // smallest key with bucket <= b
      uint32_t x = first, y = row.top;  // bucket(x) > b >= bucket(y)
      while (y - x > 1) {
        const uint32_t m = x + (y - x) / 2;
        (row.bucket(rows_value(m)) > b ? x : y) = m;
      }
      g.lo = y;
    }
    g.keyed = true;
  }

  // Splits a range of keys and narrows it to the first part where a border is
  // reached (else the last with any token); returns the tokens in it.
  __device__ uint32_t split(Range& g, const Targets& want) {
    if (!g.keyed) to_keys(g);
    int shift = 0;
    while (((g.hi - g.lo) >> shift) >= (uint32_t)kRowsBuckets) ++shift;
    const uint32_t width = (1u << shift) - 1;
    cl.sync();  // the others have read the last slices
    const uint32_t lo = g.lo, hi = g.hi;
    histogram(true, [&](float v, auto add) {
      const uint32_t key = rows_key(v);
      if (key >= lo && key <= hi) add((int)((hi - key) >> shift));
    });
    // without a border: the last part with any token
    Targets all{INFINITY, INFINITY, 0};
    unsigned long long c, m;
    totals(c, m);
    all.k = (double)c;
    const int last = find(all, 0, 0.0, false, kRowsBuckets - 1, [](int) { return false; }).b;
    const Found f = find(want, g.count, g.mass, true, last, [&](int b) {
      return want.least && hi - ((uint32_t)b << shift) - width <= want.least;
    });
    g.count = f.above_c;
    g.mass += (double)f.above_m * unit;
    const uint32_t first_key = hi - ((uint32_t)f.b << shift);
    if (first_key - lo > width) g.lo = first_key - width;
    g.hi = first_key;
    return f.cnt;
  }

  // The cluster's tokens in the range (at most kRowsList), sorted in rank order
  // into sh.sort; returns their number. `which`: the list to use.
  __device__ uint32_t gather(const Range& g, int which) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sh.count[which] = 0;
    __syncthreads();
    row.each([&](float v, uint32_t token) {
      const uint32_t key = rows_key(v);
      bool in = Row::real(v);
      if (g.keyed) {
        in = in && key >= g.lo && key <= g.hi;
      } else {
        const int b = row.bucket(v);
        in = in && b >= g.b0 && b <= g.b1;
      }
      if (in) {
        const uint32_t at = atomicAdd(&sh.count[which], 1u);
        if (at < (uint32_t)kRowsList)
          sh.list[which][at] = ((unsigned long long)key << 32) | (uint32_t)~token;
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
    // two warps copy each CTA's list
    {
      const int q = warp & (kRowsMaxCtas - 1);
      const uint32_t n = __shfl_sync(0xffffffffu, k, q), base = __shfl_sync(0xffffffffu, incl, q) - n;
      if (q < ctas) {
        const unsigned long long* src = cl.map_shared_rank(&sh.list[which][0], q);
        for (uint32_t i = lane + 32 * (warp / kRowsMaxCtas); i < n; i += 64)
          if (base + i < (uint32_t)kRowsList) sh.sort[base + i] = src[i];
      }
    }
    uint32_t N = 2;
    while (N < m) N <<= 1;
    for (uint32_t i = m + tid; i < N; i += kRowsThreads) sh.sort[i] = 0ull;
    __syncthreads();
    // bitonic, descending; pairs less than 64 apart stay within one warp's 64
    // entries
    for (uint32_t kk = 2; kk <= N; kk <<= 1)
      for (uint32_t j = kk >> 1; j > 0; j >>= 1) {
        for (uint32_t i = tid; i < N / 2; i += kRowsThreads) {
          const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;  // pairs j apart
          const unsigned long long x = sh.sort[a], y = sh.sort[b];
          if ((a & kk) == 0 ? x < y : x > y) {
            sh.sort[a] = y;
            sh.sort[b] = x;
          }
        }
        if (j > 32 || (j == 1 && kk >= 64))
          __syncthreads();
        else
          __syncwarp();
      }
    __syncthreads();
    return m;
  }

  // Token of the t-th (1-based) element in index order with this key; in the
  // CTA that holds it.
  __device__ uint32_t nth_tie(uint32_t key, unsigned long long t) {
    const int tid = threadIdx.x;
    if (tid == 0) sh.result = 0xffffffffu;
    const float* x = row.x + (row.base - row.first);
    const uint32_t per = (row.count + kRowsThreads - 1) / kRowsThreads;
    const uint32_t lo = min(row.count, tid * per), hi = min(row.count, lo + per);
    unsigned long long mine = 0;
    for (uint32_t i = lo; i < hi; ++i) mine += rows_key(x[i]) == key;
    unsigned long long total;
    unsigned long long before = rows_scan(mine, sh.redu, total);
    if (tid == 0) sh.ties = total;
    cl.sync();
    const int rank = (int)cl.block_rank();
    for (int c = 0; c < rank; ++c) before += *cl.map_shared_rank(&sh.ties, c);
    if (before < t && t <= before + mine)
      for (uint32_t i = lo; i < hi; ++i)
        if (rows_key(x[i]) == key && ++before == t) {
          sh.result = row.base + i;
          break;
        }
    __syncthreads();
    return sh.result;
  }

  // The draw of a filtered row; the token in the CTA that writes it.
  __device__ uint32_t filtered(const Targets& borders, double top_p, double u) {
    const int tid = threadIdx.x, rank = (int)cl.block_rank();
    const bool by_p = top_p < 1.0;
    Targets kept = borders;
    // a mass histogram unless top-k alone makes the kept tokens fit a list;
    // then top-p needs the row's whole mass only
    bool mass = by_p && kept.k > (double)kRowsList / 2;
    if (by_p && !mass) {
      double mine = 0.0, total;
      row.each([&](float v, uint32_t) { mine += Row::real(v) ? row.weight(v) : 0.0; });
      rows_scan(mine, sh.red, total);
      if (tid == 0) sh.total = total;  // read after the histogram's barrier
    }
    const auto whole = [&](float v, auto add) {
      if (Row::real(v)) add(row.bucket(v));
    };
    const auto never = [](int) { return false; };
    double z = 0.0;  // the row's mass (by_p or mass)
    Found end;       // bucket of the last kept token; kRowsBuckets: every token is kept
    for (;;) {
      histogram(mass, whole);
      unsigned long long tc, tm;
      totals(tc, tm);
      if (mass) {
        z = (double)tm * unit;
      } else if (by_p) {
        const double x = rows_lane<double>(ctas, [&](int q) { return *cl.map_shared_rank(&sh.total, q); });
        z = 0.0;
#pragma unroll
        for (int q = 0; q < kRowsMaxCtas; ++q) z += __shfl_sync(0xffffffffu, x, q);
      }
      if (by_p) kept.mass = top_p * z;
      // (without a mass histogram the border by mass is found in the list)
      const int most = kept.least ? row.bucket(rows_value(kept.least)) : kRowsBuckets;
      end = find(kept, 0, 0.0, mass, most, never);
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
    double kept_mass = z;
    uint32_t end_key = kKeyNone + 1;  // no key below it is kept
    double end_ties = INFINITY;       // and of it so many
    bool fresh = true;                // the slices are those of the whole row
    // phase 0: where the kept tokens end; phase 1: where the draw falls, if
    // not among the tokens that phase 0 listed
    for (int phase = 0; phase < 2; ++phase) {
      Targets want = kept;
      Range g{false, 0, min(end.b, kRowsBuckets - 1), 0, 0, 0, 0.0};
      uint32_t members = end.cnt;
      if (!one_list) {
        Found f = end;
        if (phase == 0) {
          if (end.b >= kRowsBuckets) continue;  // everything is kept
          f.cnt = end.cnt - end.above_c;
        } else {
          want = Targets{INFINITY, u * kept_mass, 0};
          if (!fresh) {
            cl.sync();
            histogram(true, whole);
          }
          f = find(want, 0, 0.0, true, min(end.b, kRowsBuckets - 1), never);
        }
        g.b0 = g.b1 = f.b;
        g.count = f.above_c;
        g.mass = (double)f.above_m * unit;
        members = f.cnt;
        // a crowded bucket is split by the key's bits until it fits, or is one key
        while (members > (uint32_t)kRowsList && (!g.keyed || g.lo < g.hi)) {
          members = split(g, want);
          fresh = false;
        }
      }
      // --- settle the border among the listed tokens (or equal keys)
      if (members > (uint32_t)kRowsList) {  // `members` equal logits
        const double w = row.key_weight(g.lo);
        double n = want.k - (double)g.count;
        if (w > 0.0) n = fmin(n, ceil((want.mass - g.mass) / w));
        n = fmax(1.0, fmin(n, (double)members));
        if (phase == 1) {
          if (g.lo == end_key) n = fmin(n, end_ties);
          return nth_tie(g.lo, (unsigned long long)n);
        }
        if (want.least > g.lo) n = 0.0;  // min-p ends above them
        end_key = n > 0.0 ? g.lo : g.lo + 1;
        end_ties = n > 0.0 ? n : INFINITY;
        kept_mass = g.mass + n * w;
        continue;
      }
      const uint32_t m = gather(g, phase);
      const uint32_t at = 2 * tid;
      uint32_t key[2];
      double w[2], tw;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        key[i] = at + i < m ? (uint32_t)(sh.sort[at + i] >> 32) : 0u;
        w[i] = row.key_weight(key[i]);
      }
      const double ew = g.mass + rows_scan(w[0] + w[1], sh.red, tw);
      const double run[2] = {ew + w[0], ew + w[0] + w[1]};
      // entries that a border allows, and the first that reaches one
      __syncthreads();
      if (tid == 0) sh.pick[0] = (int)m - 1, sh.pick[1] = 0;
      __syncthreads();
      const uint32_t floor_key = phase == 0 ? want.least : end_key;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (at + i < m) {
          if ((double)(g.count + at + i + 1) >= want.k ||
              ((phase == 0 || w[i] > 0.0) && run[i] >= want.mass))
            atomicMin(&sh.pick[0], (int)(at + i));
          if (key[i] >= floor_key) atomicMax(&sh.pick[1], (int)(at + i) + 1);
        }
      __syncthreads();
      int e = min(sh.pick[0], sh.pick[1] - 1);  // the last kept entry, or the draw; -1: above all
      if (phase == 0) {
        __syncthreads();
        if ((uint32_t)e >= at && (uint32_t)e < at + 2) sh.pickd = run[e - at];
        __syncthreads();
        kept_mass = e >= 0 ? sh.pickd : g.mass;
        if (!one_list && !(u * kept_mass > g.mass)) {
          // above this list: no key of it may be drawn
          uint32_t hi = g.hi;
          if (!g.keyed) {
            to_keys(g);
            hi = g.hi;
          }
          end_key = hi + 1;
          continue;
        }
        // the draw is among these, too
        const double target = u * kept_mass;
        if (tid == 0) sh.pick[0] = e;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((int)at + i < e && w[i] > 0.0 && run[i] >= target)
            atomicMin(&sh.pick[0], (int)(at + i));
        __syncthreads();
        e = sh.pick[0];
      }
      return rank == 0 ? ~(uint32_t)sh.sort[max(0, e)] : 0xffffffffu;
    }
    return 0xffffffffu;  // not reached: phase 1 returns
  }

  // The draw of an unfiltered row, by the running sum in index order; the
  // token in the CTA that holds it.
  __device__ uint32_t unfiltered(double u) {
    const int tid = threadIdx.x, rank = (int)cl.block_rank();
    if (tid == 0) sh.result = 0xffffffffu, sh.last = 0;
    const float* x = row.x + (row.base - row.first);
    const uint32_t per = (row.count + kRowsThreads - 1) / kRowsThreads | 1u;  // odd: no bank twice
    const uint32_t lo = min(row.count, tid * per), hi = min(row.count, lo + per);
    double mine = 0.0;
    uint32_t last = 0xffffffffu;
    for (uint32_t i = lo; i < hi; ++i) {
      const double w = Row::real(x[i]) ? row.weight(x[i]) : 0.0;
      mine += w;
      if (w > 0.0) last = i;
    }
    double total;
    const double before = rows_scan(mine, sh.red, total);
    if (tid == 0) sh.total = total;
    cl.sync();
    const double xs = rows_lane<double>(ctas, [&](int q) { return *cl.map_shared_rank(&sh.total, q); });
    double z = 0.0, base = 0.0, run = 0.0;
    int holder = 0;  // the CTA whose sums reach the draw (else the last with any)
    bool reached = false;
#pragma unroll
    for (int q = 0; q < kRowsMaxCtas; ++q) z += __shfl_sync(0xffffffffu, xs, q);
    const double target = u * z;
#pragma unroll
    for (int q = 0; q < kRowsMaxCtas; ++q) {
      const double v = __shfl_sync(0xffffffffu, xs, q);
      if (v > 0.0 && !reached) {
        holder = q;
        base = run;
        reached = run + v >= target;
      }
      run += v;
    }
    if (holder != rank) return 0xffffffffu;
    // the first chunk that reaches the draw holds the token; where rounding at
    // its seam leaves the inner scan short, its last one
    if (last != 0xffffffffu) {
      atomicMax(&sh.last, last);
      if (base + before + mine >= target) {
        double r = base + before;
        uint32_t hit = last;
        for (uint32_t i = lo; i < hi; ++i) {
          const double w = Row::real(x[i]) ? row.weight(x[i]) : 0.0;
          r += w;
          if (w > 0.0 && r >= target) {
            hit = i;
            break;
          }
        }
        atomicMin(&sh.result, hit);
      }
    }
    __syncthreads();
    return row.base + (sh.result != 0xffffffffu ? sh.result : sh.last);
  }
};

__global__ void __launch_bounds__(kRowsThreads, 2)
    sample_rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(16) float s_row[];
  __shared__ RowsShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t r = blockIdx.x / ctas;
  Row row;
  row.base = min(p.n, p.chunk * (uint32_t)rank);
  row.count = min(p.n, row.base + p.chunk) - row.base;
  const float* src = p.logits + r * p.stride + row.base;
  row.cached = p.cached;
  row.x = src;
  row.first = row.base;
  row.n4 = (row.count + 3) / 4;
  if (tid == 0) mbar_init(&sh.bar, 1);
  mbar_fence_init();
  if (tid < kRowsTable) sh.table[tid] = exp2((double)tid / kRowsTable);
  __syncthreads();
  pdl_wait();
  if (p.cached) {
    // the 16-byte aligned middle by bulk copies, the ragged ends by loads; the
    // copy keeps the row's misalignment, the ends are padded
    const uint32_t mis = (uint32_t)((reinterpret_cast<uintptr_t>(src) >> 2) & 3);
    float* dst = s_row + mis;
    const uint32_t head = min(row.count, (4 - mis) & 3), body = (row.count - head) / 4 * 4;
    if (tid == 0 && body) {
      mbar_arrive_expect_tx(&sh.bar, body * 4);
      for (uint32_t o = 0; o < body; o += 4096)
        bulk_g2s(dst + head + o, src + head + o, min(4096u, body - o) * 4, &sh.bar);
    }
    const uint32_t tail = head + body, end = mis + row.count;
    if ((uint32_t)tid < mis) s_row[tid] = __uint_as_float(kRowsPad);
    if ((uint32_t)tid < head) dst[tid] = src[tid];
    if (tid < 4 && tail + tid < row.count) dst[tail + tid] = src[tail + tid];
    if (tid < 4 && end + tid < (end + 3) / 4 * 4) s_row[end + tid] = __uint_as_float(kRowsPad);
    if (body) mbar_wait_timed(&sh.bar, 0, &g_rows_status);
    __syncthreads();
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
    row.each([&](float v, uint32_t token) {
      const unsigned long long x = argmax_pack(v, token);
      best = x > best ? x : best;
    });
  } else {
    uint32_t top = 0;
    row.each([&](float v, uint32_t) { top = max(top, rows_key(v)); });
    best = (unsigned long long)top << 32;
  }
  best = warp_max_u64(best);
  if (lane == 0) sh.redu[warp] = best;
  __syncthreads();
  best = warp_max_u64(lane < kRowsWarps ? sh.redu[lane] : 0ull);
  if (tid == 0) sh.best = best;
  cl.sync();
  best = warp_max_u64(rows_lane<unsigned long long>(
      ctas, [&](int q) { return *cl.map_shared_rank(&sh.best, q); }));
  row.top = (uint32_t)(best >> 32);
  uint32_t token = 0xffffffffu;  // set in the CTA that writes it
  if (greedy) {
    if (rank == 0) token = ~(uint32_t)best;
  } else if (row.top <= kKeyNone) {
    if (rank == 0) token = 0;  // nothing to draw from
  } else {
    row.fmax = rows_value(row.top);
    const float tt = fmaxf(t, 1e-30f);  // (what lies below differs from it by nothing)
    row.per = kRowsPerNat / tt;
    row.dmax = (double)row.fmax;
    row.scale = (kRowsTable * 1.4426950408889634074) / (double)tt;
    row.table = sh.table;
    Search s{p, sh, row, cl, ctas, ldexp(1.0, -p.mass_bits)};
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
        uint32_t lo = kKeyNone, hi = row.top;  // w(lo) < bar <= w(hi)
        while (hi - lo > 1) {
          const uint32_t step = (hi - lo - 1) / 32 + 1;
          const uint32_t probe = min(lo + step * (lane + 1), hi);
          const uint32_t yes = __ballot_sync(
              0xffffffffu, probe == hi || row.weight(rows_value(probe)) >= min_p);
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
  p.cached = p.chunk <= kRowsCached - 4;
  int chunk_bits = 0, n_bits = 0;
  while ((1u << chunk_bits) < p.chunk) ++chunk_bits;
  while ((1u << n_bits) < p.n) ++n_bits;
  p.part_bits = 32 - chunk_bits < 16 ? 32 - chunk_bits : 16;
  p.mass_bits = 3 * p.part_bits - 1 < 62 - n_bits ? 3 * p.part_bits - 1 : 62 - n_bits;
  if (p.mass_bits > 47) p.mass_bits = 47;
  const size_t smem = p.cached ? ((size_t)p.chunk + 8) * sizeof(float) : 0;
  const void* fn = reinterpret_cast<const void*>(sample_rows_kernel);
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
  MINQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_rows_kernel, p));
  return MINQ_OK;
}

}  // extern "C"
