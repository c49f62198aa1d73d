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
// All weights and sums are f64: next to a border a draw is decided by digits
// that an f32 sum over a vocabulary does not hold.
//
// One CTA per row. A prefix of the rank order is a key tau (the logits' order
// as an unsigned integer) and a number of ties at tau in index order, so every
// search is a bisection over the 32 bits of the key.
#include <math.h>

#include <string>

#include "common.cuh"
#include "kernels.h"

namespace minq {

namespace {

constexpr int kRowsThreads = 1024;

struct RowsParams {
  const float* logits;
  size_t stride, n;
  const float* temperature;  // null: 1
  const int* top_k;          // null or <= 0: off
  const float* top_p;        // null or >= 1: off
  const float* min_p;        // null or <= 0: off
  const float* u;
  uint32_t* out;
};

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
constexpr uint32_t kKeyInf = 0xff800000u;   // key of +infinity

struct RowsShared {
  double red[32];
  unsigned long long redu[32];
  uint32_t result, last;
};

__device__ double rows_sum(double v, RowsShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) sh.red[warp] = v;
  __syncthreads();
  v = lane < nw ? sh.red[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Row {
  const float* x;
  uint32_t n;
  uint32_t top;  // key of the maximum
  double vmax, inv_t;
  __device__ double weight(uint32_t key) const {
    if (key == top) return 1.0;
    if (key <= kKeyNone) return 0.0;
    return exp(((double)rows_value(key) - vmax) * inv_t);
  }
};

// Count and mass of the keys >= x.
__device__ void rows_measure(const Row& row, uint32_t x, double& cnt, double& mass,
                             RowsShared& sh) {
  double c = 0.0, m = 0.0;
  for (uint32_t i = threadIdx.x; i < row.n; i += blockDim.x) {
    const uint32_t k = rows_key(row.x[i]);
    if (k >= x) {
      c += 1.0;
      m += row.weight(k);
    }
  }
  cnt = rows_sum(c, sh);
  mass = rows_sum(m, sh);
}

// A prefix of the rank order: keys above tau, then the first t at tau.
struct Prefix {
  uint32_t tau;
  double t, above_mass;
};

// Shortest prefix that holds `target` tokens (or mass).
__device__ Prefix rows_walk(const Row& row, bool by_mass, double target, RowsShared& sh) {
  uint32_t lo = kKeyNone + 1, hi = row.top + 1;  // F(lo) >= target > F(hi)
  double clo, mlo, chi = 0.0, mhi = 0.0;
  rows_measure(row, lo, clo, mlo, sh);
  target = fmin(target, by_mass ? mlo : clo);
  if (by_mass) target = fmax(target, 1e-300);
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    double c, m;
    rows_measure(row, mid, c, m, sh);
    if ((by_mass ? m : c) >= target) {
      lo = mid;
      clo = c;
      mlo = m;
    } else {
      hi = mid;
      chi = c;
      mhi = m;
    }
  }
  Prefix f;
  f.tau = lo;
  f.above_mass = mhi;
  const double avail = clo - chi, w = row.weight(lo);
  f.t = by_mass ? (w > 0.0 ? ceil((target - mhi) / w) : avail) : target - chi;
  f.t = fmax(1.0, fmin(f.t, avail));
  return f;
}

__device__ __forceinline__ bool shorter(const Prefix& a, const Prefix& b) {
  return a.tau > b.tau || (a.tau == b.tau && a.t < b.t);
}

// Index of the t-th element (1-based, index order) with key == tau.
__device__ uint32_t rows_nth(const Row& row, uint32_t tau, double t, RowsShared& sh) {
  if (threadIdx.x == 0) sh.result = 0;
  const uint32_t per = (row.n + blockDim.x - 1) / blockDim.x;
  const uint32_t lo = min(row.n, threadIdx.x * per), hi = min(row.n, lo + per);
  unsigned long long mine = 0;
  for (uint32_t i = lo; i < hi; ++i) mine += rows_key(row.x[i]) == tau;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  __syncthreads();
  if (lane == 31) sh.redu[warp] = incl;
  __syncthreads();
  for (int w = 0; w < warp; ++w) incl += sh.redu[w];
  const unsigned long long want = (unsigned long long)t, before = incl - mine;
  if (before < want && want <= incl) {
    unsigned long long seen = before;
    for (uint32_t i = lo; i < hi; ++i)
      if (rows_key(row.x[i]) == tau && ++seen == want) {
        sh.result = i;
        break;
      }
  }
  __syncthreads();
  return sh.result;
}

// First index whose running mass reaches r (index order, w > 0).
__device__ uint32_t rows_scan(const Row& row, double u, RowsShared& sh) {
  if (threadIdx.x == 0) sh.result = 0xffffffffu, sh.last = 0;
  const uint32_t per = (row.n + blockDim.x - 1) / blockDim.x;
  const uint32_t lo = min(row.n, threadIdx.x * per), hi = min(row.n, lo + per);
  double mine = 0.0;
  uint32_t last = 0xffffffffu;
  for (uint32_t i = lo; i < hi; ++i) {
    const double w = row.weight(rows_key(row.x[i]));
    mine += w;
    if (w > 0.0) last = i;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  __syncthreads();
  if (lane == 31) sh.red[warp] = incl;
  __syncthreads();
  double base = 0.0, total = 0.0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) base += sh.red[w];
    total += sh.red[w];
  }
  const double before = base + (incl - mine), r = u * total;
  // the first chunk that reaches r holds the token; rounding at its seam may
  // leave the inner scan short, then it is the chunk's last token
  if (mine > 0.0 && before + mine >= r) {
    double run = before;
    uint32_t hit = last;
    for (uint32_t i = lo; i < hi; ++i) {
      const double w = row.weight(rows_key(row.x[i]));
      run += w;
      if (w > 0.0 && run >= r) {
        hit = i;
        break;
      }
    }
    atomicMin(&sh.result, hit);
  }
  if (last != 0xffffffffu) atomicMax(&sh.last, last);
  __syncthreads();
  return sh.result != 0xffffffffu ? sh.result : sh.last;  // u = 1 and rounding
}

__global__ void __launch_bounds__(kRowsThreads) sample_rows_kernel(RowsParams p) {
  __shared__ RowsShared sh;
  pdl_wait();
  const size_t r = blockIdx.x;
  const float t = p.temperature ? p.temperature[r] : 1.0f;
  const int k = p.top_k ? p.top_k[r] : 0;
  const double top_p = p.top_p ? (double)p.top_p[r] : 1.0;
  const double min_p = p.min_p ? (double)p.min_p[r] : 0.0;
  const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
  Row row;
  row.x = p.logits + r * p.stride;
  row.n = (uint32_t)p.n;
  const bool greedy = !(t > 0.0f) || k == 1;
  // the maximum, lowest index first (greedy: the total order of minq_argmax)
  unsigned long long best = 0;
  if (greedy) {
    for (uint32_t i = threadIdx.x; i < row.n; i += blockDim.x) {
      const unsigned long long v = argmax_pack(row.x[i], i);
      best = v > best ? v : best;
    }
  } else {
    for (uint32_t i = threadIdx.x; i < row.n; i += blockDim.x) {
      const unsigned long long v = ((unsigned long long)rows_key(row.x[i]) << 32) | (uint32_t)~i;
      best = v > best ? v : best;
    }
  }
  best = warp_max_u64(best);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sh.redu[warp] = best;
  __syncthreads();
  best = warp_max_u64(lane < (int)(blockDim.x >> 5) ? sh.redu[lane] : 0ull);
  row.top = (uint32_t)(best >> 32);
  uint32_t token = ~(uint32_t)best;
  if (!greedy) {
    row.vmax = (double)rows_value(row.top);
    row.inv_t = 1.0 / (double)t;
    const bool by_k = k > 0 && (size_t)k < p.n, by_p = top_p < 1.0, by_m = min_p > 0.0;
    if (row.top <= kKeyNone) {
      token = 0;
    } else if (!by_k && !by_p && !by_m) {
      token = rows_scan(row, u, sh);
    } else {
      Prefix kept{kKeyNone, 0.0, 0.0};
      double cnt, z;
      rows_measure(row, kKeyNone + 1, cnt, z, sh);
      double kept_mass = z;
      if (by_k) {
        kept = rows_walk(row, false, (double)k, sh);
        kept_mass = kept.above_mass + kept.t * row.weight(kept.tau);
      }
      if (by_p) {
        const Prefix f = rows_walk(row, true, top_p * z, sh);
        if (shorter(f, kept)) kept = f, kept_mass = f.above_mass + f.t * row.weight(f.tau);
      }
      if (by_m) {  // smallest key with w >= min_p: w grows with the key
        uint32_t lo = kKeyNone, hi = row.top;
        while (hi - lo > 1) {
          const uint32_t mid = lo + (hi - lo) / 2;
          if (row.weight(mid) >= min_p)
            hi = mid;
          else
            lo = mid;
        }
        double c, m;
        rows_measure(row, hi, c, m, sh);
        if (min_p > 1.0)
          kept = Prefix{row.top, 1.0, 0.0}, kept_mass = 1.0;  // no token reaches it: the first
        else if (hi > kept.tau)
          kept = Prefix{hi, c, 0.0}, kept_mass = m;
      }
      Prefix f = rows_walk(row, true, u * kept_mass, sh);
      if (kept.tau > kKeyNone && shorter(kept, f)) f = kept;  // rounding at the last token
      token = rows_nth(row, f.tau, f.t, sh);
    }
  }
  if (threadIdx.x == 0) p.out[r] = token;
  pdl_launch_dependents();
}

}  // namespace

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
  p.n = n;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.u = uniforms;
  p.out = tokens;
  MINQ_CUDA_TRY(launch_k(sample_rows_kernel, dim3((unsigned)n_rows), dim3(kRowsThreads), 0,
                         (cudaStream_t)stream, p));
  return MINQ_OK;
}

}  // extern "C"
