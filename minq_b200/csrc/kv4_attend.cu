// Causal attention of a step's new tokens over the paged 4-bit K/V cache.
//
// Request r holds len_r positions (the step's tokens, already written, are
// the last n_r = q_start[r+1] - q_start[r] of them); its token i sits at
// position pos = len_r - n_r + i and attends over positions 0..=pos of its
// pages: the reference's attend (model.rs:223-248) with K and V the values
// the Q4_0 blocks stand for. Positions beyond the table row, in a page whose
// id is outside the pool, or before the start (pos < 0) do not exist; a row
// that sees nothing is zero.
//
// Three kernels. Prompt chunks of head_dim 64 and 128 have tcgen05's
// (kv4_attend_umma.cu); other head dims than those two have a plain one (below).
// The kernel for single tokens and short runs of them, mma.sync: 4 to 16 columns
// are too few to fill tcgen05's 128 rows. With k_t = d_tb (c_tb - 8) for
// block b of 32 dimensions, scale s and codes c in 0..15,
//   score  z_t  = sum_b d_tb sum_i s q_i (c_ti - 8)
//   output o_i  = sum_t (p_t e_tb) (c_ti - 8)      (e: the scales of V)
// so the codes enter the MMAs exactly and the scales stay f32: they multiply
// the 32-dimension partial scores, and the weights before P V. q and p_t e_tb
// are split into two f16 parts (22 bits), each part one MMA with f32
// accumulation, which keeps the products to about f32's own rounding:
//   * q is scaled per row by a power of two that puts its largest value in
//     [2^10, 2^11), so the low part's smallest step is 2^-35 of that value;
//   * p e is scaled by 2^10 / 2^floor(log2 max e), which follows the largest
//     value scale seen, like the running maximum of the softmax; a step of its
//     low part is 2^-34 of the largest p e, whichever block of dimensions has that:
//     a block whose values are far smaller than another's is summed in its steps.
//     (V's scales may lie anywhere from 2^-64 to 2^100. Below, the steps no longer
//     shrink with them; above, weights under 2^-36 of the largest are flushed.)
// Codes become exact signed f16 integers, two per instruction pair. (Left
// unsigned, as the subnormals that their bits are, they cost half as much,
// but the offset 8 sum q then costs the scores a digit.)
//
// Tiles are transposed, scores = K (16 positions) x q^T (8 columns) and
// o^T = V^T (16 dimensions) x p^T: a column is a (token, query head) pair of one
// kv head, so the 4 to 8 heads of a group fill the MMA's narrow side. A V tile
// has its positions along k; two positions' codes are paired by one byte
// permutation of their words.
//
// Each warp works through its own tiles of 32 positions and keeps its own
// running maximum, sum and accumulator; its K and V rows (16 or 32 rows of one
// page: a contiguous run each) come by bulk copies into a private ring, so no warp waits
// for another until the item's end. The maximum is only moved when a weight
// would exceed 2^4 (one vote a tile), which leaves the accumulator alone
// almost always.
//
// Work split. An item is (request, kv head, column tile); its weight is its
// number of positions plus a constant for its start and end. The items of the
// step lie on one line, and every warp takes an equal piece of it, computed on
// the device from the lengths (no host synchronisation, graphs replay over
// changing lengths). An item inside one warp's piece is written out directly;
// the pieces of the others go to the workspace, one per warp, or one per CTA
// where an item fills it, and a second small launch joins them in a fixed
// order, so results repeat bit for bit.
//
// What bounds it: 64 requests of 1 to 8192 positions (8 kv heads of 128, 306 MB,
// 47 us at the measured copy rate) take 89 us, 3.4 TB/s: the parts of q and p e, the
// scales and the moves between lanes cost 460 warp instructions per 16 positions of a
// kv head, and a scheduler issues one in 0.67 of its cycles. 2 x 131071 positions of 2 kv heads
// of 64 take 31 us (41 MB), a third of it the join; 1 x 1000 positions 18 us, the
// launches and the dependent loads.
#include <limits.h>
#include <math.h>

#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kv4_attend.cuh"
#include "pipeline.cuh"

namespace minq {

namespace {

// Request of token t, or -1 where t lies behind the last sequence (or the
// starts are not a valid run of tokens there, see kv_req).
__device__ __forceinline__ int kv4_request_of(const Kv4AttnParams& p, int t) {
  int lo = 0, hi = p.n_req;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int a = p.q_start[lo], b = p.q_start[lo + 1];
  return a >= 0 && a <= t && t < b && b <= p.n_tokens ? lo : -1;
}

// One CTA per (token, query head), any head_dim that is a multiple of 32: the
// kernel for the head dims that no model of this library has (64 and 128 have
// the tensor-core kernels). Its warps take turns at 32 positions. Scores: a lane
// per position; values: a lane per dimension of each block. Measured: 8 requests
// of 2048 positions, 16 heads of 96, 207 us (128 dims on tensor cores 24).
constexpr int kKvRowsWarps = 8;
__global__ void __launch_bounds__(kKvRowsWarps * 32) kv4_attend_rows_kernel(Kv4AttnParams p) {
  __shared__ float s_q[256];
  __shared__ float s_o[kKvRowsWarps][256];
  __shared__ float s_m[kKvRowsWarps], s_l[kKvRowsWarps];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x / p.nh, h = blockIdx.x % p.nh;
  const int r = kv4_request_of(p, t);
  if (r < 0) return;
  const int nb = p.hd / kBlock, kvh = h / (p.nh / p.nkv);
  const float* q = s_q;
  for (int d = threadIdx.x; d < p.hd; d += kKvRowsWarps * 32)
    s_q[d] = p.q[t * p.q_stride + (size_t)h * p.hd + d] * p.scale;
  __syncthreads();
  const long long pos = (long long)p.lens[r] - (p.q_start[r + 1] - t);
  const long long cap = (long long)p.table_stride << p.page_shift;
  const long long n = pos + 1 < cap ? pos + 1 : cap;  // positions seen (< 1: none)
  float m = -INFINITY, l = 0.0f, o[8] = {};
  bool seen = false;
  for (long long p0 = 32 * warp; p0 < n; p0 += 32 * kKvRowsWarps) {
    // P >= 16: the 32 positions lie in one or two pages; a lane has its own row
    const long long i = p0 + lane;
    const int id = i < n ? p.table[(size_t)r * p.table_stride + (size_t)(i >> p.page_shift)] : -1;
    const bool on = id >= 0 && id < p.n_pages;
    size_t off = 0;
    float s = -INFINITY;
    if (on) {
      off = ((((size_t)id * p.nkv + kvh) << p.page_shift) +
             (size_t)(i & ((1ll << p.page_shift) - 1))) * nb * kQ4Bytes;
      s = 0.0f;
      for (int b = 0; b < nb; ++b) {
        const uint32_t* blk = reinterpret_cast<const uint32_t*>(p.k_pages + off + b * kQ4Bytes);
        float acc = 0.0f;
        for (int w = 0; w < 4; ++w) {
          const uint32_t c = blk[1 + w];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            acc += q[b * 32 + w * 8 + e] * (float)((int)((c >> (4 * e)) & 15u) - 8);
        }
        s += acc * __uint_as_float(blk[0]);
      }
    }
    if (!__any_sync(0xffffffffu, on)) continue;
    seen = true;
    // (a maximum over NaN alone is -inf: the weights are NaN relative to anything)
    const float mn = fmaxf(m, warp_max(s)), ref = mn == -INFINITY ? 0.0f : mn;
    const float a = expf(m - ref), w = on ? expf(s - ref) : 0.0f;
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int b = 0; b < 8; ++b) o[b] *= a;
#pragma unroll 4
    for (int j = 0; j < 32; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const bool onj = __shfl_sync(0xffffffffu, (int)on, j) != 0;
      const size_t offj = __shfl_sync(0xffffffffu, (unsigned long long)off, j);
      if (!onj) continue;
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (b < nb) {
          const uint8_t* blk = p.v_pages + offj + b * kQ4Bytes;
          const uint8_t byte = blk[4 + lane / 2];
          const int c = (lane & 1) ? (byte >> 4) : (byte & 15);
          o[b] += wj * ((float)(c - 8) * *reinterpret_cast<const float*>(blk));
        }
    }
  }
  l = warp_sum(l);
#pragma unroll
  for (int b = 0; b < 8; ++b)
    if (b < nb) s_o[warp][b * 32 + lane] = o[b];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  const bool any = __syncthreads_or(seen) != 0;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kKvRowsWarps; ++w) M = fmaxf(M, s_m[w]);
  const float ref = M == -INFINITY ? 0.0f : M;
  float* out = p.out + (size_t)t * p.out_stride + (size_t)h * p.hd;
  for (int d = threadIdx.x; d < p.hd; d += kKvRowsWarps * 32) {
    float sum = 0.0f, L = 0.0f;
    for (int w = 0; w < kKvRowsWarps; ++w) {
      const float a = expf(s_m[w] - ref);  // 0 for a warp that saw nothing, NaN stays NaN
      sum += s_o[w][d] * a;
      L += s_l[w] * a;
    }
    // what is seen but weighs nothing (every score -inf) is not a number
    out[d] = any ? sum / L : 0.0f;
  }
}

// ---- tensor cores ------------------------------------------------------------

// Set when a bounded wait gave up (read and cleared by take_kv4_status): a
// file-scope word, so that no call allocates.
__device__ int g_kv4_status;

constexpr int kKvWarps = 4;
constexpr int kKvTile = 32;     // positions per tile
constexpr int kKvExtra = 64;    // an item's start and end, in positions
constexpr int kKvMinPiece = 96;  // smallest piece of the line per warp

// Requests of so many (token, head) rows of a kv head go to the tcgen05 kernel,
// whose tile has 128 rows whether they are filled or not. Measured (call, us,
// it / this one) at 32, 48, 64 and 128 rows a request: 32 requests of 2048
// positions, 8 kv heads, 163 / 124, 167 / 175, 169 / 220, 173 / 407; one of 8192
// positions 52 / 42, 54 / 52, 56 / 54, 69 / 77.
constexpr size_t kKvUmmaMin = 64;
constexpr int kKvUmmaSpread = 8;  // blocks that share the columns of its join's pieces

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// The part of (x, y) that a lane holds: round(x), or with neg = -1.0 (f16)
// round(x - round(x)).
__device__ __forceinline__ uint32_t part2(float x, float y, uint32_t neg) {
  const uint32_t hi = h2_bits(__floats2half2_rn(x, y));
  float a, b;
  asm("{\n\t.reg .f16 l, h, m, z;\n\tmov.b32 {l, h}, %2;\n\tmov.b32 {m, z}, %5;\n\t"
      "fma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, h, m, %4;\n\t}"
      : "=f"(a), "=f"(b)
      : "r"(hi), "f"(x), "f"(y), "r"(neg));
  return h2_bits(__floats2half2_rn(a, b));
}

// o[0..1] += c[0..1], one packed addition.
__device__ __forceinline__ void add2(float* o, const float* c) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(o[0]), "+f"(o[1])
      : "f"(c[0]), "f"(c[1]));
}

// Four 8x8 matrices of half words, transposed: lane i gives row i's address
// (16-byte aligned) and gets rows 2t, 2t + 1 of column g of each.
__device__ __forceinline__ void load_trans(uint32_t* d, const uint8_t* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(smem_u32(row))
               : "memory");
}

// First of the 4 dimensions of block b that lane group g holds of V. With
// head_dim 128 a row is five 16-byte chunks, which the transposing load reads
// whole: block b's half word h lies in column (2 b + 2 + h) mod 8 of its chunk.
template <int HD>
__device__ __forceinline__ int kv_dim(int b, int g) {
  return b * 32 + 4 * (HD == 128 ? (g - 2 * b - 2) & 7 : g);
}

template <int HD, int NT>
struct KvGeom {
  static constexpr int NB = HD / 32;             // blocks per row
  static constexpr int ROW = NB * kQ4Bytes;      // bytes per row
  static constexpr int HALF = 16 * ROW;          // K (or V) bytes of 16 positions
  static constexpr int SIDE = 2 * HALF;          // and of a tile
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int RING = STAGES * 2 * SIDE;
  static constexpr int COLS = 8 * NT;
  static constexpr int OP = HD + 8;              // row pitch of the merge area (floats)
  static constexpr int MERGE = COLS * OP * 4;
  static constexpr int PER_WARP = RING > MERGE ? RING : MERGE;
  static constexpr int SMEM = kKvWarps * PER_WARP + kKvWarps * COLS * 8 + kKvWarps * STAGES * 8 +
                              256;
};

// One warp's state for an item.
template <int HD, int NT, bool SPLIT>
struct KvState {
  static constexpr int NB = HD / 32;
  // [..][k step]: b0 b1 of the high, b0 b1 of the low part; SPLIT: of the
  // part that the lane's column g holds (high for g < 4, low of column g - 4)
  uint32_t q[NT][NB][2][SPLIT ? 2 : 4];
  float cn[NT][2];           // scores to log2 units
  int lim[NT][2];            // positions the column sees
  // running maximum less vlog, and sum: weights are 2^(z - m) = p 2^10 / vref
  float m[NT][2], l[NT][2];
  float o[NT][NB][2][4];
  float vref, vlog;          // 2^floor(log2 max value scale), log2(2^10 / vref)
  uint32_t neg_hi;           // SPLIT: f16 -1 where the lane's columns are low parts, else 0
  bool first;                // no tile seen yet (uniform over the warp)
};

// One tile of 32 positions, two halves of 16, whose K and V rows are at k and
// v; ok: the halves that were loaded (MASK: the others may hold anything).
template <int HD, int NT, bool SPLIT, bool MASK>
__device__ __forceinline__ void kv_tile(KvState<HD, NT, SPLIT>& st, const uint8_t* k, const uint8_t* v,
                                        int pos0, int lim_max, int n_nt, int ok) {
  constexpr int NB = HD / 32;
  constexpr int ROW = NB * kQ4Bytes;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // scores
  float s[2][NT][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][n][i] = 0.0f;
    const uint8_t* k0 = k + (16 * u + g) * ROW;
    const uint8_t* k1 = k0 + 8 * ROW;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t a0[4], a1[4];  // dimensions (0, 4), (1, 5), (2, 6), (3, 7) of the lane's eight
      codes4(*reinterpret_cast<const uint32_t*>(k0 + b * kQ4Bytes + 4 + 4 * t), a0);
      codes4(*reinterpret_cast<const uint32_t*>(k1 + b * kQ4Bytes + 4 + 4 * t), a1);
      const float d0 = *reinterpret_cast<const float*>(k0 + b * kQ4Bytes);
      const float d1 = *reinterpret_cast<const float*>(k1 + b * kQ4Bytes);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (NT > 1 && n >= n_nt) break;
        float c[4];
        const auto& q = st.q[n][b];
        if constexpr (SPLIT) {
          mma_f16_zero(c, a0[0], a1[0], a0[1], a1[1], q[0][0], q[0][1]);
        } else {
          // the small parts first: an MMA truncates its terms, and a truncation
          // next to the small sums is worth nothing
          mma_f16_zero(c, a0[0], a1[0], a0[1], a1[1], q[0][2], q[0][3]);
          mma_f16(c, a0[2], a1[2], a0[3], a1[3], q[1][2], q[1][3]);
          mma_f16(c, a0[0], a1[0], a0[1], a1[1], q[0][0], q[0][1]);
        }
        mma_f16(c, a0[2], a1[2], a0[3], a1[3], q[1][0], q[1][1]);
        s[u][n][0] = fmaf(c[0], d0, s[u][n][0]);
        s[u][n][1] = fmaf(c[1], d0, s[u][n][1]);
        s[u][n][2] = fmaf(c[2], d1, s[u][n][2]);
        s[u][n][3] = fmaf(c[3], d1, s[u][n][3]);
      }
    }
  }
  if (SPLIT) {  // columns n and n + 4 are the two parts of one
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][0][i] += __shfl_xor_sync(0xffffffffu, s[u][0][i], 2);
  }
  // value scales of positions g and g + 8 of each half
  float e[2][2][NB];
  float emax = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float x = *reinterpret_cast<const float*>(v + (16 * u + 8 * y + g) * ROW + b * kQ4Bytes);
        // what no column sees may be anything
        if (MASK && (!((ok >> u) & 1) || pos0 + 16 * u + 8 * y + g >= lim_max)) x = 0.0f;
        e[u][y][b] = x;
        emax = fmaxf(emax, fabsf(x));
      }
  if (__any_sync(0xffffffffu, emax >= 2.0f * st.vref)) {
    emax = 0.0f;  // infinite and NaN scales stay out of the reference
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          emax = fmaxf(emax, fabsf(e[u][y][b]) < INFINITY ? fabsf(e[u][y][b]) : 0.0f);
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) emax = fmaxf(emax, __shfl_xor_sync(0xffffffffu, emax, o));
    const float ref = fmaxf(__uint_as_float(__float_as_uint(emax) & 0x7f800000u), st.vref);
    const float f = st.vref / ref;  // powers of two
    const float up = (float)((int)(__float_as_uint(ref) >> 23) -
                             (int)(__float_as_uint(st.vref) >> 23));
    st.vref = ref;
    st.vlog -= up;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        st.m[n][c] += up;
        st.l[n][c] *= f;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) st.o[n][b][j][i] *= f;
    }
  }
  // softmax: x = z - m in log2 units
  float most = -INFINITY;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (NT > 1 && n >= n_nt) break;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = fmaf(s[u][n][i], st.cn[n][i & 1], -st.m[n][i & 1]);
        if (MASK && (!((ok >> u) & 1) || pos0 + 16 * u + g + (i >> 1) * 8 >= st.lim[n][i & 1]))
          x = -INFINITY;
        s[u][n][i] = x;
        most = fmaxf(most, x);
      }
  }
  if (st.first || __any_sync(0xffffffffu, most > 4.0f + st.vlog)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (NT > 1 && n >= n_nt) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        // the first tile sets the maximum (a column that sees none of it sees
        // none of the later ones), then it only grows
        x -= st.vlog;
        if (st.first)
          x = x == -INFINITY ? 0.0f : x;
        else
          x = fmaxf(x, 0.0f);
        const float a = st.first ? 1.0f : ex2(-x);
        st.m[n][c] += x;
        st.l[n][c] *= a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][n][c] -= x;
          s[u][n][c + 2] -= x;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            st.o[n][b][j][c] *= a;
            st.o[n][b][j][c + 2] *= a;
          }
      }
    }
    st.first = false;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (NT > 1 && n >= n_nt) break;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][n][i] = ex2(s[u][n][i]);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      st.l[n][c] += (s[0][n][c] + s[0][n][c + 2]) + (s[1][n][c] + s[1][n][c + 2]);
  }
  // o^T += V^T p^T: lane g holds 4 dimensions of a block (a half word, see
  // kv_dim), positions 2t, 2t + 1, 2t + 8, 2t + 9 of each half
  uint32_t chunk[4], next_chunk[4];
  if constexpr (HD == 128) load_trans(chunk, v + lane * ROW);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    uint32_t y[2][2][4];  // [half][pair of positions][dimension]
    if constexpr (HD == 128) {
      // half words 10 b + 2 .. 10 b + 9 of the row: lane g takes the one in its
      // column of 16-byte chunk b, lanes below 2 b + 2 that of chunk b + 1
      uint32_t x[4];
      if (b < 3) {
        load_trans(next_chunk, v + lane * ROW + 16 * (b + 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = g < 2 * b + 2 ? next_chunk[i] : chunk[i];
          chunk[i] = next_chunk[i];
        }
      } else {
        load_trans(x, v + lane * ROW + 64);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) codes4(x[i], y[i >> 1][i & 1]);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* w = v + (16 * u + 8 * h + 2 * t) * ROW + b * kQ4Bytes + 4 + 2 * g;
          const uint32_t x0 = *reinterpret_cast<const uint16_t*>(w);
          const uint32_t x1 = *reinterpret_cast<const uint16_t*>(w + ROW);
          codes4(__byte_perm(x0, x1, 0x5410), y[u][h]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (NT > 1 && n >= n_nt) break;
      uint32_t hi[2][2], lo[2][2];  // SPLIT: hi holds the lane's part
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w0 = s[u][n][2 * h], w1 = s[u][n][2 * h + 1];
          float p0 = w0 * e[u][h][b], p1 = w1 * e[u][h][b];
          if (MASK) {  // a weight of zero stays zero whatever the scale is
            p0 = w0 == 0.0f ? 0.0f : p0;
            p1 = w1 == 0.0f ? 0.0f : p1;
          }
          if (SPLIT) {
            hi[u][h] = transpose8x8(part2(p0, p1, st.neg_hi));
          } else {
            split2(p0, p1, hi[u][h], lo[u][h]);
            hi[u][h] = transpose8x8(hi[u][h]);
            lo[u][h] = transpose8x8(lo[u][h]);
          }
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // the tile's sum by itself, then added with rounding: MMAs into the
        // running sum would truncate it once each, always towards zero
        float c[4];
        if (SPLIT) {
          mma_f16_zero(c, y[0][0][2 * j], y[0][0][2 * j + 1], y[0][1][2 * j], y[0][1][2 * j + 1],
                       hi[0][0], hi[0][1]);
        } else {  // the small parts first: a truncation next to them costs nothing
          mma_f16_zero(c, y[0][0][2 * j], y[0][0][2 * j + 1], y[0][1][2 * j], y[0][1][2 * j + 1],
                       lo[0][0], lo[0][1]);
          mma_f16(c, y[1][0][2 * j], y[1][0][2 * j + 1], y[1][1][2 * j], y[1][1][2 * j + 1],
                  lo[1][0], lo[1][1]);
          mma_f16(c, y[0][0][2 * j], y[0][0][2 * j + 1], y[0][1][2 * j], y[0][1][2 * j + 1],
                  hi[0][0], hi[0][1]);
        }
        mma_f16(c, y[1][0][2 * j], y[1][0][2 * j + 1], y[1][1][2 * j], y[1][1][2 * j + 1],
                hi[1][0], hi[1][1]);
        add2(st.o[n][b][j], c);
        add2(st.o[n][b][j] + 2, c + 2);
      }
    }
  }
}

// The pieces of an item that starts in piece a: the warps' in the first and the
// last CTA that it touches, and one per CTA that it fills.
__device__ __forceinline__ KvRec kv_parts(const KvItem& it, int a, long long per, long long total) {
  const long long end = it.start + it.w, cta = per * kKvWarps;
  const int z = (int)((end - 1) / per), ca = a / kKvWarps, cz = z / kKvWarps;
  auto full = [&](int c) { return cta * c >= it.start && min(cta * (c + 1), total) <= end; };
  KvRec k;
  k.r = it.rq.r;
  k.h = it.h;
  k.j = (int)it.j;
  k.a = a;
  k.z0 = cz * kKvWarps;
  k.n_first = full(ca) ? 1 : min(z, ca * kKvWarps + kKvWarps - 1) - a + 1;
  k.n_mid = cz > ca ? cz - ca - 1 : 0;
  k.parts = k.n_first + k.n_mid + (cz > ca ? (full(cz) ? 1 : z - k.z0 + 1) : 0);
  return k;
}

// A warp's ring of tiles in flight.
struct KvRing {
  uint8_t* buf;
  uint64_t* bar;
  uint32_t fill, used;  // tiles issued and consumed so far
  bool alive;           // no wait has given up
};

// One warp's share of the part [x0, x1) of an item: every step-th of its tiles
// from tile `lead` on.
template <int HD, int NT, bool SPLIT>
__device__ __forceinline__ void kv_run(const Kv4AttnParams& p, const KvItem& it, int lead, int step,
                                       KvRing& ring, KvState<HD, NT, SPLIT>& st) {
  using GM = KvGeom<HD, NT>;
  constexpr int NB = GM::NB;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n_tiles = (it.lim_max + kKvTile - 1) / kKvTile;
  auto tile_at = [](long long x) { return x > kKvExtra ? (x - kKvExtra + kKvTile - 1) / kKvTile : 0; };
  const long long xa = tile_at(it.x0), xb = it.x1 == it.w ? n_tiles : tile_at(it.x1);
  const int ta = (int)min(xa, (long long)n_tiles) + lead, tb = (int)min(xb, (long long)n_tiles);
  const int my = tb > ta ? (tb - ta + step - 1) / step : 0;
  const int lim_max = it.lim_max;
  const size_t row0 = ((size_t)it.kvh << p.page_shift) * GM::ROW;
  const size_t page_bytes = ((size_t)p.nkv << p.page_shift) * GM::ROW;
  const int* tab = p.table + (size_t)it.rq.r * p.table_stride;
  // page ids of the halves of this warp's next 16 tiles, one per lane; -1
  // behind the last position
  auto tile_pos = [&](int i) { return (ta + i * step) * kKvTile; };
  auto load_ids = [&](int i0) {
    const int i = i0 + (lane >> 1);
    const int pos = tile_pos(i) + 16 * (lane & 1);
    int id = -1;
    if (i < my && pos < lim_max) id = tab[pos >> p.page_shift];
    return id < p.n_pages ? id : -1;
  };
  int ids = load_ids(0);
  // the columns' queries
  float v[NT][NB][8];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = SPLIT ? g & 3 : n * 8 + g, ct = col / p.gsz, ch = col - ct * p.gsz;
    const bool on = ct < it.ntok && ch < it.nhead;
    const float* qp = p.q + (size_t)(it.rq.t0 + it.tok0 + (on ? ct : 0)) * p.q_stride +
                      (size_t)(it.h0 + (on ? ch : 0)) * HD + 8 * t;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[n][b][e] = on ? qp[b * 32 + e] : 0.0f;
  }
  // tile i into the ring: lanes 0..3 copy a half of K or V each (16 rows of
  // one page); `from` holds the ids of its group of 16 tiles
  const int half = lane & 1;
  const uint8_t* side = (lane & 2 ? p.v_pages : p.k_pages) + row0;
  const int page_mask = (1 << p.page_shift) - 1;
  auto issue = [&](int i, int from) {
    const uint32_t sidx = ring.fill % GM::STAGES;
    uint64_t* bar = &ring.bar[sidx];
    const int id = __shfl_sync(0xffffffffu, from, 2 * (i & 15) + half);
    const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
    if (lane == 0 && ring.alive) {
      const uint32_t n = (have & 1) + ((have >> 1) & 1);
      if (n)
        mbar_arrive_expect_tx(bar, n * 2 * GM::HALF + p.stall);
      else
        mbar_arrive(bar);
    }
    __syncwarp();  // the bytes are expected before they can come
    if (lane < 4 && id >= 0 && ring.alive) {
      const int row = (tile_pos(i) + 16 * half) & page_mask;
      bulk_g2s(ring.buf + sidx * 2 * GM::SIDE + (lane >> 1) * GM::SIDE + half * GM::HALF,
               side + (size_t)id * page_bytes + row * GM::ROW, GM::HALF, bar);
    }
    if (ring.alive) ++ring.fill;
  };
  const int first = min(my, GM::STAGES);
  for (int i = 0; i < first; ++i) issue(i, ids);
  int ids_next = my > 16 ? load_ids(16) : -1;

  // q as f16 parts, limits
  const int n_nt = (it.ntok * p.gsz + 7) / 8;
  int lim_min = it.lim_max;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = SPLIT ? g & 3 : n * 8 + g, ct = col / p.gsz, ch = col - ct * p.gsz;
    const bool on = ct < it.ntok && ch < it.nhead;
    float amax = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[n][b][e]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // f: a power of two with amax * f in [2^10, 2^11)
    const int ex = min(max((int)(__float_as_uint(amax) >> 23), 24), 254);
    const float f = __uint_as_float((uint32_t)(264 - ex) << 23);
    const float cn = p.scale * 1.4426950408889634f * (1.0f / f);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float* e = v[n][b] + 2 * x + y;
          uint32_t hi, lo;
          split2(e[0] * f, e[4] * f, hi, lo);
          if constexpr (SPLIT) {
            st.q[n][b][x][y] = g < 4 ? hi : lo;
          } else {
            st.q[n][b][x][y] = hi;
            st.q[n][b][x][y + 2] = lo;
          }
        }
    st.cn[n][0] = __shfl_sync(0xffffffffu, cn, 8 * t);
    st.cn[n][1] = __shfl_sync(0xffffffffu, cn, 8 * t + 4);
    long long lim = on ? (long long)it.prior + it.tok0 + ct + 1 : 0;
    lim = lim < 0 ? 0 : lim < it.cap ? lim : it.cap;
    st.lim[n][0] = __shfl_sync(0xffffffffu, (int)lim, 8 * t);
    st.lim[n][1] = __shfl_sync(0xffffffffu, (int)lim, 8 * t + 4);
    if (on) lim_min = min(lim_min, (int)lim);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      st.m[n][c] = -74.0f;
      st.l[n][c] = 0.0f;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][b][y][i] = 0.0f;
  }
  lim_min = (int)__reduce_min_sync(0xffffffffu, (unsigned)lim_min);
  st.vref = 5.4210109e-20f;  // 2^-64: the weights' sums stay finite
  st.vlog = 74.0f;
  st.first = true;
  st.neg_hi = SPLIT && t >= 2 ? 0xbc00bc00u : 0u;

  for (int i = 0; i < my; ++i) {
    const uint32_t sidx = ring.used % GM::STAGES;
    if (ring.alive)
      ring.alive = mbar_wait_timed(&ring.bar[sidx], (ring.used / GM::STAGES) & 1, &g_kv4_status);
    ring.alive = __all_sync(0xffffffffu, ring.alive);
    if (ring.alive) ++ring.used;
    const int ok = (int)(__ballot_sync(0xffffffffu, ids >= 0) >> (2 * (i & 15))) & 3;
    if (ring.alive && ok) {
      const int pos0 = tile_pos(i);
      const uint8_t* kt = ring.buf + sidx * 2 * GM::SIDE;
      if (pos0 + kKvTile > lim_min || ok != 3)
        kv_tile<HD, NT, SPLIT, true>(st, kt, kt + GM::SIDE, pos0, lim_max, n_nt, ok);
      else
        kv_tile<HD, NT, SPLIT, false>(st, kt, kt + GM::SIDE, pos0, lim_max, n_nt, ok);
    }
    __syncwarp();
    const int nx = i + GM::STAGES;
    if (nx < my) issue(nx, (nx >> 4) == (i >> 4) ? ids : ids_next);
    if ((i & 15) == 15) {
      ids = ids_next;
      ids_next = load_ids(i + 17);
    }
  }
  if (!ring.alive) {  // a wait gave up: let the copies in flight end before the CTA does
    for (; ring.used < ring.fill; ++ring.used)
      mbar_wait_timed(&ring.bar[ring.used % GM::STAGES], (ring.used / GM::STAGES) & 1, &g_kv4_status);
  }
  // sums over the positions' lanes
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1)
        st.l[n][c] += __shfl_xor_sync(0xffffffffu, st.l[n][c], o);
      // the plain maximum and sum; o keeps the factor 2^10 / vref
      st.m[n][c] = st.l[n][c] == 0.0f ? -3.0e38f : st.m[n][c] + st.vlog;  // saw nothing
      st.l[n][c] *= st.vref * 0.0009765625f;
    }
}

template <int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(kKvWarps * 32, NT == 1 ? 4 : 2)
    kv4_attend_kernel(const __grid_constant__ Kv4AttnParams p) {
  using GM = KvGeom<HD, NT>;
  constexpr int NB = GM::NB, COLS = GM::COLS;
  extern __shared__ __align__(128) uint8_t smem[];
  float2* s_ml = reinterpret_cast<float2*>(smem + kKvWarps * GM::PER_WARP);  // [warp][cols]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_ml + kKvWarps * COLS);
  __shared__ long long s_red[kKvWarps];
  __shared__ long long s_start[kKvWarps];  // the request at each warp's start: its place
  __shared__ int s_req[kKvWarps];          // and its number
  __shared__ KvItem s_item[kKvWarps];      // the warps' items
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  KvRing ring{smem + warp * GM::PER_WARP, bars + warp * GM::STAGES, 0, 0, true};
  if (lane < GM::STAGES) mbar_init(&ring.bar[lane], 1);
  mbar_fence_init();
  pdl_wait();
  pdl_launch_dependents();

  // the line's length, and where the warps' pieces start
  const int H = p.nkv * p.hgroups;
  long long total = 0;
  for (int r = tid; r < p.n_req; r += kKvWarps * 32) {
    const KvReq q = kv_req(p, r);
    total += H * kv_cum(q, p.tpt, q.J);
  }
  const long long mine = total;  // with at most one round: request tid's weight
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_red[warp] = total;
  if (tid < kKvWarps) s_req[tid] = -1;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) total += s_red[w];
  long long per = (total + p.n_piece - 1) / p.n_piece;
  if (per < kKvMinPiece) per = kKvMinPiece;
  const long long c0 = per * kKvWarps * blockIdx.x, c1 = min(c0 + per * kKvWarps, total);
  KvRec* rec = p.rec + blockIdx.x * kKvWarps;
  if (c0 >= c1) {
    if (tid < kKvWarps) rec[tid].parts = 0;
    return;
  }
  long long before = 0;  // weight of the requests of earlier rounds
  for (int r0 = 0; r0 < p.n_req; r0 += kKvWarps * 32) {
    const int r = r0 + tid;
    long long w = mine;
    if (p.n_req > kKvWarps * 32) {
      w = 0;
      if (r < p.n_req) {
        const KvReq q = kv_req(p, r);
        w = H * kv_cum(q, p.tpt, q.J);
      }
    }
    long long incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) s_red[warp] = incl;
    __syncthreads();
    long long start = before + incl - w;
    for (int x = 0; x < kKvWarps; ++x) {
      if (x < warp) start += s_red[x];
      before += s_red[x];
    }
    if (r < p.n_req)
#pragma unroll
      for (int x = 0; x < kKvWarps; ++x) {
        const long long u = c0 + per * x;
        if (start <= u && u < start + w) {
          s_req[x] = r;
          s_start[x] = start;
        }
      }
    if (before > c1) break;  // uniform
  }
  __syncthreads();
  if (s_req[0] < 0) {  // cannot happen: the items cover the line
    if (tid < kKvWarps) rec[tid].parts = 0;
    return;
  }

  KvState<HD, NT, SPLIT> st;
  KvItem& it = s_item[warp];
  // One item that fills the whole CTA: the warps take turns at its tiles and
  // join in shared memory. Otherwise every warp takes its own piece of the line.
  bool joint;
  long long end;
  {
    KvItem x;
    kv_item_at(p, x, s_req[0], s_start[0], c0);
    joint = x.start + x.w >= c1;
    const long long u = joint ? c0 : c0 + per * warp;
    end = joint ? c1 : min(u + per, total);
    if (lane == 0) rec[warp].parts = 0;
    if (!joint && warp) {
      if (u >= end || s_req[warp] < 0) return;
      kv_item_at(p, x, s_req[warp], s_start[warp], u);
    }
    x.x0 = u - x.start;
    x.x1 = min(end - x.start, x.w);
    if (lane == 0) it = x;
    __syncwarp();
  }
  for (;;) {
    kv_run<HD, NT, SPLIT>(p, it, joint ? warp : 0, joint ? kKvWarps : 1, ring, st);
    const bool whole = it.x0 == 0 && it.x1 == it.w;
    const int slot = it.x0 > 0 ? 0 : 1;
    if (!whole && slot == 1 && lane == 0 && (!joint || warp == 0))
      rec[warp] = kv_parts(it, blockIdx.x * kKvWarps + warp, per, total);
    if (joint) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (g == 0) s_ml[warp * COLS + n * 8 + 2 * t + c] = make_float2(st.m[n][c], st.l[n][c]);
      __syncthreads();
      float* area = reinterpret_cast<float*>(ring.buf);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float M = -3.0e38f;
#pragma unroll
          for (int x = 0; x < kKvWarps; ++x)
            M = fmaxf(M, s_ml[x * COLS + n * 8 + 2 * t + c].x);
          f[c] = ex2(st.m[n][c] - M) * (st.vref * 0.0009765625f);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float* a = area + (n * 8 + 2 * t) * GM::OP + kv_dim<HD>(b, g) + 2 * y;
            const float* o = st.o[n][b][y];
            *reinterpret_cast<float2*>(a) = make_float2(o[0] * f[0], o[2] * f[0]);
            *reinterpret_cast<float2*>(a + GM::OP) = make_float2(o[1] * f[1], o[3] * f[1]);
          }
      }
      __syncthreads();
      for (int i = tid; i < (SPLIT ? 4 : COLS) * HD; i += kKvWarps * 32) {
        const int col = i / HD, d = i - col * HD;
        const int ct = col / p.gsz, ch = col - ct * p.gsz;
        if (ct >= it.ntok || ch >= it.nhead) continue;
        float M = -3.0e38f, L = 0.0f, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < kKvWarps; ++x) M = fmaxf(M, s_ml[x * COLS + col].x);
#pragma unroll
        for (int x = 0; x < kKvWarps; ++x) {
          const float2 ml = s_ml[x * COLS + col];
          L += ml.y * ex2(ml.x - M);
          const float* a = reinterpret_cast<const float*>(smem + x * GM::PER_WARP);
          sum += a[col * GM::OP + d];
          if (SPLIT) sum += a[(col + 4) * GM::OP + d];
        }
        if (whole) {
          p.out[(size_t)(it.rq.t0 + it.tok0 + ct) * p.out_stride + (size_t)(it.h0 + ch) * HD + d] =
              L != 0.0f ? sum / L : 0.0f;
        } else {
          const size_t at = ((size_t)blockIdx.x * kKvWarps * 2 + slot) * COLS + col;
          p.part_o[at * HD + d] = sum;
          if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
        }
      }
      return;
    }
    const size_t at = ((size_t)(blockIdx.x * kKvWarps + warp) * 2 + slot) * COLS;
    const float f = st.vref * 0.0009765625f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* dst[2];
      float r[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = SPLIT ? (2 * t + c) & 3 : n * 8 + 2 * t + c;
        const int ct = col / p.gsz, ch = col - ct * p.gsz;
        const float L = st.l[n][c];
        const bool on = ct < it.ntok && ch < it.nhead && (!SPLIT || t < 2);
        r[c] = !whole ? f : L != 0.0f ? f / L : 0.0f;
        dst[c] = !on     ? nullptr
                 : whole ? p.out + (size_t)(it.rq.t0 + it.tok0 + ct) * p.out_stride +
                               (size_t)(it.h0 + ch) * HD
                         : p.part_o + (at + col) * HD;
        if (on && !whole && g == 0)
          *reinterpret_cast<float2*>(p.part_ml + (at + col) * 2) = make_float2(st.m[n][c], L);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float o = st.o[n][b][y][i];
            if (SPLIT) o += __shfl_xor_sync(0xffffffffu, o, 2);
            if (dst[i & 1]) dst[i & 1][kv_dim<HD>(b, g) + 2 * y + (i >> 1)] = o * r[i & 1];
          }
    }
    KvItem x = it;
    __syncwarp();
    if (x.start + x.w >= end || !kv_item_next(p, x)) break;
    x.x0 = 0;
    x.x1 = min(end - x.start, x.w);
    if (lane == 0) it = x;
    __syncwarp();
  }
}

// Joins the pieces of the items that start in join_pieces pieces and go on
// behind them, always in a fixed order. An item of few pieces is summed by a warp
// per column, the (item, column) pairs dealt out to the eight warps; one of many
// by all eight warps, column by column. Columns are spread over gridDim.y blocks.
// (At four blocks an SM head_dim 128 spills 80 bytes, 64 four.)
constexpr int kKvJoinWarps = 8;
constexpr int kKvJoinAlone = 32;  // pieces
constexpr int kKvJoinRecs = 16;   // most pieces that a block looks through
template <int HD>
__global__ void __launch_bounds__(kKvJoinWarps * 32, 4)
    kv4_join_kernel(const __grid_constant__ Kv4AttnParams p0, const __grid_constant__ Kv4AttnParams p1) {
  // the first p0.join_blocks blocks have p0's pieces, the others p1's
  const bool second = (int)blockIdx.x >= p0.join_blocks;
  const Kv4AttnParams& p = second ? p1 : p0;
  const int block = second ? blockIdx.x - p0.join_blocks : blockIdx.x;
  constexpr int PER = HD / 32;  // values per lane
  __shared__ float s_o[kKvJoinWarps][HD];
  __shared__ float s_l[kKvJoinWarps];
  __shared__ KvRec s_rec[kKvJoinRecs];
  __shared__ int2 s_tok[kKvJoinRecs];  // the request's first token, its tokens
  __shared__ int s_n;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {  // the items that there are, in order
    const int c = block * p.join_pieces + lane;
    KvRec rec{};
    if (lane < p.join_pieces && c < p.n_piece) rec = p.rec[c];
    const uint32_t some = __ballot_sync(0xffffffffu, rec.parts > 0);
    const int at = __popc(some & ((1u << lane) - 1));
    if (rec.parts > 0) {
      s_rec[at] = rec;
      const int a = p.q_start[rec.r];
      s_tok[at] = make_int2(a, p.q_start[rec.r + 1] - a);
    }
    if (lane == 0) s_n = __popc(some);
  }
  __syncthreads();
  const int n_rec = s_n;
  const int G = p.nh / p.nkv, used = p.tpt * p.gsz;  // columns that hold anything
  // the item's row of `out` for a column, or null
  auto row = [&](int k, int col) -> float* {
    const KvRec& rec = s_rec[k];
    const int ct = col / p.gsz, ch = col - ct * p.gsz;
    const int kvh = rec.h / p.hgroups, head = (rec.h - kvh * p.hgroups) * p.gsz + ch;
    const int tok = rec.j * p.tpt + ct;
    if (tok >= s_tok[k].y || head >= G) return nullptr;
    return p.out + (size_t)(s_tok[k].x + tok) * p.out_stride + (size_t)(kvh * G + head) * HD;
  };
  // pieces w, w + step, .. of an item: their sum relative to the maximum M of all
  // (B: loads in flight)
  auto sum = [&](auto batch, const KvRec& rec, int col, int w, int step, float& L, float* acc) {
    constexpr int B = decltype(batch)::value;
    auto at = [&](int i) {
      const int piece = i < rec.n_first ? rec.a + i
                        : i < rec.n_first + rec.n_mid
                            ? (rec.a / kKvWarps + 1 + i - rec.n_first) * kKvWarps
                            : rec.z0 + (i - rec.n_first - rec.n_mid);
      return ((size_t)piece * 2 + (i == 0 ? 1 : 0)) * p.cols + col;
    };
    float M = -3.0e38f;
    for (int i0 = 0; i0 < rec.parts; i0 += 32 * B) {
      float m[B];
#pragma unroll
      for (int e = 0; e < B; ++e) {
        const int i = i0 + 32 * e + lane;
        m[e] = i < rec.parts ? p.part_ml[at(i) * 2] : M;
      }
#pragma unroll
      for (int e = 0; e < B; ++e) M = fmaxf(M, m[e]);
    }
    M = warp_max(M);
    L = 0.0f;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] = 0.0f;
    for (int i0 = w; i0 < rec.parts; i0 += B * step) {
      float2 ml[B];
      float v[B][PER];
#pragma unroll
      for (int e = 0; e < B; ++e) {
        const int i = i0 + e * step;
        if (i >= rec.parts) {
          ml[e] = make_float2(-INFINITY, 0.0f);
#pragma unroll
          for (int d = 0; d < PER; ++d) v[e][d] = 0.0f;
          continue;
        }
        ml[e] = *reinterpret_cast<const float2*>(p.part_ml + at(i) * 2);
        const float* o = p.part_o + at(i) * HD + PER * lane;
#pragma unroll
        for (int d = 0; d < PER; d += 2) {
          const float2 x = *reinterpret_cast<const float2*>(o + d);
          v[e][d] = x.x;
          v[e][d + 1] = x.y;
        }
      }
#pragma unroll
      for (int e = 0; e < B; ++e) {
        const float f = ex2(ml[e].x - M);
        L += ml[e].y * f;
#pragma unroll
        for (int d = 0; d < PER; ++d) acc[d] += v[e][d] * f;
      }
    }
  };
  float L, acc[PER];
  for (int i = warp * gridDim.y + blockIdx.y; i < n_rec * used; i += kKvJoinWarps * gridDim.y) {
    const int k = i / used, col = i - k * used;
    if (s_rec[k].parts > kKvJoinAlone) continue;
    float* out = row(k, col);
    if (!out) continue;
    sum(std::integral_constant<int, 2>(), s_rec[k], col, 0, 1, L, acc);
#pragma unroll
    for (int d = 0; d < PER; ++d) out[PER * lane + d] = L != 0.0f ? acc[d] / L : 0.0f;
  }
  for (int k = 0; k < n_rec; ++k) {
    if (s_rec[k].parts <= kKvJoinAlone) continue;
    for (int col = blockIdx.y; col < used; col += gridDim.y) {
      float* out = row(k, col);
      if (!out) continue;
      sum(std::integral_constant<int, 8>(), s_rec[k], col, warp, kKvJoinWarps, L, acc);
      __syncthreads();  // the sums before have been read
#pragma unroll
      for (int d = 0; d < PER; ++d) s_o[warp][PER * lane + d] = acc[d];
      if (lane == 0) s_l[warp] = L;
      __syncthreads();
      for (int d = threadIdx.x; d < HD; d += kKvJoinWarps * 32) {
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int x = 0; x < kKvJoinWarps; ++x) {
          o += s_o[x][d];
          l += s_l[x];
        }
        out[d] = l != 0.0f ? o / l : 0.0f;
      }
    }
  }
}

// How the tensor-core kernel is launched for a call, or n_cta = 0 where the
// rows kernel serves it.
struct KvPlan {
  int nt, n_cta;
  bool split;    // columns hold the two parts of q: up to 4 columns a tile
  int umma_lo;   // requests of so many tokens go to the tcgen05 kernel (0: none)
  size_t ws, umma_ws;
  size_t bytes() const { return ws + umma_ws; }
};
KvPlan kv_plan(size_t n_req, size_t n_tokens, size_t n_heads, size_t n_kv, size_t hd) {
  KvPlan k{};
  if ((hd != 64 && hd != 128) || n_kv == 0 || n_req == 0) return k;
  const size_t G = n_heads / n_kv;
  // Columns of a tile and what is in them. Measured (call with 64 x 8192 cold, us):
  // G = 4, one token each: both parts of q in one tile of 8 columns 171, a tile a
  // part 256, two tiles a part 329. Two tiles a part or one: 12 to 16 heads to a
  // kv head, 32 x 4096, 52 / 60; 2, 3, 4, 8 tokens each of G = 4, 32 x 2048,
  // 91 / 83, 97 / 105, 99 / 124, 144 / 200 (two tokens lose a little this way: the
  // host has the step's totals only). Of the variants, <128, 1, false> spills 168 bytes
  // at its 128 registers, <128, 1, true> 40; the ones of two tiles have 229 to 254 and
  // spill nothing.
  // With kKvUmmaMin rows a request and more, the chunks are the tcgen05 kernel's and what
  // is left for the other one are mostly single tokens.
  const size_t gsz = G < (size_t)kKvUmmaRows ? G : kKvUmmaRows;
  const bool chunks = n_tokens > n_req && n_tokens * gsz >= kKvUmmaMin;
  const bool single = n_tokens <= n_req || n_tokens * gsz >= kKvUmmaMin * n_req;
  k.nt = G > 8 || !single ? 2 : 1;
  k.split = k.nt == 1 && G <= 4;
  k.n_cta = sm_count() * (k.nt == 1 ? 4 : 2);
  k.ws = (size_t)k.n_cta * kKvWarps * (2 * 8 * k.nt * (hd + 2) * 4 + sizeof(KvRec));
  if (chunks) {
    k.umma_lo = (int)((kKvUmmaMin + gsz - 1) / gsz);
    k.umma_ws = kv4_umma_workspace(hd);
  }
  return k;
}

template <int HD, int NT, bool SPLIT>
minq_status launch_kv4_attend(const Kv4AttnParams& p, cudaStream_t s) {
  using GM = KvGeom<HD, NT>;
  MINQ_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kv4_attend_kernel<HD, NT, SPLIT>), GM::SMEM));
  MINQ_CUDA_TRY(launch_k(kv4_attend_kernel<HD, NT, SPLIT>, dim3(p.n_piece / kKvWarps), dim3(kKvWarps * 32),
                         GM::SMEM, s, p));
  return MINQ_OK;
}

// One launch joins the pieces of both kernels (u: null where the tcgen05 kernel did not run).
template <int HD>
minq_status launch_kv4_join(Kv4AttnParams p, const Kv4AttnParams* u, cudaStream_t s) {
  // With few items (of one token each) every one has many pieces: their columns
  // are spread over blocks, and few blocks look for them. With many there are
  // some in every CTA. Measured (join alone, us): 2 x 131071 positions of 2 kv
  // heads 13 this way and 24 the other, 64 x 8192 of 8 kv heads 11 and 8.
  const bool few = (size_t)p.n_req * p.nkv * p.hgroups * 4 < (size_t)p.n_piece / kKvWarps;
  p.join_pieces = few ? kKvJoinRecs : kKvWarps;
  p.join_blocks = (p.n_piece + p.join_pieces - 1) / p.join_pieces;
  int blocks = p.join_blocks, spread = few ? 8 : (p.tpt * p.gsz + 3) / 4;
  Kv4AttnParams v = u ? *u : p;
  if (u) {
    v.join_pieces = 1;
    blocks += v.n_piece;
    spread = kKvUmmaSpread;
  }
  MINQ_CUDA_TRY(launch_k(kv4_join_kernel<HD>, dim3(blocks, spread), dim3(kKvJoinWarps * 32), 0, s, p, v));
  return MINQ_OK;
}

}  // namespace

minq_status take_kv4_status() {
  int v = 0;
  int u = 0;
  MINQ_TRY(take_kv4_umma_status(&u));
  MINQ_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv4_status, sizeof(int)));
  if (v != 0) {
    const int zero = 0;
    MINQ_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int)));
  }
  if ((u | v) == 0) return MINQ_OK;
  return fail(MINQ_ERR_TIMEOUT, "a bounded wait of kv4_attend timed out");
}

}  // namespace minq

using namespace minq;

extern "C" {

size_t minq_kv4_attend_workspace_bytes(size_t n_req, size_t n_tokens, size_t n_heads, size_t n_kv,
                                       size_t head_dim) {
  return kv_plan(n_req, n_tokens, n_heads, n_kv, head_dim).bytes();
}

minq_status minq_kv4_attend(const float* q, size_t q_stride, const int32_t* q_start,
                            size_t n_tokens, const int32_t* lens, size_t n_req,
                            const int32_t* table, size_t table_stride, const void* k_pages,
                            const void* v_pages, size_t n_pages, size_t page_size, size_t n_heads,
                            size_t n_kv, size_t head_dim, float scale, float* out,
                            size_t out_stride, void* workspace, size_t workspace_bytes,
                            void* stream) {
  if (n_kv == 0 || n_heads % n_kv != 0)
    return fail(MINQ_ERR_MODEL, "n_heads must be a multiple of n_kv_heads");
  if (head_dim == 0 || head_dim % kBlock != 0 || head_dim > 256)
    return fail(MINQ_ERR_SHAPE, "kv4_attend: head_dim must be a multiple of 32 up to 256, got " +
                                    std::to_string(head_dim));
  if (!kv4_page_size_ok(page_size))
    return fail(MINQ_ERR_SHAPE, "kv4_attend: page size must be a power of two in 16..1024, got " +
                                    std::to_string(page_size));
  if (n_heads > 4096 || n_req > 8192 || n_tokens > (1u << 24) || n_pages > (1u << 30) ||
      table_stride == 0 || table_stride > (1u << 30))
    return fail(MINQ_ERR_SHAPE, "kv4_attend: heads, requests, tokens, pages or table width out of "
                                "range");
  if (n_tokens * n_heads > 0x7fffffffu)
    return fail(MINQ_ERR_SHAPE, "kv4_attend: n_tokens * n_heads must be below 2^31");
  if (n_tokens > 1 && (q_stride < n_heads * head_dim || out_stride < n_heads * head_dim))
    return fail(MINQ_ERR_ARG, "kv4_attend: token strides must be at least n_heads * head_dim");
  if (n_tokens == 0 || n_req == 0 || n_heads == 0) return MINQ_OK;
  if (!q || !q_start || !lens || !table || !out || (n_pages && (!k_pages || !v_pages)))
    return fail(MINQ_ERR_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15)
    return fail(MINQ_ERR_ARG, "kv4_attend: pools must be 16-byte aligned");
  const KvPlan plan = kv_plan(n_req, n_tokens, n_heads, n_kv, head_dim);
  if (plan.ws && (!workspace || workspace_bytes < plan.bytes()))
    return fail(MINQ_ERR_ARG, "workspace smaller than minq_kv4_attend_workspace_bytes");
  if (plan.ws && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(MINQ_ERR_ARG, "kv4_attend: workspace must be 16-byte aligned");
  MINQ_TRY(require_device());
  Kv4AttnParams p{};
  p.q = q;
  p.q_stride = q_stride;
  p.q_start = q_start;
  p.n_tokens = (int)n_tokens;
  p.lens = lens;
  p.n_req = (int)n_req;
  p.table = table;
  p.table_stride = table_stride;
  p.k_pages = static_cast<const uint8_t*>(k_pages);
  p.v_pages = static_cast<const uint8_t*>(v_pages);
  p.n_pages = (int)n_pages;
  while ((size_t(1) << p.page_shift) < page_size) ++p.page_shift;
  p.nh = (int)n_heads;
  p.nkv = (int)n_kv;
  p.hd = (int)head_dim;
  p.scale = scale;
  p.out = out;
  p.out_stride = out_stride;
  if (plan.ws) {
    const int G = (int)(n_heads / n_kv), cols = 8 * plan.nt, most = plan.split ? 4 : cols;
    p.cols = cols;
    p.gsz = G < most ? G : most;
    p.hgroups = (G + p.gsz - 1) / p.gsz;
    p.tpt = most / p.gsz;
    cudaStream_t s = (cudaStream_t)stream;
    Kv4AttnParams u = p;
    if (plan.umma_lo) {
      u.n_lo = plan.umma_lo;
      u.n_hi = INT_MAX;
      u.stall = take_stall(kStallAttendChunks);
      MINQ_TRY(launch_kv4_umma(u, static_cast<uint8_t*>(workspace) + plan.ws, s));
    }
    p.n_lo = 1;
    p.n_hi = plan.umma_lo ? plan.umma_lo - 1 : INT_MAX;
    p.extra = kKvExtra;
    p.stall = take_stall(kStallAttend);
    p.n_piece = plan.n_cta * kKvWarps;
    p.rec = static_cast<KvRec*>(workspace);
    p.part_o = reinterpret_cast<float*>(p.rec + p.n_piece);
    p.part_ml = p.part_o + (size_t)p.n_piece * 2 * cols * head_dim;
    if (head_dim == 64) {
      MINQ_TRY((plan.split     ? launch_kv4_attend<64, 1, true>(p, s)
               : plan.nt == 1 ? launch_kv4_attend<64, 1, false>(p, s)
                              : launch_kv4_attend<64, 2, false>(p, s)));
      return launch_kv4_join<64>(p, plan.umma_lo ? &u : nullptr, s);
    }
    MINQ_TRY((plan.split     ? launch_kv4_attend<128, 1, true>(p, s)
             : plan.nt == 1 ? launch_kv4_attend<128, 1, false>(p, s)
                            : launch_kv4_attend<128, 2, false>(p, s)));
    return launch_kv4_join<128>(p, plan.umma_lo ? &u : nullptr, s);
  }
  MINQ_CUDA_TRY(launch_k(kv4_attend_rows_kernel, dim3((unsigned)(n_tokens * n_heads)),
                         dim3(kKvRowsWarps * 32), 0, (cudaStream_t)stream, p));
  return MINQ_OK;
}

}  // extern "C"
