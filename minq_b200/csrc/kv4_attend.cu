// Causal attention of a step's new tokens over the paged 4-bit K/V cache.
//
// Request r holds len_r positions (the step's tokens, already written, are
// the last n_r = q_start[r+1] - q_start[r] of them); its token i sits at
// position pos = len_r - n_r + i and attends over positions 0..=pos of its
// pages: the reference's attend (model.rs:223-248) with K and V the values
// the Q4_0 blocks stand for. Positions beyond the table row, in a page whose
// id is outside the pool, or before the start (pos < 0) do not exist; a row
// that sees nothing is zero.
#include <math.h>

#include <string>

#include "common.cuh"
#include "kernels.h"

namespace minq {

namespace {

struct Kv4AttnParams {
  const float* q;  // token t, head h at q + t * q_stride + h * hd
  size_t q_stride;
  const int* q_start;
  int n_tokens;
  const int* lens;
  int n_req;
  const int* table;
  size_t table_stride;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  int n_pages, page_shift;
  int nh, nkv, hd;
  float scale;
  float* out;
  size_t out_stride;
};

// Request of token t, or -1 where t lies behind the last sequence (or the
// starts are not a valid partition there).
__device__ __forceinline__ int kv4_request_of(const Kv4AttnParams& p, int t) {
  int lo = 0, hi = p.n_req;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return p.q_start[lo] <= t && t < p.q_start[lo + 1] ? lo : -1;
}

// One warp per (token, query head); any head_dim that is a multiple of 32.
// Scores: a lane per position; values: a lane per dimension of each block.
__global__ void __launch_bounds__(128) kv4_attend_rows_kernel(Kv4AttnParams p) {
  __shared__ float s_q[4][256];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row = (size_t)blockIdx.x * 4 + warp;
  if (row >= (size_t)p.n_tokens * p.nh) return;
  const int t = (int)(row / p.nh), h = (int)(row % p.nh);
  const int r = kv4_request_of(p, t);
  if (r < 0) return;
  const int nb = p.hd / kBlock, kvh = h / (p.nh / p.nkv);
  float* q = s_q[warp];
  for (int d = lane; d < p.hd; d += 32) q[d] = p.q[t * p.q_stride + (size_t)h * p.hd + d] * p.scale;
  __syncwarp();
  const long long pos = (long long)p.lens[r] - (p.q_start[r + 1] - t);
  const long long cap = (long long)p.table_stride << p.page_shift;
  const long long n = pos + 1 < cap ? pos + 1 : cap;  // positions seen (< 1: none)
  float m = -INFINITY, l = 0.0f, o[8] = {};
  for (long long p0 = 0; p0 < n; p0 += 32) {
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
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;  // nothing seen yet
    const float a = expf(m - mn), w = on ? expf(s - mn) : 0.0f;
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int b = 0; b < 8; ++b) o[b] *= a;
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
  float* out = p.out + (size_t)t * p.out_stride + (size_t)h * p.hd;
#pragma unroll
  for (int b = 0; b < 8; ++b)
    if (b < nb) out[b * 32 + lane] = l != 0.0f ? o[b] / l : 0.0f;
}

}  // namespace

}  // namespace minq

using namespace minq;

extern "C" {

size_t minq_kv4_attend_workspace_bytes(size_t n_req, size_t n_tokens, size_t n_heads, size_t n_kv,
                                       size_t head_dim) {
  return 0;
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
  if (n_tokens > 1 && (q_stride < n_heads * head_dim || out_stride < n_heads * head_dim))
    return fail(MINQ_ERR_ARG, "kv4_attend: token strides must be at least n_heads * head_dim");
  if (n_tokens == 0 || n_req == 0 || n_heads == 0) return MINQ_OK;
  if (!q || !q_start || !lens || !table || !out || (n_pages && (!k_pages || !v_pages)))
    return fail(MINQ_ERR_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15)
    return fail(MINQ_ERR_ARG, "kv4_attend: pools must be 16-byte aligned");
  if (workspace_bytes <
      minq_kv4_attend_workspace_bytes(n_req, n_tokens, n_heads, n_kv, head_dim))
    return fail(MINQ_ERR_ARG, "workspace smaller than minq_kv4_attend_workspace_bytes");
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
  const size_t rows = n_tokens * n_heads;
  MINQ_CUDA_TRY(launch_k(kv4_attend_rows_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0,
                         (cudaStream_t)stream, p));
  return MINQ_OK;
}

}  // extern "C"
