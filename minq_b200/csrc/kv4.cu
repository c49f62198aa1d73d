// The paged 4-bit K/V cache: rows written as Q4_0 blocks and read back.
//
// A pool is [page][kv head][position in page][head_dim / 32] blocks of 20
// bytes (f32 scale, then 16 bytes; value 2i in the low, 2i + 1 in the high
// half of byte i): quantize.rs:120-143's storage, so a page is a block stream
// that minq_dequantize reads. Slot s is page s / P, position s % P.
//
// Codes are bit-identical to minq_quantize (quant.cu): d = max|x| / 8 with
// NaN skipped, id = 1 / d, code = clamp(round half away(x * id), -8, 7) + 8,
// NaN -> 0, and an all-zero block stores zero bytes.
//
// Bound by memory: 4 bytes read and 0.625 written per value (write), the
// other way round (read). Four lanes own a block of 32 values, eight values
// each: two 16-byte loads, a maximum over the four lanes by two shuffles, and
// one 4-byte word of codes per lane, the scale by the first; a warp covers
// 256 consecutive values, so every global access of it is one contiguous run.
// A value's code costs seven instructions (with roundf and an integer conversion
// each it is twenty, and the write then waits for the arithmetic): the rounding half
// away from zero is two additions rounded towards zero, and four codes are
// added up in one float before a single conversion. The write runs 25 a value in
// all: the other eighteen are the two divisions by multiplication, the slot's 64-bit
// arithmetic, loads, shuffles and the loop, for a unit of eight values. Measured at 8191 tokens of 8
// heads of 128 (77 MB each): write 19.7 us, 3.9 TB/s (24.4 us before), read 16.6 us,
// 4.7 TB/s; a copy of as many bytes at the measured rate takes 12 us.
#include <string>

#include "common.cuh"
#include "kernels.h"

namespace minq {

namespace {

struct Kv4RowsParams {
  const float* k_in;  // write: token t at t * stride; null when reading
  const float* v_in;
  float* k_out;       // read
  float* v_out;
  size_t k_stride, v_stride;  // floats between tokens
  const long long* slots;
  uint32_t n_units;           // units of eight values on one side (below 2^31)
  uint32_t token_m, row_m;    // u / (units per token), u / (units per row) as a product
  int token_s, row_s;
  int n_kv, hd, page_shift;
  long long n_slots;
  uint8_t* k_pages;
  uint8_t* v_pages;
};

// Eight consecutive values at x (16-byte aligned when VEC).
template <bool VEC>
__device__ __forceinline__ void load8(const float* x, float* v) {
  if (VEC) {
    const float4 a = *reinterpret_cast<const float4*>(x);
    const float4 b = *reinterpret_cast<const float4*>(x + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
  }
}

// One unit = eight values of one token and kv head: unit u = (token * n_kv +
// head) * (hd / 8) + eighth; blockIdx.y is the side (K or V).
struct Kv4Unit {
  uint32_t token;
  int head, e;
  uint8_t* block;  // the block's bytes, or null: a slot outside the pool
};

__device__ __forceinline__ Kv4Unit kv4_unit(const Kv4RowsParams& p, uint32_t u) {
  Kv4Unit c;
  const uint32_t per_row = (uint32_t)p.hd / 8;
  c.token = __umulhi(u, p.token_m) >> p.token_s;
  const uint32_t in = u - c.token * p.n_kv * per_row;
  c.head = (int)(__umulhi(in, p.row_m) >> p.row_s);
  c.e = (int)(in - c.head * per_row);
  const long long slot = p.slots[c.token];
  c.block = nullptr;
  if (slot >= 0 && slot < p.n_slots) {
    const size_t page = (size_t)(slot >> p.page_shift);
    const size_t off = (size_t)(slot & ((1ll << p.page_shift) - 1));
    const size_t rrow = ((page * p.n_kv + c.head) << p.page_shift) + off;
    c.block = (blockIdx.y ? p.v_pages : p.k_pages) +
              (rrow * (p.hd / kBlock) + c.e / 4) * kQ4Bytes;
  }
  return c;
}

// Codes of eight values times 1 / d, in quant.cu's steps.
__device__ __noinline__ uint32_t kv4_codes_slow(const float* v, float id) {
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = roundf(__fmul_rn(v[i], id));
    const int q = isnan(y) ? 0 : (int)fminf(fmaxf(y, -8.0f), 7.0f);
    word |= (uint32_t)(q + 8) << (4 * i);
  }
  return word;
}
__device__ __forceinline__ uint32_t kv4_codes(const float* v, float id) {
  float sum[2] = {0.0f, 0.0f};  // codes less 8, in base 16
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __fmul_rn(v[i], id);
    // floor(|y| + 1/2): the sum is exact, but for 1/2 - 2^-25, which rounds to 1
    // unless towards zero; 2^23 then leaves the integer
    const float m = __fadd_rz(__fadd_rz(fabsf(y), 0.5f), 8388608.0f) - 8388608.0f;
    float q = copysignf(m, y);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(q) : "f"(7.0f));
    sum[i >> 2] = fmaf(q, (float)(1 << (4 * (i & 3))), sum[i >> 2]);
  }
  // NaN anywhere, or an infinite product (a denormal scale's reciprocal)
  if (!(fabsf(sum[0]) + fabsf(sum[1]) < 1048576.0f)) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
    return kv4_codes_slow(x, id);
  }
  // + 0x8888: the codes' offset of 8
  const uint32_t a = __float_as_uint(sum[0] + (8388608.0f + 34952.0f));
  const uint32_t b = __float_as_uint(sum[1] + (8388608.0f + 34952.0f));
  return __byte_perm(a, b, 0x5410);
}

template <bool VEC>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4RowsParams p) {
  pdl_wait();
  // whole warps take whole steps (n_units is a multiple of 4, not of 32)
  const uint32_t step = gridDim.x * 256;
  for (uint32_t u0 = blockIdx.x * 256 + (threadIdx.x & ~31u); u0 < p.n_units; u0 += step) {
    const uint32_t u = u0 + (threadIdx.x & 31);
    const bool on = u < p.n_units;
    const Kv4Unit c = kv4_unit(p, on ? u : p.n_units - 1);
    float v[8];
    const float* x = (blockIdx.y ? p.v_in + c.token * p.v_stride : p.k_in + c.token * p.k_stride) +
                     (size_t)c.head * p.hd + c.e * 8;
    load8<VEC>(x, v);
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const float d = a / 8.0f;
    const uint32_t word = d != 0.0f ? kv4_codes(v, 1.0f / d) : 0u;
    if (on && c.block) {
      // blocks are 20 bytes: 4-byte aligned words
      *reinterpret_cast<uint32_t*>(c.block + 4 + 4 * (c.e & 3)) = word;
      if ((c.e & 3) == 0) *reinterpret_cast<float*>(c.block) = d;
    }
  }
  pdl_launch_dependents();
}

template <bool VEC>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4RowsParams p) {
  pdl_wait();
  for (uint32_t u = blockIdx.x * 256 + threadIdx.x; u < p.n_units; u += gridDim.x * 256) {
    const Kv4Unit c = kv4_unit(p, u);
    float v[8] = {};
    if (c.block) {
      const float d = *reinterpret_cast<const float*>(c.block);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(c.block + 4 + 4 * (c.e & 3));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn((float)((int)((w >> (4 * i)) & 15u) - 8), d);
    }
    float* o = (blockIdx.y ? p.v_out + c.token * p.v_stride : p.k_out + c.token * p.k_stride) +
               (size_t)c.head * p.hd + c.e * 8;
    if (VEC) {
      reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[i];
    }
  }
  pdl_launch_dependents();
}

minq_status kv4_rows_check(const char* what, size_t n_tokens, size_t n_kv, size_t hd,
                           size_t k_stride, size_t v_stride, size_t n_pages, size_t page_size) {
  const std::string w(what);
  if (hd == 0 || hd % kBlock != 0 || hd > 256)
    return fail(MINQ_ERR_SHAPE, w + ": head_dim must be a multiple of 32 up to 256, got " +
                                    std::to_string(hd));
  if (!kv4_page_size_ok(page_size))
    return fail(MINQ_ERR_SHAPE, w + ": page size must be a power of two in 16..1024, got " +
                                    std::to_string(page_size));
  if (n_kv == 0 || n_kv > 4096 || n_pages > (1u << 30) || n_tokens > (1u << 30))
    return fail(MINQ_ERR_SHAPE, w + ": kv heads, pages or tokens out of range");
  if (n_tokens > 1 && (k_stride < n_kv * hd || v_stride < n_kv * hd))
    return fail(MINQ_ERR_ARG, w + ": token strides must be at least n_kv * head_dim");
  return MINQ_OK;
}

// u / d == umulhi(u, m) >> s for u < 2^31 and d >= 2.
void divisor(uint32_t d, uint32_t* m, int* s) {
  int bits = 1;
  while ((1u << bits) < d) ++bits;
  *m = (uint32_t)((1ull << (31 + bits)) / d + 1);
  *s = bits - 1;
}

// Both sides of all tokens, in as many launches as keep the units below 2^31.
template <class K>
minq_status launch_rows(K kernel, Kv4RowsParams p, size_t n_tokens, cudaStream_t s) {
  const uint32_t per_row = (uint32_t)p.hd / 8, per_token = per_row * (uint32_t)p.n_kv;
  divisor(per_token, &p.token_m, &p.token_s);
  divisor(per_row, &p.row_m, &p.row_s);
  const size_t most = ((1u << 31) - 1024) / per_token, cap = (size_t)sm_count() * 16;
  for (size_t t = 0; t < n_tokens; t += most) {
    const size_t n = n_tokens - t < most ? n_tokens - t : most;
    p.n_units = (uint32_t)(n * per_token);
    const size_t g = (p.n_units + 255) / 256;
    MINQ_CUDA_TRY(
        launch_k(kernel, dim3((unsigned)(g < cap ? g : cap), 2), dim3(256), 0, s, p));
    p.slots += n;
    if (p.k_in) p.k_in += n * p.k_stride, p.v_in += n * p.v_stride;
    if (p.k_out) p.k_out += n * p.k_stride, p.v_out += n * p.v_stride;
  }
  return MINQ_OK;
}

int page_shift_of(size_t P) {
  int s = 0;
  while ((size_t(1) << s) < P) ++s;
  return s;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

}  // namespace minq

using namespace minq;

extern "C" {

minq_status minq_kv4_write(const float* k, const float* v, size_t k_stride, size_t v_stride,
                           const int64_t* slots, size_t n_tokens, size_t n_kv, size_t head_dim,
                           void* k_pages, void* v_pages, size_t n_pages, size_t page_size,
                           void* stream) {
  MINQ_TRY(kv4_rows_check("kv4_write", n_tokens, n_kv, head_dim, k_stride, v_stride, n_pages,
                          page_size));
  if (n_tokens == 0) return MINQ_OK;
  if (!k || !v || !slots || (n_pages && (!k_pages || !v_pages)))
    return fail(MINQ_ERR_ARG, "null pointer");
  if (!al16(k_pages) || !al16(v_pages))
    return fail(MINQ_ERR_ARG, "kv4_write: pools must be 16-byte aligned");
  MINQ_TRY(require_device());
  Kv4RowsParams p{};
  p.k_in = k;
  p.v_in = v;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.slots = reinterpret_cast<const long long*>(slots);
  p.n_kv = (int)n_kv;
  p.hd = (int)head_dim;
  p.page_shift = page_shift_of(page_size);
  p.n_slots = (long long)n_pages << p.page_shift;
  p.k_pages = static_cast<uint8_t*>(k_pages);
  p.v_pages = static_cast<uint8_t*>(v_pages);
  const bool vec = al16(k) && al16(v) && (k_stride | v_stride) % 4 == 0;
  return launch_rows(vec ? kv4_write_kernel<true> : kv4_write_kernel<false>, p, n_tokens,
                     (cudaStream_t)stream);
}

minq_status minq_kv4_read(const void* k_pages, const void* v_pages, size_t n_pages,
                          size_t page_size, const int64_t* slots, size_t n_tokens, size_t n_kv,
                          size_t head_dim, float* k, float* v, size_t k_stride, size_t v_stride,
                          void* stream) {
  MINQ_TRY(kv4_rows_check("kv4_read", n_tokens, n_kv, head_dim, k_stride, v_stride, n_pages,
                          page_size));
  if (n_tokens == 0) return MINQ_OK;
  if (!k || !v || !slots || (n_pages && (!k_pages || !v_pages)))
    return fail(MINQ_ERR_ARG, "null pointer");
  if (!al16(k_pages) || !al16(v_pages))
    return fail(MINQ_ERR_ARG, "kv4_read: pools must be 16-byte aligned");
  MINQ_TRY(require_device());
  Kv4RowsParams p{};
  p.k_out = k;
  p.v_out = v;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.slots = reinterpret_cast<const long long*>(slots);
  p.n_kv = (int)n_kv;
  p.hd = (int)head_dim;
  p.page_shift = page_shift_of(page_size);
  p.n_slots = (long long)n_pages << p.page_shift;
  p.k_pages = const_cast<uint8_t*>(static_cast<const uint8_t*>(k_pages));
  p.v_pages = const_cast<uint8_t*>(static_cast<const uint8_t*>(v_pages));
  const bool vec = al16(k) && al16(v) && (k_stride | v_stride) % 4 == 0;
  return launch_rows(vec ? kv4_read_kernel<true> : kv4_read_kernel<false>, p, n_tokens,
                     (cudaStream_t)stream);
}

}  // extern "C"
