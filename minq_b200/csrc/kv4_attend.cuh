// What the kernels of kv4_attend share: the call's parameters, the line of
// items that is split over warps or CTAs, and the exact f16 codes.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace minq {

// The item that starts in a piece of the line and goes on behind it.
struct KvRec {
  int parts, r, h, j;  // number of pieces (0: no item), request, head tile, column tile
  int a, n_first, n_mid, z0;  // first piece and pieces in its CTA, CTAs between, first in the last
};

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
  // tensor-core kernels
  // requests of n_lo to n_hi tokens are this kernel's; an item's start and end, in positions
  int n_lo, n_hi, extra;
  // columns of a tile (room for), heads per tile, head tiles per kv head, tokens per tile
  int cols, gsz, hgroups, tpt;
  int n_piece;       // pieces of the line
  int join_pieces, join_blocks;  // those that a block of the join looks through, its blocks
  float* part_o;     // [n_piece][2][cols][hd] unnormalised partial outputs
  float* part_ml;    // [n_piece][2][cols][2] their maxima and sums
  KvRec* rec;        // [n_piece]
  uint32_t stall;    // bytes a tile's wait expects beyond its copies (tests)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// (x, y) as two f16 pairs, high and low parts.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = h2_bits(__floats2half2_rn(x, y));
  float a, b;  // hi - x, exact; the mixed-precision form needs no conversion
  asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\t"
      "sub.rn.f32.f16 %1, h, %4;\n\t}"
      : "=f"(a), "=f"(b)
      : "r"(hi), "f"(x), "f"(y));
  lo = h2_bits(__floats2half2_rn(-a, -b));
}

// (x & m) | o as one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(m), "r"(o));
  return d;
}

// The codes in nibbles 0..3 of both halves of x as exact signed integers:
// 0x6400 | c is 1024 + c in f16, and 0x6400 | 16 c is 1024 + 16 c.
__device__ __forceinline__ void codes4(uint32_t x, uint32_t* y) {
  const __half2 m8 = __float2half2_rn(-1032.0f), m72 = __float2half2_rn(-72.0f),
                r16 = __float2half2_rn(0.0625f);
  const uint32_t z = x >> 8;
  y[0] = h2_bits(__hadd2(bits_h2(and_or(x, 0x000f000fu, 0x64006400u)), m8));
  y[1] = h2_bits(__hfma2(bits_h2(and_or(x, 0x00f000f0u, 0x64006400u)), r16, m72));
  y[2] = h2_bits(__hadd2(bits_h2(and_or(z, 0x000f000fu, 0x64006400u)), m8));
  y[3] = h2_bits(__hfma2(bits_h2(and_or(z, 0x00f000f0u, 0x64006400u)), r16, m72));
}

// The line of items. Request r: n tokens in J column tiles per head tile.
struct KvReq {
  int r, t0, n, len;  // request, first token, tokens, positions
  long long base;     // weight of column tile j: base + (j + 1) * tpt
  long long J;
};
__device__ __forceinline__ KvReq kv_req(const Kv4AttnParams& p, int r) {
  KvReq q;
  q.r = r;
  const int a = p.q_start[r], b = p.q_start[r + 1];
  const bool ok = a >= 0 && b <= p.n_tokens && a < b;  // a valid run of tokens
  q.t0 = ok ? a : 0;
  q.n = ok ? b - a : 0;
  if (q.n < p.n_lo || q.n > p.n_hi) q.n = 0;  // another kernel's
  q.len = max(p.lens[r], 0);
  const int prior = q.len - q.n;
  q.base = (prior > 0 ? prior : 0) + p.extra;
  q.J = (q.n + p.tpt - 1) / p.tpt;
  return q;
}
// Weight of column tiles 0 .. j - 1.
__device__ __forceinline__ long long kv_cum(const KvReq& q, int tpt, long long j) {
  return j * q.base + (long long)tpt * (j * (j + 1) / 2);
}

// One item: tokens [tok0, tok0 + ntok) of a request for the heads [h0, h0 +
// nhead), at [start, start + w) on the line.
struct KvItem {
  KvReq rq;
  int h;        // head tile
  long long j;  // column tile
  long long start, w;
  int kvh, h0, nhead, tok0, ntok, prior, lim_max;
  long long cap;
  long long x0, x1;  // the part of it that this warp (or CTA) takes
};
__device__ __forceinline__ void kv_item_set(const Kv4AttnParams& p, KvItem& it) {
  const int G = p.nh / p.nkv, hg = it.h % p.hgroups;
  it.w = it.rq.base + (it.j + 1) * p.tpt;
  it.kvh = it.h / p.hgroups;
  it.h0 = it.kvh * G + hg * p.gsz;
  it.nhead = min(p.gsz, G - hg * p.gsz);
  it.tok0 = (int)(it.j * p.tpt);
  it.ntok = min(p.tpt, it.rq.n - it.tok0);
  it.prior = it.rq.len - it.rq.n;
  // positions of the table row (tile ends stay inside 31 bits)
  it.cap = min((long long)p.table_stride << p.page_shift, 0x7fffff00ll);
  // positions that the last token sees
  const long long lim = min((long long)it.prior + it.tok0 + it.ntok, it.cap);
  it.lim_max = lim > 0 ? (int)lim : 0;
}
// The item at u, in the request r that starts at `start` on the line.
__device__ __forceinline__ void kv_item_at(const Kv4AttnParams& p, KvItem& it, int r,
                                           long long start, long long u) {
  it.rq = kv_req(p, r);
  const long long W = kv_cum(it.rq, p.tpt, it.rq.J), off = u - start;
  it.h = (int)(off / W);
  const long long x = off - it.h * W;
  long long lo = 0, hi = it.rq.J;
  while (hi - lo > 1) {
    const long long mid = (lo + hi) >> 1;
    if (kv_cum(it.rq, p.tpt, mid) <= x)
      lo = mid;
    else
      hi = mid;
  }
  it.j = lo;
  it.start = start + it.h * W + kv_cum(it.rq, p.tpt, lo);
  kv_item_set(p, it);
}
// The next item on the line; false behind the last one.
__device__ __forceinline__ bool kv_item_next(const Kv4AttnParams& p, KvItem& it) {
  it.start += it.w;
  if (++it.j == it.rq.J) {
    it.j = 0;
    if (++it.h == p.nkv * p.hgroups) {
      it.h = 0;
      int r = it.rq.r;
      do {
        if (++r >= p.n_req) return false;
        it.rq = kv_req(p, r);
      } while (it.rq.J == 0);
    }
  }
  kv_item_set(p, it);
  return true;
}

// The tcgen05 kernel (kv4_attend_umma.cu) and its workspace.
constexpr int kKvUmmaRows = 128;  // (token, head) rows of a tile
size_t kv4_umma_workspace(size_t head_dim);
// Sets the fields of p that the join reads.
minq_status launch_kv4_umma(Kv4AttnParams& p, void* workspace, cudaStream_t s);
// Its status word, as take_kv4_status has its own.
minq_status take_kv4_umma_status(int* v);

}  // namespace minq
