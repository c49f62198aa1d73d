// Causal attention over the paged 4-bit cache for the prompt chunks of a step,
// on the 5th-generation tensor cores: the requests with enough new tokens to
// fill a good part of 128 (token, query head) rows. kv4_attend.cu has the
// formulas, the line of items and the kernel for all other requests.
//
// A tile is 128 rows of one kv head x 64 positions. Its K and V rows come by
// bulk copies of 16 rows of one page, are turned from codes into values once
// for all 128 rows, and every product is made of f16 parts with f32
// accumulation:
//   q f = Qh + Ql,  k f_t = Kh + Kl,  p 2^10 = Ph + Pl,  v f' = Vh + Vl
//   S = Ql Kh + Qh Kl + Qh Kh,      O = Pl Vh + Ph Vl + Ph Vh,
// 22 bits of each factor; the dropped low x low term is below 2^-23 of the
// product. f, f_t, f' are powers of two per query row, per position and per
// tile that put the largest value (of K and V: the largest scale) into the
// upper part of f16's range; they are taken out again in f32, so no size of
// the inputs matters. A tile's O is summed by itself and added to the row's
// sum in registers with f32's rounding: the tensor core truncates, always
// towards zero, and over thousands of positions that would show.
//
// One CTA per SM, four roles that work on different tiles at the same time:
//   warps 0-3    softmax: thread = row = TMEM lane. One pass over S in steps of
//                16 columns: moves the maximum only when a weight would exceed
//                2^4 (and then scales what it has written), writes P over S.
//   warps 4-7    sums: thread = row. Writes Qh and Ql, then acc = acc * a + O.
//   warps 8-15   values: raw tile -> Kh Kl, Vh Vl in 128-byte swizzled tiles.
//   warps 17-19  bulk copies, K's scales, V's scales.
//   warp 16      one thread issues the MMAs: S of the next tile, then P V.
// K and V tiles are double buffered; TMEM: Qh Ql, 4 S, O (512 columns at head_dim
// 128). P takes the place of its S, and MMAs of other accumulators and shapes may run
// in another order than they were issued in: S of tile g + 3 and later only may
// overwrite P of tile g, since P V of g + 1 waits until O of g has been read. (Two
// places of S and two of O, where S of g + 2 has to wait for P V of g by itself, took
// 259 us for the case below.)
// The order of dimensions inside S's contraction and of positions inside
// P V's is free, so both are chosen for the code layout and for stores without
// bank conflicts (q_dim and the packing of P follow them).
//
// Measured: 4 requests, two of them with 512 new tokens behind up to 3584, 32 query
// and 8 kv heads of 128 (61 GFLOP of useful products): 220 us, 0.28 PFLOP/s, three
// f16 products each, so 0.83 PFLOP/s of the tensor cores' work; the mma.sync kernel
// takes 670 us. A tile costs an SM 3,300 cycles, of which the tensor cores need
// 1,400; softmax (2,700 of its warps' time) and values (2,200) run beside them but
// share the issue slots, which are used in half of the cycles. The roles' loops are
// kept short (one step of 16 columns, not four unrolled): together they have to fit
// the instruction cache, and unrolled they took 352 us. 24 bytes spill at head_dim 128. Eight softmax warps that
// took turns at the tiles, with fewer registers each, took 234 us.
//
// A value scale that is not finite would reach rows that do not see its
// position (0 x inf): it is left out of the tile and makes the block of the
// rows that see it NaN.
#include <limits.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4_attend.cuh"
#include "pipeline.cuh"

namespace minq {

namespace {

__device__ int g_kv4_umma_status;  // see g_kv4_status

constexpr int kUTile = 64;       // positions per tile
constexpr int kUSoft = 4, kUSum = 4, kUVal = 8;  // warps of the roles
constexpr int kUThreads = 32 * (kUSoft + kUSum + kUVal + 4);
// Registers a thread: 96 at the launch (640 threads), then by role (each a
// whole number of warpgroups): 120 + 176 + 2 x 64 + 56 <= 5 x 96.
constexpr int kURegSoft = 120, kURegSum = 176, kURegVal = 64, kURegMma = 56;
static_assert(kURegSoft + kURegSum + 2 * kURegVal + kURegMma <= 5 * 96, "registers");
static_assert(kURegSoft >= 96 && kURegSum >= 96 && kURegVal <= 96 && kURegMma <= 96,
              "setmaxnreg.inc may not lower the count, .dec not raise it");
constexpr int kUValThreads = 32 * kUVal;
constexpr int kUExtra = 256;     // an item's start and end, in positions
constexpr int kUMinPiece = 512;  // smallest piece of the line per CTA
constexpr int kURaw = 4;         // raw tiles in flight
constexpr int kUScores = 4;      // places for S and P

template <int HD>
struct UmGeom {
  static constexpr int NB = HD / 32, ROW = NB * kQ4Bytes;
  static constexpr int RUN = 16 * ROW;         // 16 positions of K or V
  static constexpr int RAW = 2 * 4 * RUN;      // a raw tile: K, V
  static constexpr int KT = kUTile * HD * 2;   // Kh, Kl, Vh or Vl
  static constexpr int K = 0, V = 4 * KT, R = 8 * KT, CTL = R + kURaw * RAW;
  // TMEM columns
  static constexpr int QH = 0, QL = HD / 2, S = HD, O = HD + kUScores * kUTile;
  static_assert(O + HD <= 512, "tensor memory");
};

struct UmCtl {
  float2 corr[4][kKvUmmaRows];  // per row: the maximum used; bit b: block b becomes NaN
  float2 ml[kKvUmmaRows];
  float cn[kKvUmmaRows];        // scores to log2 units
  float kinv[8][kUTile];        // 1 / f_t of K
  // scales of the positions that exist (0: not; V: or not finite) as two f16 parts
  uint32_t kscale[kURaw][kUTile * 4], vscale[kURaw][kUTile * 4];
  float vinv[16];               // 2^-10 / f' of V
  int ok[8];                    // runs of 16 positions that exist
  uint32_t bad[8][8];           // not finite value scales: word and bit of (position * NB + block)
  int raw_ok[kURaw];
  uint64_t raw_full[kURaw], raw_free[kURaw], scale_full[kURaw];
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2];
  uint64_t o_free, q_full, drain;
  uint32_t tmem;
  int abort, more, req;
  long long req_start, red[kUThreads / 32];
  KvItem item[2];  // this one and the next
};

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// Descriptor of a K-major tile in the 128-byte swizzle layout, 8-row groups
// 1024 bytes apart: the low word (the address, which moves) and the high one.
__device__ __forceinline__ uint32_t sw128_lo(uint32_t saddr) {
  return ((saddr & 0x3FFFFu) >> 4) | (1u << 16);
}
constexpr uint32_t kSw128Hi = (1024u >> 4) | (1u << 14) | (2u << 29);
// 16-byte chunk c (0..7) of row r.
__device__ __forceinline__ uint32_t sw_chunk(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}
// D (+)= A (TMEM) x B, kind::f16: A and B f16, K-major, D f32, M = 128, N = n;
// by the elected lane. The warp runs this together, so that addresses and
// descriptors stay in uniform registers.
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d, uint32_t a, uint32_t b_lo, int n,
                                       uint32_t acc) {
  const uint32_t idesc = (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "n"(kSw128Hi), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}"
      : "=r"(on));
  return on;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
// 32 lanes x 16 columns of 32-bit words (this warp's lane quarter).
__device__ __forceinline__ void tm_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Wait for this thread's TMEM loads; the values pass through the asm so that no
// use of them is scheduled before the wait.
__device__ __forceinline__ void tm_wait_ld16(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void sts16(uint32_t a, const uint32_t* v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3])
               : "memory");
}

// Bounded wait: false after 1 s (status word and the CTA's abort flag set) or
// once another thread gave up.
__device__ __forceinline__ bool um_wait_long(uint64_t* bar, uint32_t parity, int* abort) {
  const uint64_t t0 = global_timer_ns();
  for (;;) {
    if (mbar_try_wait_sleep(bar, parity, 1000u)) return true;
    if (*reinterpret_cast<volatile int*>(abort)) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      *reinterpret_cast<volatile int*>(abort) = 1;
      atomicOr(&g_kv4_umma_status, kDeviceTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ bool um_wait1(uint64_t* bar, uint32_t parity, int* abort) {
  return mbar_try_wait_sleep(bar, parity, 20000u) || um_wait_long(bar, parity, abort);
}
// The same for a whole warp: its lanes go on or give up together.
__device__ __forceinline__ bool um_wait(uint64_t* bar, uint32_t parity, int* abort) {
  return __all_sync(0xffffffffu, um_wait1(bar, parity, abort));
}

// f (a power of two) that puts values of at most m, m normal, into [2^11, 2^12).
__device__ __forceinline__ uint32_t up_exponent(float m) {
  const int e = 265 - (int)(__float_as_uint(m) >> 23);
  return (uint32_t)min(e, 253);
}

// A scale d as two f16 parts, high in the low half word.
__device__ __forceinline__ uint32_t scale_parts(float d) {
  const __half h = __float2half_rn(d);
  return h2_bits(__halves2half2(h, __float2half_rn(d - __half2float(h))));
}
// Two values, code y times scale dh + dl, as two f16 parts: the high one
// rounded, what that leaves out (exact) plus y dl the low one. Within 2^-23.
// (Scales whose high part has 8 bits need no remainder, one instruction less
// of three, but leave 2^-20.)
__device__ __forceinline__ void value_parts(uint32_t y, uint32_t dh, uint32_t dl, uint32_t& hi,
                                            uint32_t& lo) {
  const __half2 h = __hmul2_rn(bits_h2(y), bits_h2(dh));
  const __half2 rest = __hfma2(bits_h2(y), bits_h2(dh), __hneg2(h));
  hi = h2_bits(h);
  lo = h2_bits(__hfma2(bits_h2(y), bits_h2(dl), rest));
}
// x = x * y, x = x * y + z, x + y on two f32 at once.
__device__ __forceinline__ void mul_f2(float* x, float y0, float y1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x[0]), "+f"(x[1])
      : "f"(y0), "f"(y1));
}
__device__ __forceinline__ void fma_f2(float* x, float y, float z0, float z1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\t"
      "mov.b64 c, {%3, %4};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x[0]), "+f"(x[1])
      : "f"(y), "f"(z0), "f"(z1));
}
__device__ __forceinline__ void fma_acc2(float* x, const float* y, float z) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "mov.b64 c, {%4, %4};\n\tfma.rn.f32x2 a, b, c, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x[0]), "+f"(x[1])
      : "f"(y[0]), "f"(y[1]), "f"(z));
}
__device__ __forceinline__ void add_f2(float* x, const float* y) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x[0]), "+f"(x[1])
      : "f"(y[0]), "f"(y[1]));
}

// S's column (K's row in its tile) of position r of the tile: the place that
// V's tile gives r in P V's contraction, so P can take S's place in TMEM.
__device__ __forceinline__ int s_column(int r) { return (r & 7) * 8 + (r >> 3); }

// The tiles of an item that this CTA takes.
struct UmTiles {
  int first, n;
};
__device__ __forceinline__ UmTiles um_tiles(const KvItem& it) {
  const int all = (it.lim_max + kUTile - 1) / kUTile;
  auto tile_at = [](long long x) { return x > kUExtra ? (x - kUExtra + kUTile - 1) / kUTile : 0; };
  const int a = (int)min((long long)tile_at(it.x0), (long long)all);
  const int b = it.x1 == it.w ? all : (int)min((long long)tile_at(it.x1), (long long)all);
  return {a, max(b - a, 0)};
}

// Copies: one warp, whose lanes 0..7 take a run of K or V each. Returns the number
// of tiles issued.
template <int HD>
__device__ __forceinline__ int um_copies(const Kv4AttnParams& p, UmCtl& c, const KvItem& it, uint8_t* sm,
                                         UmTiles tl, uint32_t g0) {
  using GM = UmGeom<HD>;
  const int lane = threadIdx.x & 31, run = lane & 3, lim_max = it.lim_max;
  const uint8_t* side =
      (lane & 4 ? p.v_pages : p.k_pages) + ((size_t)it.kvh << p.page_shift) * GM::ROW;
  const size_t page_bytes = ((size_t)p.nkv << p.page_shift) * GM::ROW;
  const int* tab = p.table + (size_t)it.rq.r * p.table_stride;
  auto load_id = [&](int i) {  // checked where it is used, when it has come
    const int pos = (tl.first + i) * kUTile + 16 * run;
    return lane < 8 && i < tl.n && pos < lim_max ? tab[pos >> p.page_shift] : -1;
  };
  int id = load_id(0), i = 0;
  for (; i < tl.n; ++i) {
    const int id_next = load_id(i + 1);
    const uint32_t g = g0 + i, st = g % kURaw;
    if (g >= kURaw && !um_wait(&c.raw_free[st], (g / kURaw - 1) & 1, &c.abort)) break;
    const bool on = id >= 0 && id < p.n_pages;
    const uint32_t have = __ballot_sync(0xffffffffu, on) & 15u;
    if (lane == 0) {
      c.raw_ok[st] = (int)have;
      if (have)
        mbar_arrive_expect_tx(&c.raw_full[st], 2 * __popc(have) * GM::RUN + p.stall);
      else
        mbar_arrive(&c.raw_full[st]);
    }
    __syncwarp();  // the bytes are expected before they can come
    if (on) {
      const int row = ((tl.first + i) * kUTile + 16 * run) & ((1 << p.page_shift) - 1);
      bulk_g2s(sm + GM::R + st * GM::RAW + (lane >> 2) * 4 * GM::RUN + run * GM::RUN,
               side + (size_t)id * page_bytes + (size_t)row * GM::ROW, GM::RUN, &c.raw_full[st]);
    }
    id = id_next;
  }
  return i;
}

// Scales: one warp for K's, one for V's.
template <int HD, bool V>
__device__ __forceinline__ void um_scales(UmCtl& c, const KvItem& it, const uint8_t* sm, UmTiles tl,
                                          uint32_t g0) {
  using GM = UmGeom<HD>;
  constexpr int NB = GM::NB, N = kUTile * NB / 32;
  const int lane = threadIdx.x & 31, lim_max = it.lim_max;
  for (int i = 0; i < tl.n; ++i) {
    const uint32_t g = g0 + i, st = g % kURaw;
    if (!um_wait(&c.raw_full[st], (g / kURaw) & 1, &c.abort)) return;
    const int pos0 = (tl.first + i) * kUTile, ok = c.raw_ok[st];
    const uint8_t* raw = sm + GM::R + st * GM::RAW + (V ? 4 * GM::RUN : 0);
    auto scale = [&](int j) {
      const int x = lane + 32 * j, row = x / NB;
      const bool there = ((ok >> (row >> 4)) & 1) && pos0 + row < lim_max;
      return there ? *reinterpret_cast<const float*>(raw + x * kQ4Bytes) : 0.0f;
    };
    if (V) {
      uint32_t top = 0;
#pragma unroll 2
      for (int j = 0; j < N; ++j) {
        const float d = scale(j);
        const bool fin = fabsf(d) < INFINITY;
        const uint32_t bad = __ballot_sync(0xffffffffu, !fin);
        if (lane == 0) c.bad[g & 7][j] = bad;
        top = max(top, fin ? __float_as_uint(fabsf(d)) : 0u);
      }
      const uint32_t e = up_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, top)));
      if (lane == 0) {
        c.vinv[g & 15] = __uint_as_float((254u - e) << 23) * 0.0009765625f;
        c.ok[g & 7] = ok;
      }
#pragma unroll 2
      for (int j = 0; j < N; ++j) {
        const float d = scale(j);
        c.vscale[st][lane + 32 * j] =
            scale_parts(fabsf(d) < INFINITY ? d * __uint_as_float(e << 23) : 0.0f);
      }
    } else {
#pragma unroll 2
      for (int j = 0; j < N; ++j) {
        const float d = scale(j);
        float m = fabsf(d) < INFINITY ? fabsf(d) : 0.0f;
#pragma unroll
        for (int o = 1; o < NB; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t e = up_exponent(m);
        const int x = lane + 32 * j;
        c.kscale[st][x] = scale_parts(d * __uint_as_float(e << 23));
        if (x % NB == 0) c.kinv[g & 7][s_column(x / NB)] = __uint_as_float((254u - e) << 23);
      }
    }
    mbar_arrive(&c.scale_full[st]);
  }
}

// Values role: the item's tiles, from codes and scales to f16 parts.
template <int HD>
__device__ __forceinline__ void um_values(UmCtl& c, const uint8_t* sm, uint32_t base, UmTiles tl,
                                          uint32_t g0) {
  using GM = UmGeom<HD>;
  constexpr int NB = GM::NB, ROW = GM::ROW;
  const int dt = threadIdx.x - 32 * (kUSoft + kUSum), lane = dt & 31;
  // K: block kb of position kr; V: positions pg + 8 i, four dimensions of block
  // vb. With head_dim 64 half of the threads have K, the other half V.
  const bool k_on = HD == 128 || dt < 128, v_on = HD == 128 || dt >= 128;
  const int kt = HD == 128 ? dt : dt & 127, kr = kt / NB, kb = kt % NB;
  const int pg = kt & 7, dq = kt >> 3, vb = dq >> 3;
  for (int i = 0; i < tl.n; ++i) {
    const uint32_t g = g0 + i, par = g >> 1, st = g & 1, rs = g % kURaw;
    if (!um_wait(&c.raw_full[rs], (g / kURaw) & 1, &c.abort) ||
        !um_wait(&c.scale_full[rs], (g / kURaw) & 1, &c.abort))
      return;
    const uint8_t* rk = sm + GM::R + rs * GM::RAW;
    const uint8_t* rv = rk + 4 * GM::RUN;
    const uint32_t d = c.kscale[rs][kt];
    // S of tile g - 2 has read this buffer
    if (g >= 2 && !um_wait(&c.s_full[st], (par - 1) & 1, &c.abort)) return;
    if (k_on) {
      const uint32_t dh = __byte_perm(d, d, 0x1010), dl = __byte_perm(d, d, 0x3232);
      const uint32_t tile = base + GM::K + st * 2 * GM::KT + (kb >> 1) * kUTile * 128;
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {
        uint32_t y[4], hi[4], lo[4];
        codes4(*reinterpret_cast<const uint32_t*>(rk + kt * kQ4Bytes + 4 + 4 * x), y);
        // blocks 2, 3: chunks in another order, against bank conflicts
        const uint32_t at = tile + sw_chunk(s_column(kr), 4 * (kb & 1) + (x ^ (kb & 2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) value_parts(y[e], dh, dl, hi[e], lo[e]);
        sts16(at, hi);
        sts16(at + GM::KT, lo);
      }
    }
    fence_async_smem();
    mbar_arrive(&c.k_full[st]);
    uint32_t hi[4][4], lo[4][4];  // [dimension][pair of positions]
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r0 = pg + 16 * q;
      const uint8_t* v0 = rv + r0 * ROW + vb * kQ4Bytes + 4 + 2 * (dq & 7);
      const uint32_t x0 = *reinterpret_cast<const uint16_t*>(v0);
      const uint32_t x1 = *reinterpret_cast<const uint16_t*>(v0 + 8 * ROW);
      const uint32_t d0 = c.vscale[rs][r0 * NB + vb], d1 = c.vscale[rs][(r0 + 8) * NB + vb];
      const uint32_t dh = __byte_perm(d0, d1, 0x5410), dl = __byte_perm(d0, d1, 0x7632);
      uint32_t y[4];
      codes4(__byte_perm(x0, x1, 0x5410), y);
#pragma unroll
      for (int e = 0; e < 4; ++e) value_parts(y[e], dh, dl, hi[e][q], lo[e][q]);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&c.raw_free[rs]);
    // P V of tile g - 2 has read this buffer
    if (g >= 2 && !um_wait(&c.pv_done[st], (par - 1) & 1, &c.abort)) return;
    if (v_on) {
      const uint32_t tile = base + GM::V + st * 2 * GM::KT;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = tile + sw_chunk(4 * dq + e, pg);
        sts16(at, hi[e]);
        sts16(at + GM::KT, lo[e]);
      }
    }
    fence_async_smem();
    mbar_arrive(&c.v_full[st]);
  }
}

// First of the eight dimensions d of chunk x of S's contraction (4 columns of
// Q, d + e and d + e + 4 in column e): see um_values.
template <int HD>
__device__ __forceinline__ constexpr int q_dim(int x) {
  return (x >> 2) * 32 + 8 * ((x & 3) ^ ((x >> 2) & 2));
}

// Softmax role.
template <int HD>
__device__ __forceinline__ void um_softmax(const Kv4AttnParams& p, UmCtl& c, const KvItem& it,
                                           uint32_t tmem, UmTiles tl, uint32_t g0) {
  using GM = UmGeom<HD>;
  constexpr int NB = GM::NB;
  const int row = threadIdx.x;
  const uint32_t tlane = tmem + ((uint32_t)(row & ~31) << 16);
  const int ct = row / p.gsz, ch = row - ct * p.gsz;
  const bool on = ct < it.ntok && ch < it.nhead;
  long long lim64 = on ? (long long)it.prior + it.tok0 + ct + 1 : 0;
  lim64 = lim64 < 0 ? 0 : lim64 < it.cap ? lim64 : it.cap;
  const int lim = (int)lim64;
  float m = -INFINITY, l = 0.0f;
  for (int i = 0; i < tl.n; ++i) {
    const uint32_t g = g0 + i, st = g & 1;
    const uint32_t place = tlane + GM::S + g % kUScores * kUTile;
    if (!um_wait(&c.s_full[st], (g >> 1) & 1, &c.abort)) return;
    fence_after();
    const int pos0 = (tl.first + i) * kUTile, ok = c.ok[g & 7];
    const float cn = c.cn[row];
    const bool all = __all_sync(0xffffffffu, ok == 15 && pos0 + kUTile <= lim);
    float sum[2] = {0.0f, 0.0f};
    // 16 columns of S; column e of part x is position 2 x + e / 8 + 8 (e mod 8)
    auto process = [&](int x, float* s) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 k = *reinterpret_cast<const float4*>(&c.kinv[g & 7][16 * x + j]);
        mul_f2(s + j, k.x, k.y);
        mul_f2(s + j + 2, k.z, k.w);
      }
      if (!all) {
        const int left = lim - pos0 - 2 * x;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((ok >> ((e & 7) >> 1)) & 1) || (e >> 3) + 8 * (e & 7) >= left) s[e] = -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top = top == -INFINITY ? top : top * cn;
      const bool more = top > m + 4.0f;  // also the first that is seen
      if (__any_sync(0xffffffffu, more)) {
        // the maximum moves by whole numbers, so the parts before are scaled exactly
        const int k = !more ? 0 : m == -INFINITY ? 127 : (int)fminf(ceilf(top - m), 127.0f);
        const float b = k == 127 ? 0.0f : __uint_as_float((uint32_t)(127 - k) << 23);
        if (more) m = m == -INFINITY ? ceilf(top) : m + ceilf(top - m);
        l *= b;
        sum[0] *= b;
        sum[1] *= b;
        const int k1 = min(k, 14), k2 = min(k - k1, 24);
        const __half2 f1 = __float2half2_rn(__uint_as_float((uint32_t)(127 - k1) << 23)),
                      f2 = __float2half2_rn(__uint_as_float((uint32_t)(127 - k2) << 23));
        // the parts that are read back were stored asynchronously (by the steps
        // before and by earlier moves), and a load may pass a store
        tm_wait_st();
        for (int y = 0; y < x; ++y) {
          float v[16];
          uint32_t part[16];
          tm_ld16(place + 16 * y, v);
          tm_wait_ld16(v);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            part[e] = h2_bits(__hmul2(__hmul2(bits_h2(__float_as_uint(v[e])), f1), f2));
          tm_st16(place + 16 * y, part);
        }
      }
      const float off = m == -INFINITY ? 0.0f : 10.0f - m;
      uint32_t part[16];  // eight columns of high, eight of low parts in S's place
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        fma_f2(s + e, cn, off, off);
        s[e] = ex2(s[e]);
        s[e + 1] = ex2(s[e + 1]);
        add_f2(sum, s + e);
        split2(s[e], s[e + 1], part[e / 2], part[e / 2 + 8]);
      }
      tm_st16(place + 16 * x, part);
    };
#pragma unroll 1
    for (int x = 0; x < kUTile / 16; ++x) {
      float s[16];
      tm_ld16(place + 16 * x, s);
      tm_wait_ld16(s);
      process(x, s);
    }
    l += sum[0] + sum[1];
    uint32_t nan = 0, any = 0;
#pragma unroll
    for (int x = 0; x < 2 * NB; ++x) any |= c.bad[g & 7][x];
    if (any) {
      constexpr int PER = 32 / NB;  // positions of a word
      for (int x = 0; x < kUTile / PER; ++x)
        for (int b = 0; b < 32; ++b)
          if (((c.bad[g & 7][x] >> b) & 1) && pos0 + x * PER + b / NB < lim) nan |= 1u << (b % NB);
    }
    c.corr[g & 3][row] = make_float2(m, __uint_as_float(nan));
    tm_wait_st();
    fence_before();
    mbar_arrive(&c.p_full[st]);
  }
  c.ml[row] = make_float2(l == 0.0f ? -3.0e38f : m, l * 0.0009765625f);
}

// The warp that issues the MMAs (one lane of it does).
template <int HD>
__device__ __forceinline__ void um_mma(UmCtl& c, uint32_t tmem, uint32_t base, UmTiles tl, uint32_t g0,
                                       uint32_t items) {
  using GM = UmGeom<HD>;
  const uint32_t on = elect_lane();
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  g0 = __shfl_sync(0xffffffffu, g0, 0);
  const int n = __shfl_sync(0xffffffffu, tl.n, 0);
  if (!um_wait(&c.q_full, items & 1, &c.abort)) return;
  auto scores = [&](int i) {
    const uint32_t g = g0 + i, st = g & 1, d = tmem + GM::S + g % kUScores * kUTile;
    const uint32_t kt = sw128_lo(base + GM::K + st * 2 * GM::KT);
    if (!um_wait(&c.k_full[st], (g >> 1) & 1, &c.abort)) return false;
    fence_after();
    // the small parts first: what the accumulation truncates next to them is nothing
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
      for (int j = 0; j < HD / 16; ++j)
        mma_ts(on, d, tmem + (part == 0 ? GM::QL : GM::QH) + 8 * j,
               kt + (((part == 1 ? GM::KT : 0) + (j >> 2) * kUTile * 128 + (j & 3) * 32) >> 4), kUTile,
               part | j);
    if (on) mma_commit(&c.s_full[st]);
    __syncwarp();
    return true;
  };
  if (n > 0 && !scores(0)) return;
  for (int i = 0; i < n; ++i) {
    if (i + 1 < n && !scores(i + 1)) return;
    const uint32_t g = g0 + i, st = g & 1, par = (g >> 1) & 1;
    const uint32_t a = tmem + GM::S + g % kUScores * kUTile, d = tmem + GM::O;
    const uint32_t vt = sw128_lo(base + GM::V + st * 2 * GM::KT);
    if (!um_wait(&c.v_full[st], par, &c.abort)) return;
    if (g >= 1 && !um_wait(&c.o_free, (g - 1) & 1, &c.abort)) return;
    if (!um_wait(&c.p_full[st], par, &c.abort)) return;
    fence_after();
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
      for (int j = 0; j < kUTile / 16; ++j)
        mma_ts(on, d, a + (part == 0 ? 8 : 0) + 16 * j, vt + (((part == 1 ? GM::KT : 0) + j * 32) >> 4), HD,
               part | j);
    if (on) mma_commit(&c.pv_done[st]);
    __syncwarp();
  }
}

// Sums role, up to the item's outputs.
template <int HD>
__device__ __forceinline__ void um_sums(const Kv4AttnParams& p, UmCtl& c, const KvItem& it, uint32_t tmem,
                                        UmTiles tl, uint32_t g0) {
  using GM = UmGeom<HD>;
  const int row = threadIdx.x - 32 * kUSoft;
  const uint32_t col = tmem + ((uint32_t)(row & ~31) << 16) + GM::O;
  const int ct = row / p.gsz, ch = row - ct * p.gsz;
  const bool on = ct < it.ntok && ch < it.nhead;
  float acc[HD];
  // the row of q, all of it in flight at once, as f16 parts into TMEM
  {
    const float* q = p.q + (size_t)(it.rq.t0 + it.tok0 + (on ? ct : 0)) * p.q_stride +
                     (size_t)(it.h0 + (on ? ch : 0)) * HD;
    if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
      for (int d = 0; d < HD; d += 4)
        *reinterpret_cast<float4*>(acc + d) = *reinterpret_cast<const float4*>(q + d);
    } else {
#pragma unroll
      for (int d = 0; d < HD; ++d) acc[d] = q[d];
    }
    float m = 0.0f;
#pragma unroll
    for (int d = 0; d < HD; ++d) {
      if (!on) acc[d] = 0.0f;
      m = fmaxf(m, fabsf(acc[d]));
    }
    const int ex = min(max((int)(__float_as_uint(m) >> 23), 24), 254);
    float f = __uint_as_float((uint32_t)(264 - ex) << 23);
    const float cn = fabsf(p.scale) * 1.4426950408889634f * (1.0f / f);
    c.cn[row] = cn == 0.0f ? 1.4e-45f : cn;  // -inf stays masked
    if (p.scale < 0.0f) f = -f;
    const uint32_t tq = tmem + ((uint32_t)(row & ~31) << 16);
#pragma unroll
    for (int x0 = 0; x0 < HD / 2; x0 += 16) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int d = q_dim<HD>((x0 + x) / 4) + (x & 3);
        split2(acc[d] * f, acc[d + 4] * f, hi[x], lo[x]);
      }
      tm_st16(tq + GM::QH + x0, hi);
      tm_st16(tq + GM::QL + x0, lo);
    }
    tm_wait_st();
    fence_before();
    mbar_arrive(&c.q_full);
  }
  float M = -3.0e38f;  // acc is relative to the maximum of the last tile
#pragma unroll
  for (int d = 0; d < HD; ++d) acc[d] = 0.0f;
  for (int i = 0; i < tl.n; ++i) {
    const uint32_t g = g0 + i, st = g & 1;
    if (!um_wait(&c.pv_done[st], (g >> 1) & 1, &c.abort)) break;
    fence_after();
    const float2 cr = c.corr[g & 3][row];
    const float f = c.vinv[g & 15];
    const bool more = cr.x > M;
    if (__any_sync(0xffffffffu, more)) {
      const float a = more ? ex2(M - cr.x) : 1.0f;
      if (more) M = cr.x;
#pragma unroll
      for (int d = 0; d < HD; d += 2) mul_f2(acc + d, a, a);
    }
    const uint32_t nan = __float_as_uint(cr.y);
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += 16) {
      float o[16];
      tm_ld16(col + d0, o);
      tm_wait_ld16(o);
      const float fn = (nan >> (d0 / 32)) & 1 ? NAN : f;
#pragma unroll
      for (int d = 0; d < 16; d += 2) fma_acc2(acc + d0 + d, o + d, fn);
    }
    fence_before();
    mbar_arrive(&c.o_free);
  }
  __syncthreads();
  if (on) {
    const float2 ml = c.ml[row];
    const bool whole = it.x0 == 0 && it.x1 == it.w;
    const size_t at = ((size_t)blockIdx.x * 2 + (it.x0 > 0 ? 0 : 1)) * kKvUmmaRows + row;
    const float r = !whole ? 1.0f : ml.y != 0.0f ? 1.0f / ml.y : 0.0f;
    float* dst = whole ? p.out + (size_t)(it.rq.t0 + it.tok0 + ct) * p.out_stride +
                             (size_t)(it.h0 + ch) * HD
                       : p.part_o + at * HD;
    if (!whole) *reinterpret_cast<float2*>(p.part_ml + at * 2) = ml;
    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
      for (int d = 0; d < HD; d += 4)
        *reinterpret_cast<float4*>(dst + d) =
            make_float4(acc[d] * r, acc[d + 1] * r, acc[d + 2] * r, acc[d + 3] * r);
    } else {
#pragma unroll
      for (int d = 0; d < HD; ++d) dst[d] = acc[d] * r;
    }
  }
}

// Thread 0, when the item's tiles are done: what the join has to know of it.
__device__ __forceinline__ void um_record(const Kv4AttnParams& p, const KvItem& it, long long per) {
  if (it.x0 != 0 || it.x1 == it.w) return;  // starts before, or is whole
  KvRec r{};
  r.r = it.rq.r;
  r.h = it.h;
  r.j = (int)it.j;
  r.a = blockIdx.x;
  r.n_first = r.parts = (int)((it.start + it.w - 1) / per) - (int)blockIdx.x + 1;
  p.rec[blockIdx.x] = r;
}

template <int HD>
__global__ void __launch_bounds__(kUThreads, 1) kv4_umma_kernel(const __grid_constant__ Kv4AttnParams p) {
  using GM = UmGeom<HD>;
  extern __shared__ uint8_t um_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(um_smem) + 1023u) & ~1023u;
  uint8_t* sm = um_smem + (base - smem_u32(um_smem));
  UmCtl& c = *reinterpret_cast<UmCtl*>(sm + GM::CTL);
  constexpr int kMmaWarp = kUSoft + kUSum + kUVal;

  // before the TMEM: a kernel before this one that still has to allocate its own
  // must not meet a CTA that holds all of it and waits
  pdl_wait();
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < kURaw; ++i) {
        mbar_init(&c.raw_full[i], 1);
        mbar_init(&c.raw_free[i], kUVal);
        mbar_init(&c.scale_full[i], 64);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&c.k_full[i], kUValThreads);
        mbar_init(&c.v_full[i], kUValThreads);
        mbar_init(&c.s_full[i], 1);
        mbar_init(&c.p_full[i], 32 * kUSoft);
        mbar_init(&c.pv_done[i], 1);
      }
      mbar_init(&c.o_free, 32 * kUSum);
      mbar_init(&c.q_full, 32 * kUSum);
      mbar_init(&c.drain, 1);
      c.abort = 0;
      c.req = -1;
      mbar_fence_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&c.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the line: every warp weighs a run of the requests, and the warp in whose
  // run the CTA's piece starts looks for the request
  const int H = p.nkv * p.hgroups, seg = (p.n_req + kUThreads / 32 - 1) / (kUThreads / 32);
  const int r_lo = min(warp * seg, p.n_req), r_hi = min(r_lo + seg, p.n_req);
  auto weight = [&](int r) {
    const KvReq q = kv_req(p, r);
    return H * kv_cum(q, p.tpt, q.J);
  };
  long long mine = 0;
  for (int r = r_lo + lane; r < r_hi; r += 32) mine += weight(r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) c.red[warp] = mine;
  fence_before();
  __syncthreads();
  fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = c.tmem;
  long long total = 0, before = 0;
  for (int x = 0; x < kUThreads / 32; ++x) {
    if (x < warp) before += c.red[x];
    total += c.red[x];
  }
  long long per = (total + p.n_piece - 1) / p.n_piece;
  if (per < kUMinPiece) per = kUMinPiece;
  const long long c0 = per * blockIdx.x, c1 = min(c0 + per, total);
  if (c0 < c1 && before <= c0 && c0 < before + mine) {
    for (int r0 = r_lo; r0 < r_hi; r0 += 32) {
      const long long w = r0 + lane < r_hi ? weight(r0 + lane) : 0;
      long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const long long start = before + incl - w;
      if (start <= c0 && c0 < start + w) {
        c.req = r0 + lane;
        c.req_start = start;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (tid == 0) p.rec[blockIdx.x].parts = 0;
  __syncthreads();
  if (tid == 0) {
    c.more = c0 < c1 && c.req >= 0;
    if (c.more) {
      KvItem x;
      kv_item_at(p, x, c.req, c.req_start, c0);
      x.x0 = c0 - x.start;
      x.x1 = min(c1 - x.start, x.w);
      c.item[0] = x;
    }
  }
  __syncthreads();

  // the roles; between two items all of them meet twice: when the item's tiles
  // are done, and when the next item is known
  uint32_t g0 = 0;
  bool more = c.more;
  UmTiles tl{};
  int cur = 0;
  auto next = [&]() {
    g0 += tl.n;
    cur ^= 1;
    __syncthreads();
    more = c.more;
  };
  if (warp < kUSoft) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kURegSoft));
    while (more) {
      tl = um_tiles(c.item[cur]);
      um_softmax<HD>(p, c, c.item[cur], tmem, tl, g0);
      __syncthreads();
      if (tid == 0) {
        KvItem x = c.item[cur];
        um_record(p, x, per);
        c.more = x.start + x.w < c1 && !c.abort && kv_item_next(p, x);
        x.x0 = 0;
        x.x1 = min(c1 - x.start, x.w);
        c.item[cur ^ 1] = x;
      }
      next();
    }
    __syncthreads();
    if (warp == 0) {
      fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
  } else if (warp < kUSoft + kUSum) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kURegSum));
    while (more) {
      tl = um_tiles(c.item[cur]);
      um_sums<HD>(p, c, c.item[cur], tmem, tl, g0);
      next();
    }
    fence_before();
    __syncthreads();
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kURegVal));
    while (more) {
      tl = um_tiles(c.item[cur]);
      um_values<HD>(c, sm, base, tl, g0);
      __syncthreads();
      next();
    }
    __syncthreads();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kURegMma));
    uint32_t issued = 0;  // tiles whose copies this warp has issued
    for (uint32_t items = 0; more; ++items) {
      tl = um_tiles(c.item[cur]);
      if (warp == kMmaWarp) um_mma<HD>(c, tmem, base, tl, g0, items);
      if (warp == kMmaWarp + 1) issued = g0 + um_copies<HD>(p, c, c.item[cur], sm, tl, g0);
      if (warp == kMmaWarp + 2) um_scales<HD, false>(c, c.item[cur], sm, tl, g0);
      if (warp == kMmaWarp + 3) um_scales<HD, true>(c, c.item[cur], sm, tl, g0);
      __syncwarp();
      __syncthreads();
      next();
    }
    // after a wait that gave up, anyone's: let the MMAs and the copies end
    if (warp == kMmaWarp && c.abort) {
      if (elect_lane()) mma_commit(&c.drain);  // the lane that issues them
      __syncwarp();
      mbar_wait_timed(&c.drain, 0, &g_kv4_umma_status);
    }
    if (warp == kMmaWarp + 1 && c.abort)
      for (uint32_t g = issued > kURaw ? issued - kURaw : 0; g < issued; ++g)
        mbar_wait_timed(&c.raw_full[g % kURaw], (g / kURaw) & 1, &g_kv4_umma_status);
    __syncthreads();
  }
}

template <int HD>
minq_status launch_umma(const Kv4AttnParams& p, cudaStream_t s) {
  constexpr size_t smem = 1024 + UmGeom<HD>::CTL + sizeof(UmCtl);
  static_assert(smem <= 227 * 1024, "shared memory of the tcgen05 kernel");
  auto k = kv4_umma_kernel<HD>;
  MINQ_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(k), smem));
  MINQ_CUDA_TRY(launch_k(k, dim3(p.n_piece), dim3(kUThreads), smem, s, p));
  return MINQ_OK;
}

}  // namespace

size_t kv4_umma_workspace(size_t head_dim) {
  return (size_t)sm_count() * (2 * kKvUmmaRows * (head_dim + 2) * 4 + sizeof(KvRec));
}

minq_status launch_kv4_umma(Kv4AttnParams& p, void* workspace, cudaStream_t s) {
  const int G = p.nh / p.nkv;
  p.cols = kKvUmmaRows;
  p.gsz = G < kKvUmmaRows ? G : kKvUmmaRows;
  p.hgroups = (G + p.gsz - 1) / p.gsz;
  p.tpt = kKvUmmaRows / p.gsz;
  p.extra = kUExtra;
  p.n_piece = sm_count();
  p.rec = static_cast<KvRec*>(workspace);
  p.part_o = reinterpret_cast<float*>(p.rec + p.n_piece);
  p.part_ml = p.part_o + (size_t)p.n_piece * 2 * kKvUmmaRows * p.hd;
  return p.hd == 64 ? launch_umma<64>(p, s) : launch_umma<128>(p, s);
}

minq_status take_kv4_umma_status(int* v) {
  MINQ_CUDA_TRY(cudaMemcpyFromSymbol(v, g_kv4_umma_status, sizeof(int)));
  if (*v == 0) return MINQ_OK;
  const int zero = 0;
  MINQ_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_umma_status, &zero, sizeof(int)));
  return MINQ_OK;
}

}  // namespace minq
