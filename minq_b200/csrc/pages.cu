// Block tables and slot maps of a paged K/V cache, built on the GPU from the
// requests' lengths (no reference counterpart: the reference holds one
// contiguous cache, model.rs:100-131).
//
// extend: request r grows from l_r to l_r + n_r tokens. With page size P it
// holds ceil(l_r / P) pages and wants ceil((l_r + n_r) / P); the step's new
// pages, numbered j in the order (request, position), are free[n_free-1-j]:
// taken from the top of the stack of free pages. Token t of the step belongs
// to the request with q_start[r] <= t < q_start[r+1] (q_start: exclusive
// prefix sum of n) and lies at position l_r + t - q_start[r].
// trim: request r shrinks to min(l_r, keep_r); its pages go back on the stack
// so that the one with the lowest j lies on top, which makes an extend that is
// trimmed again leave the stack as it was.
//
// One launch of one cluster of up to 8 CTAs. Every CTA scans all requests
// into shared memory (two integers a request); tokens and pages are then
// spread over the cluster's threads, each finding its request by a binary
// search in shared memory. A page id comes from the old part of the table or
// from the stack, never from a table entry written in this launch, so the
// only ordering needed is one cluster barrier: after it every input length
// and the free count have been read, and the outputs may overwrite them in
// place (lens_out == lens). Bound by latency: a few dependent loads, the scan
// and the barriers; the bytes (12 a token) are nothing. Measured, call after call
// in a graph: extend of 64 decoding requests 3.4 us, of 1000 with prompts (some
// 19,000 tokens) 9.9 us (9.5 without a look at the partly filled pages), trim of 500
// requests 6.4 us; the last alone 8.6 us (77 us with a division per page and a search
// in L2 per id).
#include <cooperative_groups.h>

#include <string>

#include "common.cuh"
#include "kernels.h"

namespace minq {

namespace {

namespace cg = cooperative_groups;

constexpr int kPagesThreads = 1024;
constexpr int kPagesMaxReq = 8192;
constexpr int kPagesMaxCtas = 8;  // the portable cluster size

struct PagesParams {
  const int* lens;
  const int* arg;  // new tokens (extend) or lengths to keep (trim)
  int n_req, page_shift;
  int* table;
  size_t table_stride;
  int* free_pages;
  int n_pages;
  const int* n_free;
  int* lens_out;
  int* n_free_out;
  int* info;
  // extend
  int max_tokens;
  int* q_start;
  long long* slots;
  int* positions;
};

struct PagesShared {
  long long wt[32], wp[32];  // warp totals of the scan
  int flags;                 // this CTA's finding, then the cluster's
};

// Exclusive prefix of (a, b) over the block; totals in every thread.
__device__ void scan2(long long& a, long long& b, long long& ta, long long& tb, PagesShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long va = __shfl_up_sync(0xffffffffu, ia, o);
    const long long vb = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia += va;
      ib += vb;
    }
  }
  __syncthreads();
  if (lane == 31) {
    sh.wt[warp] = ia;
    sh.wp[warp] = ib;
  }
  __syncthreads();
  long long ba = 0, bb = 0;
  ta = tb = 0;
  for (int w = 0; w < nw; ++w) {
    const long long va = sh.wt[w], vb = sh.wp[w];
    if (w < warp) {
      ba += va;
      bb += vb;
    }
    ta += va;
    tb += vb;
  }
  a = ba + ia - a;
  b = bb + ib - b;
}

// Largest r with start[r] <= x (start[0] = 0 <= x).
__device__ __forceinline__ int find_last(const int* start, int n, int x) {
  int lo = 0, hi = n;  // start[lo] <= x < start[hi] (start[n]: past the end)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Pages of `len` positions.
__device__ __forceinline__ int pages_of(int len, int shift) {
  return (int)(((unsigned)len + ((1u << shift) - 1)) >> shift);
}

template <bool EXTEND>
__global__ void __launch_bounds__(kPagesThreads) pages_kernel(PagesParams p) {
  extern __shared__ int dyn[];
  int* s_page = dyn;                  // [n_req] first moved page
  int* s_base = dyn + p.n_req;        // [n_req] its column in the request's table row
  int* s_tok = dyn + 2 * p.n_req;     // [n_req] first token (extend)
  int* s_len = dyn + 3 * p.n_req;     // [n_req] length before (extend)
  __shared__ PagesShared sh;
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int ncta = (int)cl.num_blocks(), cta = (int)cl.block_rank();
  const int tid = threadIdx.x, nthreads = blockDim.x;
  const int gid = cta * nthreads + tid, gthreads = ncta * nthreads;
  const int shift = p.page_shift, mask = (1 << shift) - 1;
  if (tid == 0) sh.flags = 0;
  __syncthreads();
  cl.barrier_arrive();  // this CTA's flags word may be written by the others

  // every CTA: all requests' lengths, checked and scanned
  const int n_free = *p.n_free;
  int flags = n_free < 0 || n_free > p.n_pages ? MINQ_PAGES_BAD_PAGE : 0;
  const long long cap = (long long)p.table_stride << shift;
  long long tokens = 0, pages = 0;
  for (int base = 0; base < p.n_req; base += nthreads) {
    const int r = base + tid;
    long long t = 0, g = 0;
    int len = 0, from = 0, last = 0;
    bool goes_on = false;
    if (r < p.n_req) {
      len = p.lens[r];
      const int arg = p.arg[r];
      if (len < 0 || arg < 0) {
        flags |= MINQ_PAGES_BAD_LENGTH;
      } else if (EXTEND) {
        const long long after = (long long)len + arg;
        if (after > cap || after > 0x7fffffffll) {
          flags |= MINQ_PAGES_ROW_FULL;
        } else {
          from = pages_of(len, shift);
          g = pages_of((int)after, shift) - from;
          // the partly filled page that new tokens go on in (a column of the row,
          // as len < after <= cap); looked at behind the scan, when it has come
          goes_on = arg > 0 && (len & mask);
          if (goes_on) last = p.table[(size_t)r * p.table_stride + (len >> shift)];
        }
        t = arg;
      } else {
        if (len > cap) flags |= MINQ_PAGES_ROW_FULL;
        from = pages_of(min(arg, len), shift);
        g = pages_of(len, shift) - from;
      }
    }
    long long tt, tg;
    scan2(t, g, tt, tg, sh);
    if (goes_on && (last < 0 || last >= p.n_pages)) flags |= MINQ_PAGES_BAD_PAGE;
    // offsets past 2^31 only occur in a step that is refused below
    if (r < p.n_req) {
      s_page[r] = (int)(pages + g);
      s_base[r] = from;
      if (EXTEND) {
        s_tok[r] = (int)(tokens + t);
        s_len[r] = len;
      }
    }
    tokens += tt;
    pages += tg;
  }
  if (EXTEND && tokens > p.max_tokens) flags |= MINQ_PAGES_TOO_MANY_TOKENS;
  if (EXTEND && pages > n_free) flags |= MINQ_PAGES_SHORT;
  if (!EXTEND && pages > (long long)p.n_pages - n_free) flags |= MINQ_PAGES_BAD_PAGE;
  flags = __reduce_or_sync(0xffffffffu, flags);
  if ((tid & 31) == 0 && flags) atomicOr(&sh.flags, flags);
  __syncthreads();
  flags = sh.flags;
  cl.barrier_wait();

  // the ids that move must be pages of the pool (spread over the cluster)
  const int moved = flags ? 0 : (int)pages;
  if (moved) {
    int bad = 0;
    for (int j = gid; j < moved; j += gthreads) {
      int id;
      if (EXTEND) {
        id = p.free_pages[n_free - 1 - j];
      } else {
        const int r = find_last(s_page, p.n_req, j);
        id = p.table[(size_t)r * p.table_stride + s_base[r] + (j - s_page[r])];
        // (above the free pages: no part of the list until n_free_out says so)
        p.free_pages[n_free + moved - 1 - j] = id;
      }
      bad |= id < 0 || id >= p.n_pages;
    }
    if (bad)
      for (int c = 0; c < ncta; ++c) atomicOr(cl.map_shared_rank(&sh.flags, c), MINQ_PAGES_BAD_PAGE);
  }
  // after this barrier every length and the free count have been read: they may
  // be overwritten in place
  cl.sync();
  flags = sh.flags;
  const bool ok = flags == 0;
  if (EXTEND) {
    const int n_tok = ok ? (int)tokens : 0;
    for (int t = gid; t < p.max_tokens; t += gthreads) {
      long long slot = -1;
      int pos = 0;
      if (t < n_tok) {
        const int r = find_last(s_tok, p.n_req, t);
        pos = s_len[r] + (t - s_tok[r]);
        const int col = pos >> shift;
        const int id = col < s_base[r] ? p.table[(size_t)r * p.table_stride + col]
                                       : p.free_pages[n_free - 1 - (s_page[r] + (col - s_base[r]))];
        slot = ((long long)id << shift) + (pos & mask);
      }
      p.slots[t] = slot;
      if (p.positions) p.positions[t] = pos;
    }
    if (ok)
      for (int j = gid; j < moved; j += gthreads) {
        const int r = find_last(s_page, p.n_req, j);
        p.table[(size_t)r * p.table_stride + s_base[r] + (j - s_page[r])] =
            p.free_pages[n_free - 1 - j];
      }
  }
  for (int r = gid; r < p.n_req; r += gthreads) {
    const int len = p.lens[r], arg = p.arg[r];
    p.lens_out[r] = !ok ? len : EXTEND ? len + arg : min(len, arg);
    if (EXTEND) p.q_start[r] = ok ? s_tok[r] : 0;
  }
  if (gid == 0) {
    *p.n_free_out = !ok ? n_free : EXTEND ? n_free - moved : n_free + moved;
    if (EXTEND) p.q_start[p.n_req] = ok ? (int)tokens : 0;
    p.info[0] = flags;
    const long long lack = EXTEND && n_free >= 0 ? pages - n_free : 0;
    p.info[1] = (flags & MINQ_PAGES_SHORT) ? (int)(lack > 0x7fffffffll ? 0x7fffffffll : lack) : 0;
  }
  pdl_launch_dependents();
}

template <bool EXTEND>
minq_status launch_pages(const PagesParams& p, cudaStream_t s) {
  // one thread a token, or a few pages a request (trim's are not known here); 8
  // CTAs only when there is work for them
  const int items = EXTEND ? (p.max_tokens > p.n_req ? p.max_tokens : p.n_req) : 32 * p.n_req;
  const int threads = items <= 128 ? 128 : items <= 512 ? 512 : kPagesThreads;
  int ctas = 1;
  while (ctas < kPagesMaxCtas && ctas * threads < items) ctas *= 2;
  const size_t smem = (EXTEND ? 4 : 2) * (size_t)p.n_req * sizeof(int);
  const void* fn = reinterpret_cast<const void*>(pages_kernel<EXTEND>);
  MINQ_TRY(ensure_dynamic_smem(fn, smem));
  prefer_max_shared(fn);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  count_launch();
  MINQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, pages_kernel<EXTEND>, p));
  return MINQ_OK;
}

minq_status pages_check(const char* what, size_t n_req, size_t page_size, size_t table_stride,
                        size_t n_pages) {
  if (n_req > (size_t)kPagesMaxReq)
    return fail(MINQ_ERR_SHAPE, std::string(what) + ": at most 8192 requests, got " +
                                    std::to_string(n_req));
  if (!kv4_page_size_ok(page_size))
    return fail(MINQ_ERR_SHAPE, std::string(what) + ": page size must be a power of two in "
                                    "16..1024, got " + std::to_string(page_size));
  if (table_stride == 0 || table_stride > (1u << 30) || n_pages > (1u << 30))
    return fail(MINQ_ERR_SHAPE, std::string(what) + ": table width or page count out of range");
  return MINQ_OK;
}

}  // namespace

bool kv4_page_size_ok(size_t P) { return P >= 16 && P <= 1024 && (P & (P - 1)) == 0; }

}  // namespace minq

using namespace minq;

extern "C" {

minq_status minq_pages_extend(const int32_t* lens, const int32_t* new_tokens, size_t n_req,
                              size_t page_size, int32_t* table, size_t table_stride,
                              const int32_t* free_pages, size_t n_pages, const int32_t* n_free,
                              size_t max_tokens, int32_t* lens_out, int32_t* n_free_out,
                              int32_t* q_start, int64_t* slots, int32_t* positions, int32_t* info,
                              void* stream) {
  MINQ_TRY(pages_check("pages_extend", n_req, page_size, table_stride, n_pages));
  if (max_tokens > (1u << 30))
    return fail(MINQ_ERR_SHAPE, "pages_extend: at most 2^30 tokens a step");
  if (!n_free || !n_free_out || !q_start || !info || (max_tokens && !slots) ||
      (n_req && (!lens || !new_tokens || !lens_out || !table)) || (n_pages && !free_pages))
    return fail(MINQ_ERR_ARG, "null pointer");
  MINQ_TRY(require_device());
  PagesParams p{};
  p.lens = lens;
  p.arg = new_tokens;
  p.n_req = (int)n_req;
  while ((size_t(1) << p.page_shift) < page_size) ++p.page_shift;
  p.table = table;
  p.table_stride = table_stride;
  p.free_pages = const_cast<int32_t*>(free_pages);  // only read when extending
  p.n_pages = (int)n_pages;
  p.n_free = n_free;
  p.lens_out = lens_out;
  p.n_free_out = n_free_out;
  p.info = info;
  p.max_tokens = (int)max_tokens;
  p.q_start = q_start;
  p.slots = reinterpret_cast<long long*>(slots);
  p.positions = positions;
  return launch_pages<true>(p, (cudaStream_t)stream);
}

minq_status minq_pages_trim(const int32_t* lens, const int32_t* keep, size_t n_req,
                            size_t page_size, const int32_t* table, size_t table_stride,
                            int32_t* free_pages, size_t n_pages, const int32_t* n_free,
                            int32_t* lens_out, int32_t* n_free_out, int32_t* info, void* stream) {
  MINQ_TRY(pages_check("pages_trim", n_req, page_size, table_stride, n_pages));
  if (!n_free || !n_free_out || !info ||
      (n_req && (!lens || !keep || !lens_out || !table)) || (n_pages && !free_pages))
    return fail(MINQ_ERR_ARG, "null pointer");
  MINQ_TRY(require_device());
  PagesParams p{};
  p.lens = lens;
  p.arg = keep;
  p.n_req = (int)n_req;
  while ((size_t(1) << p.page_shift) < page_size) ++p.page_shift;
  p.table = const_cast<int32_t*>(table);  // only read when trimming
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.n_pages = (int)n_pages;
  p.n_free = n_free;
  p.lens_out = lens_out;
  p.n_free_out = n_free_out;
  p.info = info;
  return launch_pages<false>(p, (cudaStream_t)stream);
}

}  // extern "C"
