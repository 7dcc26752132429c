// frn_kv_cache.cu -- data movement of a paged key-value cache: appending new
// tokens to their pages, and copying whole pages of many pools at once.
//
// Both are copies, bound by HBM: every byte is read once and written once.
//
// append   token t of sequence b goes to position start_lens[b] + t -
//          cu_seqlens[b] of that sequence, i.e. to slot position % page_size
//          of page page_table[b, position / page_size].  A CTA takes a run of
//          tokens, resolves each token's slot once (the search over cu_seqlens
//          and the page lookup are dependent loads; one thread per token does
//          them, not one per 16 bytes), then streams K and V in 16-byte
//          pieces.
//          21506 tokens (176 MB) take 30.6 us, 5.8 TB/s or 88% of a plain
//          copy's rate; 64 tokens 1.9 us, a launch.
// copy     the (src, dst) list and the pool pointers travel as kernel
//          parameters: no upload and no workspace, so a fork is one launch.
//          8 pages of 32 KB in 64 pools (34 MB) take 4.9 us, 1001 pages (4.2 GB)
//          624 us, 6.7 TB/s.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>

#include "frn_internal.h"
#include "frn_ptx.cuh"

namespace frn {

constexpr int kAppendThreads = 256;
constexpr int kAppendMaxTokens = 16;  // tokens of one CTA
constexpr int kAppendVecs = 4;        // 16-byte pieces of K and of V that a thread has in flight

struct AppendParams {
  PagedView kv;
  const char* k;
  const char* v;
  int64_t k_token, k_head, v_token, v_head;      // input strides, bytes
  int64_t pk_page, pk_slot, pk_head, pv_page, pv_slot, pv_head;  // cache strides, bytes
  const int32_t* start;
  const int32_t* cu;  // null: one token per sequence
  int64_t tokens;
  int32_t batch, tokens_per_cta, head_vecs, row_vecs;  // 16-byte pieces of a head / of all heads
};

// Index of the sequence that token t belongs to, or -1: the largest b with
// cu[b] <= t, if t < cu[b + 1].
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, int64_t t) {
  int lo = 0, hi = batch;  // cu[lo] <= t < cu[hi] is kept, if it holds at the start
  if (t < cu[0] || t >= cu[batch]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendParams p) {
  __shared__ int32_t sm_page[kAppendMaxTokens];
  __shared__ int32_t sm_slot[kAppendMaxTokens];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_cta;
  griddep_launch_dependents();
  griddep_wait();
  if (static_cast<int>(threadIdx.x) < p.tokens_per_cta) {
    const int64_t t = t0 + threadIdx.x;
    int32_t page = -1, slot = 0;
    if (t < p.tokens) {
      const int b = p.cu ? find_sequence(p.cu, p.batch, t) : static_cast<int>(t);
      if (b >= 0) {
        const int64_t first = p.cu ? p.cu[b] : t;
        const int64_t pos = p.start[b] + (t - first);
        const int64_t at = pos / p.kv.page_size;
        if (p.start[b] >= 0 && at < p.kv.max_pages) {
          page = p.kv.page_table[b * p.kv.table_stride + at];
          slot = static_cast<int32_t>(pos - at * p.kv.page_size);
        }
        if (page < 0 || page >= p.kv.num_pages) {
          page = -1;  // nothing is written for this token
          atomicOr(&g_frn_device_error, kDevErrBadPage);
        }
      }
    }
    sm_page[threadIdx.x] = page;
    sm_slot[threadIdx.x] = slot;
  }
  __syncthreads();
  const int n = p.tokens_per_cta * p.row_vecs;
  // Pieces of K and V are loaded four at a time before any is stored: one at a
  // time, 21506 tokens of 8 heads of 128 took 32.8 us instead of 30.6.
  for (int i0 = static_cast<int>(threadIdx.x); i0 < n; i0 += kAppendThreads * kAppendVecs) {
    uint4 kv[kAppendVecs], vv[kAppendVecs];
    char* kd[kAppendVecs];
    char* vd[kAppendVecs];
#pragma unroll
    for (int u = 0; u < kAppendVecs; ++u) {
      const int i = i0 + u * kAppendThreads;
      kd[u] = nullptr;
      if (i >= n) continue;
      const int tok = i / p.row_vecs, r = i - tok * p.row_vecs;
      const int head = r / p.head_vecs, c = r - head * p.head_vecs;
      const int32_t page = sm_page[tok];
      if (page < 0) continue;
      const int64_t t = t0 + tok, slot = sm_slot[tok];
      kv[u] = ld_global_nc_v4(p.k + t * p.k_token + head * p.k_head + c * 16);
      vv[u] = ld_global_nc_v4(p.v + t * p.v_token + head * p.v_head + c * 16);
      kd[u] = static_cast<char*>(p.kv.k) + page * p.pk_page + slot * p.pk_slot + head * p.pk_head +
              c * 16;
      vd[u] = static_cast<char*>(p.kv.v) + page * p.pv_page + slot * p.pv_slot + head * p.pv_head +
              c * 16;
    }
#pragma unroll
    for (int u = 0; u < kAppendVecs; ++u)
      if (kd[u]) {
        *reinterpret_cast<uint4*>(kd[u]) = kv[u];
        *reinterpret_cast<uint4*>(vd[u]) = vv[u];
      }
  }
}

int run_kv_append(const KvAppendProblem& a, cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_error("cudaGetDevice");
  const int64_t es = a.dtype == FRN_DTYPE_F32 ? 4 : 2;
  AppendParams p;
  p.kv = a.kv;
  p.k = static_cast<const char*>(a.k);
  p.v = static_cast<const char*>(a.v);
  p.k_token = a.k_token_stride * es;
  p.k_head = a.k_head_stride * es;
  p.v_token = a.v_token_stride * es;
  p.v_head = a.v_head_stride * es;
  p.pk_page = a.kv.k_page_stride * es;
  p.pk_slot = a.kv.k_token_stride * es;
  p.pk_head = a.kv.k_head_stride * es;
  p.pv_page = a.kv.v_page_stride * es;
  p.pv_slot = a.kv.v_token_stride * es;
  p.pv_head = a.kv.v_head_stride * es;
  p.start = a.start_lens;
  p.cu = a.cu_seqlens;
  p.tokens = a.tokens;
  p.batch = static_cast<int32_t>(a.batch);
  p.head_vecs = static_cast<int32_t>(a.kv.head_dim * es / 16);
  p.row_vecs = static_cast<int32_t>(a.kv.num_kv_heads) * p.head_vecs;
  // Runs as long as they leave four CTAs for every SM: few tokens are spread,
  // many share the slot look-up.
  int64_t run = a.tokens / (4 * sm_count(dev));
  if (run > kAppendMaxTokens) run = kAppendMaxTokens;
  if (run < 1) run = 1;
  p.tokens_per_cta = static_cast<int32_t>(run);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.tokens + run - 1) / run));
  cfg.blockDim = dim3(kAppendThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_append_kernel, p);
  if (e != cudaSuccess) return set_cuda_error("launch kv_append", e);
  return 0;
}

// ------------------------------------------------------------- page copies

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;  // 16-byte pieces of one thread, all loaded before any is stored
constexpr int kCopyMaxPools = 128;
constexpr int kCopyFewPairs = 64, kCopyMaxPairs = 1024;

// For up to PAIRS pairs: a launch passes the whole struct, so a fork's few pairs
// get a small one.
template <int PAIRS>
struct CopyParams {
  char* pools[kCopyMaxPools];
  int32_t src[PAIRS];
  int32_t dst[PAIRS];
  int64_t page_stride;  // bytes
  uint32_t page_vecs;   // 16-byte pieces of a page
  uint32_t npairs;
  uint64_t total;       // 16-byte pieces of all pages
};

template <int PAIRS>
__global__ void __launch_bounds__(kCopyThreads)
    kv_copy_kernel(const __grid_constant__ CopyParams<PAIRS> p) {
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (kCopyThreads * kCopyVecs);
  const uint64_t page0 = first / p.page_vecs;  // (pool, pair) number of the CTA's first piece
  const uint32_t rest = static_cast<uint32_t>(first - page0 * p.page_vecs);
  griddep_launch_dependents();
  griddep_wait();
  uint4 data[kCopyVecs];
  char* to[kCopyVecs];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i) {
    const uint32_t at = static_cast<uint32_t>(i * kCopyThreads) + threadIdx.x;
    to[i] = nullptr;
    if (first + at < p.total) {
      const uint32_t skip = (rest + at) / p.page_vecs, off = (rest + at) - skip * p.page_vecs;
      const uint32_t page = static_cast<uint32_t>(page0) + skip;
      const uint32_t pool = page / p.npairs, pair = page - pool * p.npairs;
      char* base = p.pools[pool] + static_cast<uint64_t>(off) * 16;
      data[i] = *reinterpret_cast<const uint4*>(base + p.src[pair] * p.page_stride);
      to[i] = base + p.dst[pair] * p.page_stride;
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (to[i]) *reinterpret_cast<uint4*>(to[i]) = data[i];
}

template <int PAIRS>
static int launch_kv_copy(void* const* pools, int64_t npools, int64_t page_bytes,
                          int64_t page_stride_bytes, const int32_t* src, const int32_t* dst,
                          int64_t npairs, cudaStream_t stream) {
  CopyParams<PAIRS> p;
  for (int64_t i = 0; i < npools; ++i) p.pools[i] = static_cast<char*>(pools[i]);
  for (int64_t i = 0; i < npairs; ++i) {
    p.src[i] = src[i];
    p.dst[i] = dst[i];
  }
  p.page_stride = page_stride_bytes;
  p.page_vecs = static_cast<uint32_t>(page_bytes / 16);
  p.npairs = static_cast<uint32_t>(npairs);
  p.total = static_cast<uint64_t>(npools) * npairs * p.page_vecs;
  const uint64_t per_cta = kCopyThreads * kCopyVecs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.total + per_cta - 1) / per_cta));
  cfg.blockDim = dim3(kCopyThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_copy_kernel<PAIRS>, p);
  if (e != cudaSuccess) return set_cuda_error("launch kv_copy", e);
  return 0;
}

int run_kv_pages_copy(void* const* pools, int64_t npools, int64_t page_bytes,
                      int64_t page_stride_bytes, const int32_t* src, const int32_t* dst,
                      int64_t npairs, cudaStream_t stream) {
  for (int64_t pool0 = 0; pool0 < npools; pool0 += kCopyMaxPools)
    for (int64_t pair0 = 0; pair0 < npairs; pair0 += kCopyMaxPairs) {
      const int64_t np = npools - pool0 < kCopyMaxPools ? npools - pool0 : kCopyMaxPools;
      const int64_t nq = npairs - pair0 < kCopyMaxPairs ? npairs - pair0 : kCopyMaxPairs;
      const auto launch = nq <= kCopyFewPairs ? launch_kv_copy<kCopyFewPairs>
                                              : launch_kv_copy<kCopyMaxPairs>;
      const int rc = launch(pools + pool0, np, page_bytes, page_stride_bytes, src + pair0,
                            dst + pair0, nq, stream);
      if (rc) return rc;
    }
  return 0;
}

}  // namespace frn
