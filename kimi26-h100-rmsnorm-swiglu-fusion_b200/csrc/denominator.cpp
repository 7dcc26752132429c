// denominator.cpp -- the `denominator_cuda` Python module.
//
// Same module name and RMSNorm exports as the reference's pybind11 binding
// (reference csrc/denominator.cpp:152-213), re-implemented as a thin layer
// over the C ABI in include/frn_b200.h: tensors are checked the way the
// reference's host launchers check them (csrc/denominator_kernel.cu:1999-2001,
// same messages), then their pointers, row strides and the current CUDA stream
// are handed to libfrn_b200.so.  New exports: fused_rmsnorm_linear and
// fused_rmsnorm_swiglu (single-launch fused ops), the int8-weight path, and
// device_error.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "frn_b200.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FRN_DTYPE_F32;
    case at::kHalf: return FRN_DTYPE_F16;
    case at::kBFloat16: return FRN_DTYPE_BF16;
    default: return -1;
  }
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FRN_OK, what, " failed (status ", rc, "): ", frn_last_error());
}

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void rmsnorm_normalize_impl(const at::Tensor& x, at::Tensor& raw_output, const at::Tensor& b_new,
                            int64_t h, double eps, int threads, const char* name) {
  TORCH_CHECK(x.dim() == 2, "x must be 2D");
  TORCH_CHECK(raw_output.dim() == 2, "raw_output must be 2D");
  TORCH_CHECK(x.is_cuda() && raw_output.is_cuda() && b_new.is_cuda(),
              "All tensors must be on CUDA");
  const int dt = dtype_code(x);
  TORCH_CHECK(dt >= 0, "Unsupported dtype for RMSNorm ", name,
              ": only fp32, fp16, bf16 supported");
  TORCH_CHECK(raw_output.scalar_type() == x.scalar_type() &&
                  b_new.scalar_type() == x.scalar_type(),
              "x, raw_output and b_new must share one dtype");
  TORCH_CHECK(x.size(0) == raw_output.size(0), "x and raw_output must have the same rows");
  TORCH_CHECK(h == x.size(1), "h (", h, ") must equal x.size(1) (", x.size(1), ")");
  TORCH_CHECK(b_new.numel() == raw_output.size(1), "b_new must have raw_output.size(1) elements");
  TORCH_CHECK(x.stride(1) == 1 || x.size(1) == 1, "x must have unit stride along its last dim");
  TORCH_CHECK(raw_output.stride(1) == 1 || raw_output.size(1) == 1,
              "raw_output must have unit stride along its last dim");
  const at::Tensor b = b_new.contiguous();
  const c10::cuda::CUDAGuard guard(x.device());
  check_rc(frn_rmsnorm_normalize(dt, x.data_ptr(), x.stride(0), raw_output.data_ptr(),
                                 raw_output.stride(0), b.data_ptr(), x.size(0), h,
                                 raw_output.size(1), static_cast<float>(eps), threads,
                                 stream_of(x)),
           name);
}

void rmsnorm_normalize(const at::Tensor& x, at::Tensor raw_output, const at::Tensor& b_new,
                       int64_t h, double eps) {
  rmsnorm_normalize_impl(x, raw_output, b_new, h, eps, 256, "rmsnorm_normalize");
}

void rmsnorm_normalize_512(const at::Tensor& x, at::Tensor raw_output, const at::Tensor& b_new,
                           int64_t h, double eps) {
  rmsnorm_normalize_impl(x, raw_output, b_new, h, eps, 512, "rmsnorm_normalize_512");
}

std::vector<at::Tensor> fused_rmsnorm_linear_split(const at::Tensor& x_in, const at::Tensor& w,
                                                   const c10::optional<at::Tensor>& b_new,
                                                   double eps, std::vector<int64_t> split_sizes) {
  TORCH_CHECK(x_in.dim() == 2 && w.dim() == 2, "x and W_fused must be 2D");
  TORCH_CHECK(x_in.is_cuda() && w.is_cuda() && (!b_new || b_new->is_cuda()),
              "All tensors must be on CUDA");
  TORCH_CHECK(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf,
              "fused_rmsnorm_linear_split supports bf16 and fp16 (got ", x_in.scalar_type(), ")");
  TORCH_CHECK(w.scalar_type() == x_in.scalar_type(), "x and W_fused must share one dtype");
  TORCH_CHECK(x_in.size(1) == w.size(1), "x.size(1) != W_fused.size(1)");
  const int n = static_cast<int>(split_sizes.size());
  TORCH_CHECK(n >= 1 && n <= FRN_MAX_PARTS, "split_sizes must have 1..", FRN_MAX_PARTS,
              " entries");
  const at::Tensor x = (x_in.stride(1) == 1 || x_in.size(1) == 1) ? x_in : x_in.contiguous();
  const at::Tensor wc = (w.stride(1) == 1) ? w : w.contiguous();
  const int64_t M = x.size(0), K = x.size(1), N = wc.size(0);
  at::Tensor b;
  const void* bptr = nullptr;
  if (b_new && b_new->defined()) {
    TORCH_CHECK(b_new->numel() == N && b_new->scalar_type() == x.scalar_type(),
                "b_new must have W_fused.size(0) elements of x's dtype");
    b = b_new->contiguous();
    bptr = b.data_ptr();
  }
  std::vector<at::Tensor> outs;
  int64_t cols[FRN_MAX_PARTS], strides[FRN_MAX_PARTS];
  void* ptrs[FRN_MAX_PARTS];
  for (int i = 0; i < n; ++i) {
    outs.push_back(at::empty({M, split_sizes[i]}, x.options()));
    cols[i] = split_sizes[i];
    strides[i] = outs.back().stride(0);
    ptrs[i] = outs.back().data_ptr();
  }
  const c10::cuda::CUDAGuard guard(x.device());
  check_rc(frn_fused_rmsnorm_linear_split(dtype_code(x), x.data_ptr(), M, K, x.stride(0),
                                          wc.data_ptr(), N, wc.stride(0), bptr,
                                          static_cast<float>(eps), n, cols, ptrs, strides,
                                          stream_of(x)),
           "fused_rmsnorm_linear_split");
  return outs;
}

// ---- decode-step GQA attention (gqa_attention_cuda exports of the reference)
void gqa_decode_impl(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     at::Tensor& out, double scale, const char* name) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 4 && v.dim() == 4 && out.dim() == 3,
              name, ": q/out must be [batch, heads, head_dim], caches [batch, ctx, kv_heads, head_dim]");
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda() && out.is_cuda(),
              "All tensors must be on CUDA");
  const int dt = dtype_code(q);
  TORCH_CHECK(dt >= 0, name, ": only fp32, fp16, bf16 supported");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
                  out.scalar_type() == q.scalar_type(),
              name, ": q, caches and output must share one dtype");
  TORCH_CHECK(k.sizes() == v.sizes(), name, ": k_cache and v_cache shapes differ");
  TORCH_CHECK(out.sizes() == q.sizes(), name, ": output must match q");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(2), name, ": batch/head_dim mismatch");
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous() && out.is_contiguous(),
              name, ": tensors must be contiguous");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), T = k.size(1), Hkv = k.size(2);
  const c10::cuda::CUDAGuard guard(q.device());
  const size_t ws_bytes = frn_gqa_decode_workspace_size(B, Hq, Hkv, D, T);
  at::Tensor ws;
  if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  check_rc(frn_gqa_decode_attention(dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                    B, Hq, Hkv, D, T, static_cast<float>(scale),
                                    ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream_of(q)),
           name);
}

void gqa_decode_v2(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor out,
                   double scale) {
  gqa_decode_impl(q, k, v, out, scale, "gqa_decode_v2");
}

void gqa_decode_v3(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor out,
                   int64_t group_size, double scale) {
  TORCH_CHECK(k.dim() == 4 && group_size * k.size(2) == q.size(1),
              "gqa_decode_v3: group_size * num_kv_heads must equal num_q_heads");
  gqa_decode_impl(q, k, v, out, scale, "gqa_decode_v3");
}

// ---- prompts and the paged key-value cache

// `t` [tokens, heads, dim] as the kernels read it: unit stride along dim,
// other strides multiples of 16 bytes and no smaller than a head, 16-byte
// aligned; a copy where it is not.
at::Tensor heads_legal(const at::Tensor& t) {
  const int64_t es = t.element_size(), d = t.size(2);
  bool ok = (t.stride(2) == 1 || d == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 2 && ok; ++i)
    ok = t.size(i) <= 1 || (t.stride(i) >= d && (t.stride(i) * es) % 16 == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Stride of dim i, or that of a contiguous layout where the dim has at most
// one entry and its stride means nothing.
int64_t stride_or(const at::Tensor& t, int i) {
  if (t.size(i) > 1) return t.stride(i);
  int64_t s = 1;
  for (int j = t.dim() - 1; j > i; --j) s *= std::max<int64_t>(t.size(j), 1);
  return s;
}

void check_ints(const at::Tensor& t, const at::Tensor& on, int dim, const char* name,
                const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && t.device() == on.device(), name,
              ": ", what, " must be a ", dim, "-D int32 tensor on ", on.device());
  TORCH_CHECK(t.numel() == 0 || t.stride(dim - 1) == 1 || t.size(dim - 1) <= 1, name, ": ", what,
              " must have unit stride along its last dim");
}

at::Tensor output_for(const c10::optional<at::Tensor>& out, const at::Tensor& q, int64_t d,
                      const char* name) {
  if (!out || !out->defined()) return at::empty({q.size(0), q.size(1), d}, q.options());
  TORCH_CHECK(out->dim() == 3 && out->size(0) == q.size(0) && out->size(1) == q.size(1) &&
                  out->size(2) == d && out->scalar_type() == q.scalar_type() &&
                  out->device() == q.device(),
              name, ": output must be [", q.size(0), ", ", q.size(1), ", ", d,
              "] of q's dtype and device");
  TORCH_CHECK(out->stride(2) == 1, name, ": output must have unit stride along its last dim");
  return *out;
}

at::Tensor gqa_prompt_attention(const at::Tensor& q_in, const at::Tensor& k_in,
                                const at::Tensor& v_in, const at::Tensor& cu_seqlens,
                                int64_t max_seqlen, double scale, c10::optional<at::Tensor> out) {
  const char* name = "gqa_prompt_attention";
  TORCH_CHECK(q_in.dim() == 3 && k_in.dim() == 3 && v_in.dim() == 3, name,
              ": q, k and v must be [tokens, heads, head_dim]");
  TORCH_CHECK(q_in.is_cuda() && k_in.is_cuda() && v_in.is_cuda() && cu_seqlens.is_cuda(),
              "All tensors must be on CUDA");
  TORCH_CHECK(q_in.scalar_type() == at::kBFloat16 || q_in.scalar_type() == at::kHalf, name,
              " supports bf16 and fp16 (got ", q_in.scalar_type(), ")");
  TORCH_CHECK(k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type() &&
                  k_in.device() == q_in.device() && v_in.device() == q_in.device(),
              name, ": q, k and v must share one dtype and device");
  TORCH_CHECK(k_in.size(0) == q_in.size(0) && v_in.size(0) == q_in.size(0) &&
                  k_in.size(1) == v_in.size(1) && k_in.size(2) == q_in.size(2),
              name, ": token, head or head_dim mismatch");
  check_ints(cu_seqlens, q_in, 1, name, "cu_seqlens");
  TORCH_CHECK(cu_seqlens.numel() >= 1, name, ": cu_seqlens must have batch + 1 entries");
  const at::Tensor q = heads_legal(q_in), k = heads_legal(k_in), v = heads_legal(v_in);
  at::Tensor o = output_for(out, q, v.size(2), name);
  const c10::cuda::CUDAGuard guard(q.device());
  check_rc(frn_gqa_prompt_attention(
               dtype_code(q), q.data_ptr(), stride_or(q, 0), stride_or(q, 1), k.data_ptr(),
               stride_or(k, 0), stride_or(k, 1), v.data_ptr(), stride_or(v, 0), stride_or(v, 1),
               o.data_ptr(), stride_or(o, 0), stride_or(o, 1), cu_seqlens.data_ptr<int32_t>(),
               cu_seqlens.numel() - 1, q.size(0), max_seqlen, q.size(1), k.size(1), q.size(2),
               v.size(2), static_cast<float>(scale), stream_of(q)),
           name);
  return o;
}

frn_paged_kv paged_view(const at::Tensor& k_pages, const at::Tensor& v_pages,
                        const at::Tensor& page_table, const at::Tensor& like, const char* name) {
  TORCH_CHECK(k_pages.dim() == 4 && k_pages.sizes() == v_pages.sizes(), name,
              ": pools must both be [num_pages, page_size, kv_heads, head_dim]");
  TORCH_CHECK(k_pages.is_cuda() && v_pages.is_cuda() && page_table.is_cuda(),
              "All tensors must be on CUDA");
  TORCH_CHECK(k_pages.scalar_type() == like.scalar_type() &&
                  v_pages.scalar_type() == like.scalar_type() &&
                  k_pages.device() == like.device() && v_pages.device() == like.device(),
              name, ": pools must share the new tensors' dtype and device");
  TORCH_CHECK(dtype_code(like) >= 0, name, ": only fp32, fp16, bf16 supported");
  TORCH_CHECK((k_pages.stride(3) == 1 && v_pages.stride(3) == 1) || k_pages.numel() == 0, name,
              ": pools must have unit stride along head_dim");
  check_ints(page_table, like, 2, name, "page_table");
  frn_paged_kv c;
  c.k = k_pages.data_ptr();
  c.v = v_pages.data_ptr();
  c.num_pages = k_pages.size(0);
  c.page_size = k_pages.size(1);
  c.num_kv_heads = k_pages.size(2);
  c.head_dim = k_pages.size(3);
  c.k_page_stride = stride_or(k_pages, 0);
  c.k_token_stride = stride_or(k_pages, 1);
  c.k_head_stride = stride_or(k_pages, 2);
  c.v_page_stride = stride_or(v_pages, 0);
  c.v_token_stride = stride_or(v_pages, 1);
  c.v_head_stride = stride_or(v_pages, 2);
  c.page_table = page_table.numel() ? page_table.data_ptr<int32_t>() : nullptr;
  c.page_table_stride = stride_or(page_table, 0);
  c.max_pages = page_table.size(1);
  return c;
}

at::Tensor gqa_paged_decode(const at::Tensor& q_in, const at::Tensor& k_pages,
                            const at::Tensor& v_pages, const at::Tensor& page_table,
                            const at::Tensor& seq_lens, double scale,
                            c10::optional<at::Tensor> out) {
  const char* name = "gqa_paged_decode";
  TORCH_CHECK(q_in.dim() == 3, name, ": q must be [batch, heads, head_dim]");
  TORCH_CHECK(q_in.is_cuda() && seq_lens.is_cuda(), "All tensors must be on CUDA");
  const frn_paged_kv c = paged_view(k_pages, v_pages, page_table, q_in, name);
  check_ints(seq_lens, q_in, 1, name, "seq_lens");
  TORCH_CHECK(q_in.size(2) == c.head_dim, name, ": head_dim mismatch");
  TORCH_CHECK(seq_lens.numel() == q_in.size(0) && page_table.size(0) == q_in.size(0), name,
              ": seq_lens and page_table must have an entry per sequence");
  const at::Tensor q = heads_legal(q_in);
  at::Tensor o = output_for(out, q, c.head_dim, name);
  if (q.size(0) == 0) return o;
  const c10::cuda::CUDAGuard guard(q.device());
  const int dt = dtype_code(q);
  const size_t need = frn_gqa_paged_decode_workspace_size(dt, q.size(0), q.size(1), c.num_kv_heads,
                                                          c.head_dim, c.page_size, c.max_pages);
  // The workspace straight from torch's allocator: as a tensor it would take
  // longer to make than the rest of the call.  Freed at once, it can only be
  // given to later work of this stream.
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_of(q));
  void* ws = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(need, stream);
  const int rc = frn_gqa_paged_decode_attention(
      dt, q.data_ptr(), stride_or(q, 0), stride_or(q, 1), &c, seq_lens.data_ptr<int32_t>(),
      o.data_ptr(), stride_or(o, 0), stride_or(o, 1), q.size(0), q.size(1),
      static_cast<float>(scale), ws, need, stream);
  c10::cuda::CUDACachingAllocator::raw_delete(ws);
  check_rc(rc, name);
  return o;
}

void kv_cache_append(const at::Tensor& k_in, const at::Tensor& v_in, at::Tensor k_pages,
                     at::Tensor v_pages, const at::Tensor& page_table,
                     const at::Tensor& start_lens, const c10::optional<at::Tensor>& cu_seqlens) {
  const char* name = "kv_cache_append";
  TORCH_CHECK(k_in.dim() == 3 && k_in.sizes() == v_in.sizes(), name,
              ": k and v must both be [tokens, kv_heads, head_dim]");
  TORCH_CHECK(k_in.is_cuda() && v_in.is_cuda() && start_lens.is_cuda(),
              "All tensors must be on CUDA");
  TORCH_CHECK(v_in.scalar_type() == k_in.scalar_type() && v_in.device() == k_in.device(), name,
              ": k and v must share one dtype and device");
  const frn_paged_kv c = paged_view(k_pages, v_pages, page_table, k_in, name);
  TORCH_CHECK(k_in.size(1) == c.num_kv_heads && k_in.size(2) == c.head_dim, name,
              ": kv_heads or head_dim mismatch");
  check_ints(start_lens, k_in, 1, name, "start_lens");
  const int64_t batch = start_lens.numel();
  TORCH_CHECK(page_table.size(0) == batch, name,
              ": start_lens and page_table must have an entry per sequence");
  const int32_t* cu = nullptr;
  if (cu_seqlens && cu_seqlens->defined()) {
    TORCH_CHECK(cu_seqlens->is_cuda(), "All tensors must be on CUDA");
    check_ints(*cu_seqlens, k_in, 1, name, "cu_seqlens");
    TORCH_CHECK(cu_seqlens->numel() == batch + 1, name, ": cu_seqlens must have batch + 1 entries");
    cu = cu_seqlens->data_ptr<int32_t>();
  }
  const at::Tensor k = heads_legal(k_in), v = heads_legal(v_in);
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(frn_kv_cache_append(dtype_code(k), k.data_ptr(), stride_or(k, 0), stride_or(k, 1),
                               v.data_ptr(), stride_or(v, 0), stride_or(v, 1), &c,
                               start_lens.data_ptr<int32_t>(), cu, batch, k.size(0),
                               stream_of(k)),
           name);
}

void kv_pages_copy(const std::vector<at::Tensor>& pools, const std::vector<int64_t>& src,
                   const std::vector<int64_t>& dst) {
  const char* name = "kv_pages_copy";
  TORCH_CHECK(src.size() == dst.size(), name, ": src and dst must have the same length");
  if (pools.empty() || src.empty()) return;
  const at::Tensor& first = pools[0];
  TORCH_CHECK(first.dim() >= 2, name, ": a pool must be [num_pages, ...]");
  std::vector<void*> ptrs;
  ptrs.reserve(pools.size());
  for (const at::Tensor& p : pools) {
    TORCH_CHECK(p.is_cuda(), "All tensors must be on CUDA");
    TORCH_CHECK(p.sizes() == first.sizes() && p.strides() == first.strides() &&
                    p.element_size() == first.element_size() && p.device() == first.device(),
                name, ": pools must share shape, strides, element size and device");
    ptrs.push_back(p.data_ptr());
  }
  TORCH_CHECK(first.is_contiguous() || first.size(0) == 0 ||
                  first.select(0, 0).is_non_overlapping_and_dense(),
              name, ": a page must be one dense block");
  std::vector<int32_t> from, to;
  from.reserve(src.size());
  to.reserve(src.size());
  for (size_t i = 0; i < src.size(); ++i) {
    TORCH_CHECK(src[i] >= 0 && src[i] < first.size(0) && dst[i] >= 0 && dst[i] < first.size(0),
                name, ": copy ", i, ": page ", src[i], " -> ", dst[i], " outside the ",
                first.size(0), " pages");
    from.push_back(static_cast<int32_t>(src[i]));
    to.push_back(static_cast<int32_t>(dst[i]));
  }
  const int64_t es = first.element_size();
  const c10::cuda::CUDAGuard guard(first.device());
  check_rc(frn_kv_pages_copy(ptrs.data(), static_cast<int64_t>(ptrs.size()), first.size(0),
                             first.numel() / first.size(0) * es, stride_or(first, 0) * es,
                             from.data(), to.data(), static_cast<int64_t>(from.size()),
                             stream_of(first)),
           name);
}

void rmsnorm_swiglu_impl(const at::Tensor& x, const at::Tensor& raw_output, at::Tensor& output,
                         const at::Tensor& b_new, int64_t h, int64_t intermediate, double eps,
                         int threads, const char* name) {
  TORCH_CHECK(x.dim() == 2, "x must be 2D");
  TORCH_CHECK(raw_output.dim() == 2, "raw_output must be 2D");
  TORCH_CHECK(output.dim() == 2, "output must be 2D");
  TORCH_CHECK(x.is_cuda() && raw_output.is_cuda() && output.is_cuda() && b_new.is_cuda(),
              "All tensors must be on CUDA");
  const int dt = dtype_code(x);
  TORCH_CHECK(dt >= 0, "Unsupported dtype for RMSNorm SwiGLU: only fp32, fp16, bf16 supported");
  TORCH_CHECK(raw_output.scalar_type() == x.scalar_type() &&
                  output.scalar_type() == x.scalar_type() && b_new.scalar_type() == x.scalar_type(),
              "x, raw_output, output and b_new must share one dtype");
  TORCH_CHECK(raw_output.size(0) == x.size(0) && output.size(0) == x.size(0),
              "x, raw_output and output must have the same rows");
  TORCH_CHECK(h == x.size(1), "h (", h, ") must equal x.size(1) (", x.size(1), ")");
  TORCH_CHECK(raw_output.size(1) == 2 * intermediate, "raw_output must have 2*intermediate columns");
  TORCH_CHECK(output.size(1) == intermediate, "output must have intermediate columns");
  TORCH_CHECK(b_new.numel() == 2 * intermediate, "b_new must have 2*intermediate elements");
  TORCH_CHECK(x.stride(1) == 1 && raw_output.stride(1) == 1 && output.stride(1) == 1,
              "x, raw_output and output must have unit stride along their last dim");
  const at::Tensor b = b_new.contiguous();
  const c10::cuda::CUDAGuard guard(x.device());
  check_rc(frn_rmsnorm_swiglu(dt, x.data_ptr(), x.stride(0), raw_output.data_ptr(),
                              raw_output.stride(0), output.data_ptr(), output.stride(0),
                              b.data_ptr(), x.size(0), h, intermediate, static_cast<float>(eps),
                              threads, stream_of(x)),
           name);
}

void rmsnorm_swiglu(const at::Tensor& x, const at::Tensor& raw_output, at::Tensor output,
                    const at::Tensor& b_new, int64_t h, int64_t intermediate, double eps) {
  rmsnorm_swiglu_impl(x, raw_output, output, b_new, h, intermediate, eps, 256, "rmsnorm_swiglu");
}

void rmsnorm_swiglu_512(const at::Tensor& x, const at::Tensor& raw_output, at::Tensor output,
                        const at::Tensor& b_new, int64_t h, int64_t intermediate, double eps) {
  rmsnorm_swiglu_impl(x, raw_output, output, b_new, h, intermediate, eps, 512,
                      "rmsnorm_swiglu_512");
}

at::Tensor fused_rmsnorm_swiglu(const at::Tensor& x_in, const at::Tensor& w,
                                const c10::optional<at::Tensor>& b_combined, double eps,
                                c10::optional<at::Tensor> out) {
  TORCH_CHECK(x_in.dim() == 2, "x must be 2D");
  TORCH_CHECK(w.dim() == 2, "W_combined must be 2D");
  TORCH_CHECK(x_in.is_cuda() && w.is_cuda() && (!b_combined || b_combined->is_cuda()),
              "All tensors must be on CUDA");
  TORCH_CHECK(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf,
              "fused_rmsnorm_swiglu supports bf16 and fp16 (got ", x_in.scalar_type(), ")");
  TORCH_CHECK(w.scalar_type() == x_in.scalar_type(), "x and W_combined must share one dtype");
  TORCH_CHECK(x_in.size(1) == w.size(1), "x.size(1) (", x_in.size(1),
              ") != W_combined.size(1) (", w.size(1), ")");
  TORCH_CHECK(w.size(0) % 2 == 0, "W_combined must have 2*intermediate rows");
  TORCH_CHECK(x_in.device() == w.device(), "x and W_combined must be on the same device");
  const at::Tensor x = (x_in.stride(1) == 1 || x_in.size(1) == 1) ? x_in : x_in.contiguous();
  const at::Tensor wc = (w.stride(1) == 1) ? w : w.contiguous();
  const int64_t M = x.size(0), K = x.size(1), I = wc.size(0) / 2;
  at::Tensor b;
  const void* bptr = nullptr;
  if (b_combined && b_combined->defined()) {
    TORCH_CHECK(b_combined->scalar_type() == x.scalar_type(), "b_combined must share x's dtype");
    TORCH_CHECK(b_combined->numel() == 2 * I, "b_combined must have W_combined.size(0) elements");
    b = b_combined->contiguous();
    bptr = b.data_ptr();
  }
  at::Tensor o;
  if (out && out->defined()) {
    o = *out;
    TORCH_CHECK(o.dim() == 2 && o.size(0) == M && o.size(1) == I, "out must be [M, intermediate]");
    TORCH_CHECK(o.scalar_type() == x.scalar_type() && o.is_cuda(), "out dtype/device mismatch");
    TORCH_CHECK(o.stride(1) == 1, "out must have unit stride along its last dim");
  } else {
    o = at::empty({M, I}, x.options());
  }
  const c10::cuda::CUDAGuard guard(x.device());
  check_rc(frn_fused_rmsnorm_swiglu(dtype_code(x), x.data_ptr(), M, K, x.stride(0), wc.data_ptr(),
                                    I, wc.stride(0), bptr, static_cast<float>(eps), o.data_ptr(),
                                    o.stride(0), stream_of(x)),
           "fused_rmsnorm_swiglu");
  return o;
}

at::Tensor fused_rmsnorm_linear(const at::Tensor& x_in, const at::Tensor& w,
                                const c10::optional<at::Tensor>& b_new, double eps,
                                c10::optional<at::Tensor> out, int64_t kernel) {
  TORCH_CHECK(x_in.dim() == 2, "x must be 2D");
  TORCH_CHECK(w.dim() == 2, "W_fused must be 2D");
  TORCH_CHECK(x_in.is_cuda() && w.is_cuda() && (!b_new || b_new->is_cuda()),
              "All tensors must be on CUDA");
  TORCH_CHECK(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf,
              "fused_rmsnorm_linear supports bf16 and fp16 (got ", x_in.scalar_type(), ")");
  TORCH_CHECK(w.scalar_type() == x_in.scalar_type(), "x and W_fused must share one dtype");
  TORCH_CHECK(x_in.size(1) == w.size(1), "x.size(1) (", x_in.size(1), ") != W_fused.size(1) (",
              w.size(1), ")");
  TORCH_CHECK(x_in.device() == w.device(), "x and W_fused must be on the same device");
  // Keep strided row views (k_pass in DeepseekV3 attention); only a
  // non-unit inner stride forces a copy.
  const at::Tensor x = (x_in.stride(1) == 1 || x_in.size(1) == 1) ? x_in : x_in.contiguous();
  const at::Tensor wc = (w.stride(1) == 1) ? w : w.contiguous();
  const int64_t M = x.size(0), K = x.size(1), N = wc.size(0);
  at::Tensor b;
  const void* bptr = nullptr;
  if (b_new && b_new->defined()) {
    TORCH_CHECK(b_new->scalar_type() == x.scalar_type(), "b_new must share x's dtype");
    TORCH_CHECK(b_new->numel() == N, "b_new must have W_fused.size(0) elements");
    b = b_new->contiguous();
    bptr = b.data_ptr();
  }
  at::Tensor o;
  if (out && out->defined()) {
    o = *out;
    TORCH_CHECK(o.dim() == 2 && o.size(0) == M && o.size(1) == N, "out must be [M, N]");
    TORCH_CHECK(o.scalar_type() == x.scalar_type() && o.is_cuda(), "out dtype/device mismatch");
    TORCH_CHECK(o.stride(1) == 1, "out must have unit stride along its last dim");
  } else {
    o = at::empty({M, N}, x.options());
  }
  const c10::cuda::CUDAGuard guard(x.device());
  const int dt = dtype_code(x);
  const size_t ws_bytes = frn_fused_rmsnorm_linear_workspace_size(dt, M, N, K);
  at::Tensor ws;
  if (ws_bytes > 0)
    ws = at::empty({static_cast<int64_t>(ws_bytes)}, x.options().dtype(at::kByte));
  check_rc(frn_fused_rmsnorm_linear_ex(dt, x.data_ptr(), M, K, x.stride(0), wc.data_ptr(), N,
                                       wc.stride(0), bptr, static_cast<float>(eps), o.data_ptr(),
                                       o.stride(0), ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                                       static_cast<int>(kernel), stream_of(x)),
           "fused_rmsnorm_linear");
  return o;
}

// Checks one int8 problem's tensors and fills its C-ABI descriptor; `keep`
// holds the contiguous copies (if any) alive until the launch.
static frn_w8_linear prepare_w8(const at::Tensor& x_in, const at::Tensor& qweight,
                                const at::Tensor& w_scale, const c10::optional<at::Tensor>& b_new,
                                const c10::optional<at::Tensor>& out, std::vector<at::Tensor>& keep) {
  TORCH_CHECK(x_in.dim() == 2 && qweight.dim() == 2, "x and qweight must be 2D");
  TORCH_CHECK(x_in.is_cuda() && qweight.is_cuda() && w_scale.is_cuda() &&
                  (!b_new || b_new->is_cuda()),
              "All tensors must be on CUDA");
  TORCH_CHECK(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf,
              "fused_rmsnorm_linear_w8 takes bf16 or fp16 x");
  TORCH_CHECK(qweight.scalar_type() == at::kChar, "qweight must be int8");
  TORCH_CHECK(w_scale.scalar_type() == at::kFloat && w_scale.numel() == qweight.size(0),
              "w_scale must be fp32 with qweight.size(0) elements");
  TORCH_CHECK(x_in.size(1) == qweight.size(1), "x.size(1) != qweight.size(1)");
  const at::Tensor x = (x_in.stride(1) == 1) ? x_in : x_in.contiguous();
  const at::Tensor q = qweight.stride(1) == 1 ? qweight : qweight.contiguous();
  const at::Tensor sc = w_scale.contiguous();
  const int64_t M = x.size(0), K = x.size(1), N = q.size(0);
  const void* bptr = nullptr;
  if (b_new && b_new->defined()) {
    TORCH_CHECK(b_new->scalar_type() == x.scalar_type() && b_new->numel() == N,
                "b_new must share x's dtype and have qweight.size(0) elements");
    keep.push_back(b_new->contiguous());
    bptr = keep.back().data_ptr();
  }
  at::Tensor o = (out && out->defined()) ? *out : at::empty({M, N}, x.options());
  TORCH_CHECK(o.dim() == 2 && o.size(0) == M && o.size(1) == N && o.stride(1) == 1,
              "out must be [M, N] with unit inner stride");
  keep.push_back(x);
  keep.push_back(q);
  keep.push_back(sc);
  keep.push_back(o);
  frn_w8_linear d;
  d.x = x.data_ptr();
  d.M = M;
  d.K = K;
  d.x_row_stride = x.stride(0);
  d.wq = static_cast<const int8_t*>(q.data_ptr());
  d.N = N;
  d.wq_row_stride = q.stride(0);
  d.w_scale = sc.data_ptr<float>();
  d.bias = bptr;
  d.out = o.data_ptr();
  d.out_row_stride = o.stride(0);
  return d;
}

at::Tensor fused_rmsnorm_linear_w8(const at::Tensor& x_in, const at::Tensor& qweight,
                                   const at::Tensor& w_scale, const c10::optional<at::Tensor>& b_new,
                                   double eps, c10::optional<at::Tensor> out) {
  std::vector<at::Tensor> keep;
  const frn_w8_linear d = prepare_w8(x_in, qweight, w_scale, b_new, out, keep);
  const at::Tensor& x = keep[keep.size() - 4];
  const c10::cuda::CUDAGuard guard(x.device());
  check_rc(frn_fused_rmsnorm_linear_w8(dtype_code(x), d.x, d.M, d.K, d.x_row_stride, d.wq, d.N,
                                       d.wq_row_stride, d.w_scale, d.bias,
                                       static_cast<float>(eps), d.out, d.out_row_stride,
                                       stream_of(x)),
           "fused_rmsnorm_linear_w8");
  return keep.back();
}

// Two independent int8 problems (e.g. a layer's q_b and kv_b) in one launch.
std::tuple<at::Tensor, at::Tensor> fused_rmsnorm_linear_w8_grouped(
    const at::Tensor& x_a, const at::Tensor& qweight_a, const at::Tensor& w_scale_a,
    const c10::optional<at::Tensor>& b_a, const at::Tensor& x_b, const at::Tensor& qweight_b,
    const at::Tensor& w_scale_b, const c10::optional<at::Tensor>& b_b, double eps,
    c10::optional<at::Tensor> out_a, c10::optional<at::Tensor> out_b) {
  TORCH_CHECK(x_a.scalar_type() == x_b.scalar_type() && x_a.device() == x_b.device(),
              "grouped problems must share x's dtype and device");
  std::vector<at::Tensor> keep_a, keep_b;
  frn_w8_linear d[2];
  d[0] = prepare_w8(x_a, qweight_a, w_scale_a, b_a, out_a, keep_a);
  d[1] = prepare_w8(x_b, qweight_b, w_scale_b, b_b, out_b, keep_b);
  const c10::cuda::CUDAGuard guard(x_a.device());
  check_rc(frn_fused_rmsnorm_linear_w8_grouped(dtype_code(x_a), d, 2, static_cast<float>(eps),
                                               stream_of(x_a)),
           "fused_rmsnorm_linear_w8_grouped");
  return {keep_a.back(), keep_b.back()};
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_per_channel(const at::Tensor& w_in) {
  TORCH_CHECK(w_in.dim() == 2, "weight must be 2D");
  TORCH_CHECK(w_in.is_cuda(), "All tensors must be on CUDA");
  const int dt = dtype_code(w_in);
  TORCH_CHECK(dt >= 0, "weight must be fp32, fp16 or bf16");
  const at::Tensor w = w_in.stride(1) == 1 ? w_in : w_in.contiguous();
  const int64_t N = w.size(0), K = w.size(1);
  at::Tensor q = at::empty({N, K}, w.options().dtype(at::kChar));
  at::Tensor sc = at::empty({N}, w.options().dtype(at::kFloat));
  const c10::cuda::CUDAGuard guard(w.device());
  check_rc(frn_quantize_int8_per_channel(dt, w.data_ptr(), N, K, w.stride(0),
                                         static_cast<int8_t*>(q.data_ptr()), K,
                                         sc.data_ptr<float>(), stream_of(w)),
           "quantize_int8_per_channel");
  return {q, sc};
}

int64_t device_error(int64_t device, bool clear) {
  uint32_t flags = 0;
  check_rc(frn_device_error(static_cast<int>(device), &flags, clear ? 1 : 0), "device_error");
  return static_cast<int64_t>(flags);
}

[[noreturn]] void out_of_scope(const char* name) {
  TORCH_CHECK(false, name,
              " belongs to the reference's LayerNorm (OPT) path, which this sm_100a build does "
              "not implement; use the RMSNorm exports");
}

at::Tensor compute_denominator(const at::Tensor&, c10::optional<int64_t>) {
  out_of_scope("compute_denominator");
}
void denominator_normalize(const at::Tensor&, at::Tensor, const at::Tensor&, int64_t, double) {
  out_of_scope("denominator_normalize");
}
at::Tensor compute_denominator_welford(const at::Tensor&, c10::optional<int64_t>) {
  out_of_scope("compute_denominator_welford");
}
void denominator_normalize_welford_512(const at::Tensor&, at::Tensor, const at::Tensor&, int64_t,
                                       double) {
  out_of_scope("denominator_normalize_welford_512");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "B200 (sm_100a) fused RMSNorm -> Linear; RMSNorm exports of the reference module";
  m.def("rmsnorm_normalize", &rmsnorm_normalize,
        "In-place RMSNorm rescale of a GEMM output (256 threads per row)", py::arg("x"),
        py::arg("raw_output"), py::arg("b_new"), py::arg("h"), py::arg("eps"));
  m.def("rmsnorm_normalize_512", &rmsnorm_normalize_512,
        "In-place RMSNorm rescale of a GEMM output (512 threads per row)", py::arg("x"),
        py::arg("raw_output"), py::arg("b_new"), py::arg("h"), py::arg("eps"));
  m.def("fused_rmsnorm_linear_split", &fused_rmsnorm_linear_split,
        "fused_rmsnorm_linear whose output columns are written into separate [M, n_i] tensors",
        py::arg("x"), py::arg("W_fused"), py::arg("b_new"), py::arg("eps"),
        py::arg("split_sizes"));
  m.def("gqa_decode_v2", &gqa_decode_v2,
        "Decode-step GQA attention into output (context split across SMs)", py::arg("q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("output"), py::arg("scale"));
  m.def("gqa_decode_v3", &gqa_decode_v3,
        "Decode-step GQA attention into output (context split across SMs)", py::arg("q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("output"), py::arg("group_size"),
        py::arg("scale"));
  m.def("gqa_prompt_attention", &gqa_prompt_attention,
        "Causal GQA attention over packed prompts: q [T, Hq, D], k / v [T, Hkv, D] -> [T, Hq, Dv]",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cu_seqlens"), py::arg("max_seqlen"),
        py::arg("scale"), py::arg("out") = py::none());
  m.def("gqa_paged_decode", &gqa_paged_decode,
        "Decode-step GQA attention over a paged cache: q [B, Hq, D], pools [P, page_size, Hkv, D]",
        py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
        py::arg("seq_lens"), py::arg("scale"), py::arg("out") = py::none());
  m.def("kv_cache_append", &kv_cache_append,
        "Write k, v [T, Hkv, D] to their sequences' pages, after start_lens tokens",
        py::arg("k"), py::arg("v"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
        py::arg("start_lens"), py::arg("cu_seqlens") = py::none());
  m.def("kv_pages_copy", &kv_pages_copy,
        "Copy pages src[i] -> dst[i] within every pool, one launch", py::arg("pools"),
        py::arg("src"), py::arg("dst"));
  m.def("rmsnorm_swiglu", &rmsnorm_swiglu,
        "RMSNorm + SwiGLU of a [gate | up] GEMM output into output (256 threads per row)",
        py::arg("x"), py::arg("raw_output"), py::arg("output"), py::arg("b_new"), py::arg("h"),
        py::arg("intermediate"), py::arg("eps"));
  m.def("rmsnorm_swiglu_512", &rmsnorm_swiglu_512,
        "RMSNorm + SwiGLU of a [gate | up] GEMM output into output (512 threads per row)",
        py::arg("x"), py::arg("raw_output"), py::arg("output"), py::arg("b_new"), py::arg("h"),
        py::arg("intermediate"), py::arg("eps"));
  m.def("fused_rmsnorm_swiglu", &fused_rmsnorm_swiglu,
        "silu(r * (x @ Wg.T) + bg) * (r * (x @ Wu.T) + bu), r = rsqrt(mean(x^2)+eps); one launch",
        py::arg("x"), py::arg("W_combined"), py::arg("b_combined") = py::none(),
        py::arg("eps") = 1e-6, py::arg("out") = py::none());
  m.def("fused_rmsnorm_linear", &fused_rmsnorm_linear,
        "out = rsqrt(mean(x^2)+eps)[:,None] * (x @ W_fused.T) + b_new, one tcgen05 launch",
        py::arg("x"), py::arg("W_fused"), py::arg("b_new") = py::none(), py::arg("eps") = 1e-6,
        py::arg("out") = py::none(), py::arg("kernel") = 0);
  m.def("fused_rmsnorm_linear_w8", &fused_rmsnorm_linear_w8,
        "int8 weights: rsqrt(mean(x^2)+eps)[:,None] * w_scale * (x @ qweight.T) + b_new",
        py::arg("x"), py::arg("qweight"), py::arg("w_scale"), py::arg("b_new") = py::none(),
        py::arg("eps") = 1e-6, py::arg("out") = py::none());
  m.def("fused_rmsnorm_linear_w8_grouped", &fused_rmsnorm_linear_w8_grouped,
        "two independent int8 fused RMSNorm -> Linear problems in one launch",
        py::arg("x_a"), py::arg("qweight_a"), py::arg("w_scale_a"), py::arg("b_a"),
        py::arg("x_b"), py::arg("qweight_b"), py::arg("w_scale_b"), py::arg("b_b"),
        py::arg("eps") = 1e-6, py::arg("out_a") = py::none(), py::arg("out_b") = py::none());
  m.def("quantize_int8_per_channel", &quantize_int8_per_channel,
        "Symmetric per-output-channel int8 quantization on the GPU -> (qweight, w_scale)",
        py::arg("weight"));
  m.def("device_error", &device_error, "Read (and optionally clear) the device error word",
        py::arg("device") = 0, py::arg("clear") = false);
  m.def("compute_denominator", &compute_denominator, "LayerNorm path: not implemented",
        py::arg("x"), py::arg("stream_ptr") = py::none());
  m.def("denominator_normalize", &denominator_normalize, "LayerNorm path: not implemented",
        py::arg("x"), py::arg("raw_output"), py::arg("b_new"), py::arg("h"), py::arg("eps"));
  m.def("compute_denominator_welford", &compute_denominator_welford,
        "LayerNorm path: not implemented", py::arg("x"), py::arg("stream_ptr") = py::none());
  m.def("denominator_normalize_welford_512", &denominator_normalize_welford_512,
        "LayerNorm path: not implemented", py::arg("x"), py::arg("raw_output"), py::arg("b_new"),
        py::arg("h"), py::arg("eps"));
}
