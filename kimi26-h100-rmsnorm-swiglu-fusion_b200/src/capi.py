"""ctypes binding of the C ABI in include/frn_b200.h.

This is the binding a non-torch host would write (a cgo or JNI host binds the
same symbols the same way); the parity tests use it to call libfrn_b200.so
exactly through its extern "C" entry points, passing raw device pointers,
element strides and the current CUDA stream.
"""

from __future__ import annotations

import ctypes
from ctypes import c_char_p, c_float, c_int, c_int64, c_size_t, c_uint32, c_void_p

from src._build import load_library

FRN_OK = 0
FRN_ERR_INVALID_ARGUMENT = 1
FRN_ERR_UNSUPPORTED = 2
FRN_ERR_MISALIGNED = 3
FRN_ERR_WORKSPACE = 4
FRN_ERR_CUDA = 5
FRN_ERR_DEVICE_TIMEOUT = 6

FRN_DTYPE_F32 = 0
FRN_DTYPE_F16 = 1
FRN_DTYPE_BF16 = 2

FRN_DEVERR_WAIT_TIMEOUT = 0x1
FRN_DEVERR_BAD_PAGE = 0x2
FRN_DEVERR_BAD_LENGTH = 0x4

FRN_KERNEL_AUTO = 0
FRN_KERNEL_TILE_N128 = 1
FRN_KERNEL_TILE_N192 = 2
FRN_KERNEL_TILE_N256 = 3
FRN_KERNEL_DECODE = 4
FRN_KERNEL_PAIR_N128 = 5
FRN_KERNEL_PAIR_N160 = 6
FRN_KERNEL_PAIR_N192 = 7
FRN_KERNEL_PAIR_N224 = 8
FRN_KERNEL_PAIR_N256 = 9
FRN_KERNEL_PAIR_AUTO = 10
FRN_KERNEL_WIDE_N128 = 11
FRN_KERNEL_WIDE_N192 = 12
FRN_KERNEL_WIDE_N224 = 13
FRN_KERNEL_WIDE_N256 = 14
FRN_KERNEL_WIDE_N176 = 21

# name -> (restype, argtypes); must cover every function in include/frn_b200.h
class W8Linear(ctypes.Structure):
    """struct frn_w8_linear of include/frn_b200.h (one problem of a grouped
    int8 call)."""
    _fields_ = [("x", c_void_p), ("M", c_int64), ("K", c_int64), ("x_row_stride", c_int64),
                ("wq", c_void_p), ("N", c_int64), ("wq_row_stride", c_int64),
                ("w_scale", c_void_p), ("bias", c_void_p), ("out", c_void_p),
                ("out_row_stride", c_int64)]


class PagedKV(ctypes.Structure):
    """struct frn_paged_kv of include/frn_b200.h."""
    _fields_ = ([("k", c_void_p), ("v", c_void_p)]
                + [(n, c_int64) for n in ("num_pages", "page_size", "num_kv_heads", "head_dim",
                                          "k_page_stride", "k_token_stride", "k_head_stride",
                                          "v_page_stride", "v_token_stride", "v_head_stride")]
                + [("page_table", c_void_p), ("page_table_stride", c_int64),
                   ("max_pages", c_int64)])


PROTOTYPES = {
    "frn_abi_version": (c_int, []),
    "frn_last_error": (c_char_p, []),
    "frn_rmsnorm_normalize": (
        c_int,
        [c_int, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64, c_int64,
         c_float, c_int, c_void_p],
    ),
    "frn_fused_rmsnorm_linear_workspace_size": (c_size_t, [c_int, c_int64, c_int64, c_int64]),
    "frn_fused_rmsnorm_linear": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p,
         c_float, c_void_p, c_int64, c_void_p, c_size_t, c_void_p],
    ),
    "frn_fused_rmsnorm_linear_ex": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p,
         c_float, c_void_p, c_int64, c_void_p, c_size_t, c_int, c_void_p],
    ),
    "frn_fused_rmsnorm_linear_w8": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p,
         c_void_p, c_float, c_void_p, c_int64, c_void_p],
    ),
    "frn_fused_rmsnorm_linear_w8_grouped": (
        c_int, [c_int, ctypes.POINTER(W8Linear), c_int, c_float, c_void_p]),
    "frn_quantize_int8_per_channel": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_void_p, c_void_p],
    ),
    "frn_fused_rmsnorm_linear_split": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p,
         c_float, c_int, ctypes.POINTER(c_int64), ctypes.POINTER(c_void_p),
         ctypes.POINTER(c_int64), c_void_p],
    ),
    "frn_rmsnorm_swiglu": (
        c_int,
        [c_int, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64,
         c_int64, c_int64, c_float, c_int, c_void_p],
    ),
    "frn_fused_rmsnorm_swiglu": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p,
         c_float, c_void_p, c_int64, c_void_p],
    ),
    "frn_gqa_decode_workspace_size": (c_size_t, [c_int64, c_int64, c_int64, c_int64, c_int64]),
    "frn_gqa_decode_attention": (
        c_int,
        [c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_float, c_void_p, c_size_t, c_void_p],
    ),
    "frn_gqa_decode_attention_noalloc": (
        c_int,
        [c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_float, c_void_p],
    ),
    "frn_gqa_prompt_attention": (
        c_int,
        [c_int] + [c_void_p, c_int64, c_int64] * 4
        + [c_void_p] + [c_int64] * 7 + [c_float, c_void_p],
    ),
    "frn_gqa_paged_decode_workspace_size": (c_size_t, [c_int] + [c_int64] * 6),
    "frn_gqa_paged_decode_attention": (
        c_int,
        [c_int, c_void_p, c_int64, c_int64, ctypes.POINTER(PagedKV), c_void_p, c_void_p, c_int64,
         c_int64, c_int64, c_int64, c_float, c_void_p, c_size_t, c_void_p],
    ),
    "frn_kv_cache_append": (
        c_int,
        [c_int] + [c_void_p, c_int64, c_int64] * 2
        + [ctypes.POINTER(PagedKV), c_void_p, c_void_p, c_int64, c_int64, c_void_p],
    ),
    "frn_kv_pages_copy": (
        c_int,
        [ctypes.POINTER(c_void_p), c_int64, c_int64, c_int64, c_int64, ctypes.POINTER(ctypes.c_int32),
         ctypes.POINTER(ctypes.c_int32), c_int64, c_void_p],
    ),
    "frn_device_error": (c_int, [c_int, ctypes.POINTER(c_uint32), c_int]),
    "frn_selftest_wait_timeout": (c_int, [c_int, c_void_p]),
}

_lib = None


class FrnError(RuntimeError):
    def __init__(self, code: int, what: str, message: str):
        super().__init__(f"{what} failed (status {code}): {message}")
        self.code = code


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        handle = load_library()
        for name, (res, args) in PROTOTYPES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def last_error() -> str:
    return lib().frn_last_error().decode()


def check(rc: int, what: str) -> None:
    if rc != FRN_OK:
        raise FrnError(rc, what, last_error())


# ------------------------------------------------------------ torch helpers
def _dtype_code(t) -> int:
    import torch

    return {torch.float32: FRN_DTYPE_F32, torch.float16: FRN_DTYPE_F16,
            torch.bfloat16: FRN_DTYPE_BF16}[t.dtype]


def _stream_ptr(device) -> int:
    import torch

    return torch.cuda.current_stream(device).cuda_stream


def _on(device):
    """Makes `device` current for the call: every frn_* entry point works on
    the caller's current CUDA device (its SM count, its static scratch)."""
    import torch

    return torch.cuda.device(device)


def workspace_size(dtype_code: int, M: int, N: int, K: int) -> int:
    return int(lib().frn_fused_rmsnorm_linear_workspace_size(dtype_code, M, N, K))


def fused_rmsnorm_linear(x, w, bias=None, eps: float = 1e-6, out=None,
                         kernel: int = FRN_KERNEL_AUTO, workspace=None):
    """out = rsqrt(mean(x^2)+eps)[:,None] * (x @ w.T) + bias through the C ABI.

    x: [M, K] with unit inner stride (any 16B-legal row stride); w: [N, K].
    """
    import torch

    assert x.dim() == 2 and w.dim() == 2 and x.stride(1) == 1 and w.stride(1) == 1
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=x.dtype, device=x.device)
    dt = _dtype_code(x)
    need = workspace_size(dt, M, N, K)
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() if workspace is not None else 0
    with _on(x.device):
        rc = lib().frn_fused_rmsnorm_linear_ex(
            dt, x.data_ptr(), M, K, x.stride(0), w.data_ptr(), N, w.stride(0),
            bias.data_ptr() if bias is not None else None, float(eps), out.data_ptr(),
            out.stride(0), ws_ptr, ws_bytes, int(kernel), _stream_ptr(x.device))
    check(rc, "frn_fused_rmsnorm_linear")
    return out


def rmsnorm_normalize(x, raw_output, b_new, h: int, eps: float, threads: int = 256):
    """In-place raw_output = raw_output * inv_rms(x) + b_new through the C ABI."""
    with _on(x.device):
        rc = lib().frn_rmsnorm_normalize(
            _dtype_code(x), x.data_ptr(), x.stride(0), raw_output.data_ptr(), raw_output.stride(0),
            b_new.data_ptr(), x.shape[0], h, raw_output.shape[1], float(eps), int(threads),
            _stream_ptr(x.device))
    check(rc, "frn_rmsnorm_normalize")
    return raw_output


def fused_rmsnorm_linear_w8(x, wq, w_scale, bias=None, eps: float = 1e-6, out=None):
    """out = inv_rms[:,None] * w_scale[None,:] * (x @ wq.T) + bias (int8 wq)."""
    import torch

    assert x.dim() == 2 and wq.dim() == 2 and x.stride(1) == 1 and wq.stride(1) == 1
    M, K = x.shape
    N = wq.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = lib().frn_fused_rmsnorm_linear_w8(
            _dtype_code(x), x.data_ptr(), M, K, x.stride(0), wq.data_ptr(), N, wq.stride(0),
            w_scale.data_ptr(), bias.data_ptr() if bias is not None else None, float(eps),
            out.data_ptr(), out.stride(0), _stream_ptr(x.device))
    check(rc, "frn_fused_rmsnorm_linear_w8")
    return out


def fused_rmsnorm_linear_w8_grouped(problems, eps: float = 1e-6):
    """One launch for one or two independent int8 problems, each a tuple
    (x, wq, w_scale, bias, out) as in fused_rmsnorm_linear_w8 (out required);
    returns the outputs."""
    assert 1 <= len(problems) <= 2
    arr = (W8Linear * len(problems))()
    for a, (x, wq, w_scale, bias, out) in zip(arr, problems):
        assert x.dim() == 2 and wq.dim() == 2 and x.stride(1) == 1 and wq.stride(1) == 1
        assert x.device == problems[0][0].device and x.dtype == problems[0][0].dtype
        a.x, a.M, a.K, a.x_row_stride = x.data_ptr(), x.shape[0], x.shape[1], x.stride(0)
        a.wq, a.N, a.wq_row_stride = wq.data_ptr(), wq.shape[0], wq.stride(0)
        a.w_scale = w_scale.data_ptr()
        a.bias = bias.data_ptr() if bias is not None else None
        a.out, a.out_row_stride = out.data_ptr(), out.stride(0)
    x0 = problems[0][0]
    with _on(x0.device):
        rc = lib().frn_fused_rmsnorm_linear_w8_grouped(_dtype_code(x0), arr, len(problems),
                                                       float(eps), _stream_ptr(x0.device))
    check(rc, "frn_fused_rmsnorm_linear_w8_grouped")
    return [p[4] for p in problems]


def quantize_int8_per_channel(w):
    """(q int8 [N,K], scale fp32 [N]) of a weight on the GPU."""
    import torch

    N, K = w.shape
    q = torch.empty(N, K, dtype=torch.int8, device=w.device)
    scale = torch.empty(N, dtype=torch.float32, device=w.device)
    with _on(w.device):
        rc = lib().frn_quantize_int8_per_channel(_dtype_code(w), w.data_ptr(), N, K, w.stride(0),
                                                 q.data_ptr(), K, scale.data_ptr(),
                                                 _stream_ptr(w.device))
    check(rc, "frn_quantize_int8_per_channel")
    return q, scale


def fused_rmsnorm_linear_split(x, w, bias, eps: float, split_sizes, outs=None):
    """Fused RMSNorm -> Linear whose output columns land directly in
    len(split_sizes) separate [M, n_i] tensors (returned as a list)."""
    import torch

    assert x.dim() == 2 and w.dim() == 2 and x.stride(1) == 1 and w.stride(1) == 1
    M, K = x.shape
    N = w.shape[0]
    n = len(split_sizes)
    if outs is None:
        outs = [torch.empty(M, c, dtype=x.dtype, device=x.device) for c in split_sizes]
    cols = (c_int64 * n)(*[int(c) for c in split_sizes])
    ptrs = (c_void_p * n)(*[o.data_ptr() for o in outs])
    strides = (c_int64 * n)(*[o.stride(0) for o in outs])
    with _on(x.device):
        rc = lib().frn_fused_rmsnorm_linear_split(
            _dtype_code(x), x.data_ptr(), M, K, x.stride(0), w.data_ptr(), N, w.stride(0),
            bias.data_ptr() if bias is not None else None, float(eps), n, cols, ptrs, strides,
            _stream_ptr(x.device))
    check(rc, "frn_fused_rmsnorm_linear_split")
    return outs


def rmsnorm_swiglu(x, raw_output, output, b_new, h: int, intermediate: int, eps: float,
                   threads: int = 256):
    """output = silu(g * inv_rms + b_g) * (u * inv_rms + b_u) of a [gate | up]
    GEMM output, through the C ABI."""
    with _on(x.device):
        rc = lib().frn_rmsnorm_swiglu(
            _dtype_code(x), x.data_ptr(), x.stride(0), raw_output.data_ptr(), raw_output.stride(0),
            output.data_ptr(), output.stride(0), b_new.data_ptr(), x.shape[0], h, intermediate,
            float(eps), int(threads), _stream_ptr(x.device))
    check(rc, "frn_rmsnorm_swiglu")
    return output


def fused_rmsnorm_swiglu(x, w_combined, bias=None, eps: float = 1e-6, out=None):
    """One-launch RMSNorm -> [gate | up] projection -> SwiGLU through the C ABI.

    x: [M, K]; w_combined: [2I, K] (gate rows first); bias: [2I] or None;
    returns out [M, I]."""
    import torch

    assert x.dim() == 2 and w_combined.dim() == 2 and x.stride(1) == 1
    assert w_combined.stride(1) == 1 and w_combined.shape[0] % 2 == 0
    M, K = x.shape
    inter = w_combined.shape[0] // 2
    if out is None:
        out = torch.empty(M, inter, dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = lib().frn_fused_rmsnorm_swiglu(
            _dtype_code(x), x.data_ptr(), M, K, x.stride(0), w_combined.data_ptr(), inter,
            w_combined.stride(0), bias.data_ptr() if bias is not None else None, float(eps),
            out.data_ptr(), out.stride(0), _stream_ptr(x.device))
    check(rc, "frn_fused_rmsnorm_swiglu")
    return out


def gqa_decode_attention(q, k_cache, v_cache, scale: float, out=None, use_workspace=True):
    """Decode-step GQA attention through the C ABI: q [B, Hq, D], caches
    [B, T, Hkv, D] (contiguous); returns out [B, Hq, D]."""
    import torch

    B, Hq, D = q.shape
    T, Hkv = k_cache.shape[1], k_cache.shape[2]
    if out is None:
        out = torch.empty_like(q)
    with _on(q.device):
        ws_bytes = (int(lib().frn_gqa_decode_workspace_size(B, Hq, Hkv, D, T))
                    if use_workspace else 0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    with _on(q.device):
        rc = lib().frn_gqa_decode_attention(
            _dtype_code(q), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
            B, Hq, Hkv, D, T, float(scale), ws.data_ptr() if ws is not None else None, ws_bytes,
            _stream_ptr(q.device))
    check(rc, "frn_gqa_decode_attention")
    return out


def gqa_decode_attention_noalloc(q, k_cache, v_cache, scale: float, out):
    """frn_gqa_decode_attention_noalloc: the library's static scratch instead of
    a workspace; `out` must be preallocated (nothing is allocated here)."""
    B, Hq, D = q.shape
    T, Hkv = k_cache.shape[1], k_cache.shape[2]
    with _on(q.device):
        rc = lib().frn_gqa_decode_attention_noalloc(
            _dtype_code(q), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
            B, Hq, Hkv, D, T, float(scale), _stream_ptr(q.device))
    check(rc, "frn_gqa_decode_attention_noalloc")
    return out


def _check_heads(like, **tensors) -> None:
    """3-D tensors [tokens, heads, dim] of like's dtype and device, unit stride along dim."""
    for name, t in tensors.items():
        assert t.dim() == 3 and t.dtype == like.dtype and t.device == like.device, name
        assert t.stride(2) == 1 or t.shape[2] == 1 or t.numel() == 0, name


def _check_ints(like, **tensors) -> None:
    """int32 tensors on like's device, unit stride along the last dim."""
    for name, t in tensors.items():
        assert str(t.dtype) == "torch.int32" and t.device == like.device, name
        assert t.stride(-1) == 1 or t.shape[-1] <= 1 or t.numel() == 0, name


def gqa_prompt_attention(q, k, v, cu_seqlens, max_seqlen: int, scale: float, out=None):
    """Causal attention over packed prompts through the C ABI: q [T, Hq, Dqk],
    k [T, Hkv, Dqk], v [T, Hkv, Dv], cu_seqlens int32 [B + 1] on the GPU;
    returns out [T, Hq, Dv]."""
    import torch

    _check_heads(q, q=q, k=k, v=v)
    _check_ints(q, cu_seqlens=cu_seqlens)
    T, Hq, Dqk = q.shape
    Hkv, Dv = v.shape[1], v.shape[2]
    assert tuple(k.shape) == (T, Hkv, Dqk) and v.shape[0] == T
    assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1
    if out is None:
        out = torch.empty(T, Hq, Dv, dtype=q.dtype, device=q.device)
    _check_heads(q, out=out)
    assert tuple(out.shape) == (T, Hq, Dv)
    with _on(q.device):
        rc = lib().frn_gqa_prompt_attention(
            _dtype_code(q), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
            k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), out.stride(0),
            out.stride(1), cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, T, int(max_seqlen), Hq,
            Hkv, Dqk, Dv, float(scale), _stream_ptr(q.device))
    check(rc, "frn_gqa_prompt_attention")
    return out


def paged_kv(k_pages, v_pages, page_table) -> PagedKV:
    """The struct frn_paged_kv of pools [P, page_size, Hkv, D] and a table [B, max_pages]."""
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape
    assert k_pages.dtype == v_pages.dtype and k_pages.device == v_pages.device
    assert (k_pages.stride(3) == 1 and v_pages.stride(3) == 1) or k_pages.numel() == 0
    assert page_table.dim() == 2
    _check_ints(k_pages, page_table=page_table)
    P, page_size, Hkv, D = k_pages.shape
    return PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), P, page_size, Hkv, D,
                   k_pages.stride(0), k_pages.stride(1), k_pages.stride(2), v_pages.stride(0),
                   v_pages.stride(1), v_pages.stride(2), page_table.data_ptr(),
                   page_table.stride(0), page_table.shape[1])


def gqa_paged_decode_attention(q, k_pages, v_pages, page_table, seq_lens, scale: float, out=None,
                               workspace=None):
    """Decode-step GQA attention over a paged cache through the C ABI: q
    [B, Hq, D], pools [P, page_size, Hkv, D], page_table int32 [B, max_pages]
    and seq_lens int32 [B] on the GPU; returns out [B, Hq, D]."""
    import torch

    _check_heads(q, q=q)
    _check_ints(q, seq_lens=seq_lens)
    B, Hq, D = q.shape
    if out is None:
        out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    _check_heads(q, out=out)
    assert out.shape == q.shape
    cache = paged_kv(k_pages, v_pages, page_table)
    assert k_pages.dtype == q.dtype and k_pages.device == q.device and k_pages.shape[3] == D
    assert tuple(seq_lens.shape) == (B,) and page_table.shape[0] == B
    with _on(q.device):
        if workspace is None:
            need = lib().frn_gqa_paged_decode_workspace_size(
                _dtype_code(q), B, Hq, cache.num_kv_heads, D, cache.page_size, cache.max_pages)
            workspace = torch.empty(int(need), dtype=torch.uint8, device=q.device)
        rc = lib().frn_gqa_paged_decode_attention(
            _dtype_code(q), q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(cache),
            seq_lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), B, Hq, float(scale),
            workspace.data_ptr(), workspace.numel(), _stream_ptr(q.device))
    check(rc, "frn_gqa_paged_decode_attention")
    return out


def kv_cache_append(k, v, k_pages, v_pages, page_table, start_lens, cu_seqlens=None) -> None:
    """Writes k, v [T, Hkv, D] to their sequences' pages through the C ABI."""
    _check_heads(k, k=k, v=v)
    _check_ints(k, start_lens=start_lens)
    assert k.shape == v.shape and k.shape[1:] == k_pages.shape[2:]
    cache = paged_kv(k_pages, v_pages, page_table)
    assert k_pages.dtype == k.dtype and k_pages.device == k.device
    assert start_lens.dim() == 1 and page_table.shape[0] == start_lens.numel()
    if cu_seqlens is not None:
        _check_ints(k, cu_seqlens=cu_seqlens)
        assert tuple(cu_seqlens.shape) == (start_lens.numel() + 1,)
    with _on(k.device):
        rc = lib().frn_kv_cache_append(
            _dtype_code(k), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), ctypes.byref(cache), start_lens.data_ptr(),
            cu_seqlens.data_ptr() if cu_seqlens is not None else None, start_lens.numel(),
            k.shape[0], _stream_ptr(k.device))
    check(rc, "frn_kv_cache_append")


def kv_pages_copy(pools, src, dst) -> None:
    """Copies pages src[i] -> dst[i] in every pool [P, ...] through the C ABI."""
    n = len(src)
    assert len(dst) == n and all(p.shape == pools[0].shape and p.stride() == pools[0].stride()
                                 and p.dtype == pools[0].dtype and p.device == pools[0].device
                                 for p in pools)
    if pools[0].shape[0]:  # a page is one block, its dims in any order
        page = pools[0][0]
        order = sorted(range(page.dim()), key=lambda i: (-page.stride(i), -page.shape[i]))
        assert page.permute(order).is_contiguous()
    ptrs = (c_void_p * len(pools))(*[p.data_ptr() for p in pools])
    first = pools[0]
    es = first.element_size()
    with _on(first.device):
        rc = lib().frn_kv_pages_copy(
            ptrs, len(pools), first.shape[0], first[0].numel() * es, first.stride(0) * es,
            (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, _stream_ptr(first.device))
    check(rc, "frn_kv_pages_copy")


def selftest_wait_timeout(timeout_ms: int, stream=None) -> None:
    """Launch the bounded-wait self-test kernel (see include/frn_b200.h)."""
    check(lib().frn_selftest_wait_timeout(int(timeout_ms), stream), "frn_selftest_wait_timeout")


def device_error(device: int = 0, clear: bool = False) -> int:
    flags = c_uint32(0)
    check(lib().frn_device_error(device, ctypes.byref(flags), 1 if clear else 0),
          "frn_device_error")
    return int(flags.value)
