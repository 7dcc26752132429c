"""CPU oracle of the serving attention operators: packed prompts and the paged
key-value cache.

TEST INFRASTRUCTURE ONLY (see oracle/rmsnorm_linear.py).  Every function is the
operator's definition in fp64 on the CPU.  The attention functions return the
result and, per output element, sum_j p_j |v_j|: the size that rounding p_j (or
an error in it) to a relative u can move that element by is u times this.
"""

from __future__ import annotations

import torch

# Unit roundoff of each type.  An output element carries one rounding of the
# result, and the roundings of the probabilities for the product with v:
# at most u * |out| + u * sum_j p_j |v_j|; twice that covers the approximate
# exponential and fp32 sums (both far below u of the 16-bit types).  For fp32
# the scores dominate: a dot product of 128 terms of size ~1 is off by some
# 1e-6 relative to the scores' own size (a few units), which p takes over as a
# relative error.
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11, torch.float32: 4e-6}


def assert_close(got: torch.Tensor, ref: torch.Tensor, spread: torch.Tensor) -> None:
    """|got - ref| <= 2 u (|ref| + spread) elementwise, and NaN only where ref is."""
    u = UNIT[got.dtype]
    g = got.double().cpu()
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), "NaN in other places than the oracle's"
    # fp16 results near zero are rounded to multiples of 2^-24.
    tiny = 2.0 ** -23 if got.dtype == torch.float16 else 0.0
    off = (g - ref).abs() - 2 * u * (ref.abs() + spread) - tiny
    worst = torch.nan_to_num(off, nan=0.0).max().item() if off.numel() else 0.0
    assert worst <= 0.0, f"off by {worst:.3g} more than the bound"


def assert_same(got: torch.Tensor, ref: torch.Tensor, spread: torch.Tensor) -> None:
    """assert_close, and infinite exactly where ref is, by sign."""
    infinite = torch.isinf(ref)
    g = got.double().cpu()
    assert torch.equal(g[infinite], ref[infinite]), "other infinities than the oracle's"
    assert not torch.isinf(g[~infinite]).any(), "infinities in other places than the oracle's"
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), "NaN in other places than the oracle's"
    assert_close(got[finite.to(got.device)], ref[finite], spread[finite])


def _attend(q, k, v, scale, causal):
    """q [n, Hq, D] against k, v [m, Hkv, *] -> (out, spread) [n, Hq, Dv]."""
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    spread = torch.zeros_like(out)
    if k.shape[0] == 0:
        return out, spread
    for h in range(q.shape[1]):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        if causal:
            for i in range(q.shape[0]):  # nothing after i takes part at all
                p = torch.softmax(kh[: i + 1] @ q[i, h].double() * scale, 0)
                out[i, h] = p @ vh[: i + 1]
                spread[i, h] = p @ vh[: i + 1].abs()
        else:
            p = torch.softmax(q[:, h].double() @ kh.T * scale, 1)
            out[:, h], spread[:, h] = p @ vh, p @ vh.abs()
    return out, spread


def prompt_attention(q, k, v, cu_seqlens, scale):
    """Causal attention of each packed sequence on its own; rows of no sequence are zeros."""
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    spread = torch.zeros_like(out)
    for a, b in zip(cu_seqlens[:-1], cu_seqlens[1:]):
        out[a:b], spread[a:b] = _attend(q[a:b], k[a:b], v[a:b], scale, True)
    return out, spread


def gather_tokens(pages, table_row, n):
    """The n first tokens of one sequence, [n, Hkv, D]."""
    size = pages.shape[1]
    t = torch.arange(n)
    return pages[table_row.long()[t // size], t % size]


def paged_decode(q, k_pages, v_pages, page_table, seq_lens, scale):
    """One query row per sequence against its first seq_lens[b] cached tokens."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    spread = torch.zeros_like(out)
    for b, n in enumerate(seq_lens.tolist()):
        out[b:b + 1], spread[b:b + 1] = _attend(
            q[b:b + 1], gather_tokens(k_pages, page_table[b], n),
            gather_tokens(v_pages, page_table[b], n), scale, False)
    return out, spread


def append(k, v, k_pages, v_pages, page_table, start_lens, cu_seqlens=None):
    """The pools after the append (copies)."""
    k_pages, v_pages = k_pages.clone(), v_pages.clone()
    size = k_pages.shape[1]
    cu = list(range(k.shape[0] + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    for b in range(len(cu) - 1):
        for t in range(cu[b], cu[b + 1]):
            pos = int(start_lens[b]) + t - cu[b]
            page = int(page_table[b, pos // size])
            k_pages[page, pos % size], v_pages[page, pos % size] = k[t], v[t]
    return k_pages, v_pages


def make_paged(lens, page_size, Hkv, D, seed=0, dtype=torch.bfloat16, spare=2, width=None,
               fill=0.0):
    """Pools with every slot that holds a token drawn from N(0, 1) and every other slot `fill`,
    and a shuffled page table whose unused entries are -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_size) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g)[: sum(need)]
    width = max(need + [1]) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.full((total, page_size, Hkv, D), fill, dtype=dtype)
    v = torch.full((total, page_size, Hkv, D), fill, dtype=dtype)
    at = 0
    for b, (n, m) in enumerate(zip(lens, need)):
        table[b, :m] = order[at:at + m].int()
        at += m
        t = torch.arange(n)
        rows = table[b].long()[t // page_size], t % page_size
        k[rows] = torch.randn(n, Hkv, D, generator=g).to(dtype)
        v[rows] = torch.randn(n, Hkv, D, generator=g).to(dtype)
    return k, v, table
