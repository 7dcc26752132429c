"""The paged cache's data movement on the GPU (frn_kv_cache_append,
frn_kv_pages_copy and their Python surface): bit for bit what the CPU oracle
does, and nothing else touched."""
import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def new_tokens(T, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, Hkv, D, generator=g).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("counts,page,Hkv,D", [
    (None, 16, 8, 128), (None, 1, 1, 64), ([1], 8, 2, 128), ([0, 5, 0, 40, 1], 16, 3, 64),
    ([700, 33], 64, 2, 128), ([17] * 50, 24, 1, 64), ([0, 0], 16, 2, 64)])
def test_append(counts, page, Hkv, D, dtype):
    B = 13 if counts is None else len(counts)
    news = [1] * B if counts is None else counts
    starts = [(7 * b) % 40 for b in range(B)]
    k_pages, v_pages, table = orc.make_paged([s + n for s, n in zip(starts, news)], page, Hkv, D,
                                             seed=page, dtype=dtype)
    k, v = new_tokens(sum(news), Hkv, D, dtype, 5)
    cu = None if counts is None else torch.tensor([0] + counts).cumsum(0).int()
    start = torch.tensor(starts, dtype=torch.int32)
    want = orc.append(k, v, k_pages, v_pages, table, start, cu)
    kd, vd = k_pages.to(DEV), v_pages.to(DEV)
    capi.kv_cache_append(k.to(DEV), v.to(DEV), kd, vd, table.to(DEV), start.to(DEV),
                         None if cu is None else cu.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
    assert capi.device_error(0) == 0


def test_append_strides():
    """k and v as views of a QKV projection, pools with heads before tokens."""
    from src.load_gqa_attention import gqa_attention_cuda as ops

    news, starts = [30, 4], [3, 50]
    k_pages, v_pages, table = orc.make_paged([33, 54], 16, 2, 128, seed=1)
    qkv = torch.randn(34, 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16()
    k, v = qkv[:, 4:6], qkv[:, 6:]
    cu, start = torch.tensor([0, 30, 34]).int(), torch.tensor(starts).int()
    want = orc.append(k, v, k_pages, v_pages, table, start, cu)
    pools = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (k_pages, v_pages)]
    qd = qkv.to(DEV)
    ops.kv_cache_append(qd[:, 4:6], qd[:, 6:], *pools, table.to(DEV), start.to(DEV), cu.to(DEV))
    assert torch.equal(pools[0].cpu(), want[0]) and torch.equal(pools[1].cpu(), want[1])
    # Layouts the kernel cannot read are copied first.
    fresh = [t.to(DEV) for t in (k_pages, v_pages)]
    odd = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    ops.kv_cache_append(*odd, *fresh, table.to(DEV), start.to(DEV), cu.to(DEV))
    assert torch.equal(fresh[0].cpu(), want[0]) and torch.equal(fresh[1].cpu(), want[1])


def test_append_outside_the_cache():
    """Tokens of no sequence are skipped; tokens with no page are, and are reported."""
    k_pages, v_pages, table = orc.make_paged([32, 32], 16, 2, 64, seed=3)
    k, v = new_tokens(12, 2, 64, torch.bfloat16, 4)
    args = [t.to(DEV) for t in (k, v)]
    kd, vd = k_pages.to(DEV), v_pages.to(DEV)
    cu = torch.tensor([2, 6, 10]).int()
    start = torch.tensor([30, 4]).int()
    bad = table.clone()
    bad[1, 0] = k_pages.shape[0]
    capi.kv_cache_append(*args, kd, vd, bad.to(DEV), start.to(DEV), cu.to(DEV))
    torch.cuda.synchronize()
    assert capi.device_error(0, clear=True) == capi.FRN_DEVERR_BAD_PAGE
    want_k, want_v = k_pages.clone(), v_pages.clone()
    page = int(table[0, 1])  # of the tokens 2..5 the first two fit, at positions 30 and 31
    want_k[page, 14:], want_v[page, 14:] = k[2:4], v[2:4]
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v)
    capi.kv_cache_append(*args, kd, vd, table.to(DEV), torch.tensor([-1, 60]).int().to(DEV),
                         cu.to(DEV))
    torch.cuda.synchronize()
    assert capi.device_error(0, clear=True) == capi.FRN_DEVERR_BAD_PAGE
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v)


def test_append_then_decode_in_stream_order():
    """The appended token is there for the decode call that follows it."""
    lens = [40, 7]
    k_pages, v_pages, table = orc.make_paged([41, 8], 16, 2, 128, seed=6)
    k, v = new_tokens(2, 2, 128, torch.bfloat16, 7)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(8)).bfloat16()
    start = torch.tensor(lens).int()
    want = orc.append(k, v, k_pages, v_pages, table, start)
    ref, spread = orc.paged_decode(q, *want, table, start + 1, 0.1)
    kd, vd, td = k_pages.to(DEV), v_pages.to(DEV), table.to(DEV)
    qd, kn, vn, sd, ld = (t.to(DEV) for t in (q, k, v, start, start + 1))
    capi.kv_cache_append(kn, vn, kd, vd, td, sd)
    got = capi.gqa_paged_decode_attention(qd, kd, vd, td, ld, 0.1)
    orc.assert_close(got, ref, spread)


@pytest.mark.parametrize("shape,dtype", [((40, 16, 2, 64), torch.bfloat16), ((40, 8), torch.bfloat16),
                                         ((40, 1, 3, 64), torch.float32), ((9, 100000), torch.half)])
@pytest.mark.parametrize("npools", [1, 5, 131])
def test_pages_copy(shape, dtype, npools):
    if npools == 131 and shape[1] == 100000:
        npools = 3
    g = torch.Generator().manual_seed(npools)
    pools = [torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(npools)]
    order = torch.randperm(shape[0], generator=g).tolist()
    n = shape[0] // 2
    src, dst = order[:n], order[n:2 * n]
    src[1] = src[0]  # a page may be copied twice
    want = [p.clone() for p in pools]
    for w in want:
        w[dst] = w[src]
    capi.kv_pages_copy(pools, src, dst)
    torch.cuda.synchronize()
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_pages_copy_many_pairs():
    pools = [torch.randn(6000, 2, 64, device=DEV) for _ in range(2)]
    order = torch.randperm(6000).tolist()
    src, dst = order[:2700], order[2700:5400]
    want = [p.clone() for p in pools]
    for w in want:
        w[dst] = w[src]
    capi.kv_pages_copy(pools, src, dst)
    torch.cuda.synchronize()
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_offsets_past_32_bits():
    """Pools of more than 2^32 elements: tokens appended to the last page, the page copied."""
    P, page, Hkv, D = 4200, 1024, 8, 128
    pools = [torch.zeros(P, page, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    assert pools[0].numel() > 2 ** 32
    k, v = (t.to(DEV) for t in new_tokens(5, Hkv, D, torch.bfloat16, 9))
    table = torch.tensor([[0, P - 1]], dtype=torch.int32, device=DEV)
    start = torch.tensor([2 * page - 5], dtype=torch.int32, device=DEV)
    capi.kv_cache_append(k, v, *pools, table, start, torch.tensor([0, 5]).int().to(DEV))
    capi.kv_pages_copy(pools, [P - 1, P - 1], [P - 3, 1])
    for pool, new in zip(pools, (k, v)):
        for at in (P - 1, P - 3, 1):
            assert torch.equal(pool[at, page - 5:], new) and (pool[at, :page - 5] == 0).all()
        assert (pool[P - 2] == 0).all() and (pool[0] == 0).all()
    assert capi.device_error(0) == 0


def test_pages_copy_surface():
    from src.load_gqa_attention import gqa_attention_cuda as ops

    both = torch.randn(10, 2, 16, 2, 64, device=DEV)  # K and V interleaved: strided pools
    pools = [both[:, 0], both[:, 1]]
    want = both.clone()
    want[[4, 5]] = want[[1, 2]]
    ops.kv_pages_copy(pools, [1, 2], [4, 5])
    assert torch.equal(both, want)
    ops.kv_pages_copy(pools, [], [])
    ops.kv_pages_copy([], [1], [2])
    for src, dst, match in [([1], [10], "outside"), ([-1], [2], "outside"),
                            ([1, 2], [3, 3], "destination of two"), ([1, 2], [2, 3], "both a source"),
                            ([1], [2, 3], "same length")]:
        with pytest.raises(RuntimeError, match=match):
            ops.kv_pages_copy(pools, src, dst)
    with pytest.raises(RuntimeError, match="dense"):
        ops.kv_pages_copy([both[..., :32]], [1], [2])
    with pytest.raises(RuntimeError, match="share shape"):
        ops.kv_pages_copy([both[:, 0], both[:, 1, :8]], [1], [2])
    assert torch.equal(both, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv_pages_copy(pools, [4], [0])
    side.synchronize()
    want[0] = want[4]
    assert torch.equal(both, want)
    assert capi.device_error(0) == 0
