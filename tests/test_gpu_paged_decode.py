"""GPU parity of decode attention over a paged cache
(frn_gqa_paged_decode_attention and its Python surface) against the fp64 CPU
oracle."""
import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"


def queries(B, Hq, D, dtype, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    return torch.randn(B, Hq, D, generator=g).to(dtype)


def run(q, k, v, table, lens, scale, **kw):
    got = capi.gqa_paged_decode_attention(
        q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV),
        torch.tensor(lens, dtype=torch.int32, device=DEV), scale, **kw)
    torch.cuda.synchronize()
    return got


def check(lens, Hq, Hkv, D, page, dtype=torch.bfloat16, seed=0, scale=None, **kw):
    scale = D ** -0.5 if scale is None else scale
    k, v, table = orc.make_paged(lens, page, Hkv, D, seed=seed, dtype=dtype, **kw)
    q = queries(len(lens), Hq, D, dtype, seed)
    got = run(q, k, v, table, lens, scale)
    ref, spread = orc.paged_decode(q, torch.nan_to_num(k), torch.nan_to_num(v), table,
                                   torch.tensor(lens), scale)
    orc.assert_close(got, ref, spread)
    assert capi.device_error(0) == 0


DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
LENS = [[1], [16, 17, 15], [0, 64, 0, 65, 63], [1000], [4096, 1, 0, 333], [0], [0, 0],
        [129] * 40, list(range(300))]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_lengths(lens, dtype):
    check(lens, 8, 2, 128, 16, dtype=dtype, seed=len(lens))


@pytest.mark.parametrize("page", [1, 3, 8, 24, 32, 64, 128, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(page, D):
    check([777, 5, 64], 8, 4, D, page, seed=page)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (6, 2), (7, 1), (8, 1), (9, 1), (28, 4),
                                    (26, 2), (16, 1), (64, 8)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_head_layouts(Hq, Hkv, D, dtype):
    check([200, 31], Hq, Hkv, D, 16, dtype=dtype, seed=Hq)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_long_context(dtype):
    check([40000, 3], 4, 1, 64, 32, dtype=dtype, seed=2)


def test_many_sequences():
    check([(37 * i) % 211 for i in range(700)], 4, 2, 64, 16, seed=3)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_scales(dtype):
    for scale in (0.0, 3.0, -0.2):
        check([500], 8, 2, 128, 16, dtype=dtype, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_unused_slots_have_no_effect(dtype):
    """NaN in every slot past the lengths and in every page of no sequence."""
    check([100, 1, 0, 65], 8, 2, 128, 48, dtype=dtype, seed=5, fill=float("nan"), spare=4, width=9)


def test_shared_pages_and_wide_tables():
    k, v, table = orc.make_paged([100, 100, 40], 16, 2, 128, seed=6, width=40)
    table[1] = table[0]
    lens = [100, 90, 40]
    q = queries(3, 8, 128, k.dtype, 6)
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor(lens), 0.1)
    orc.assert_close(run(q, k, v, table, lens, 0.1), ref, spread)


def test_strides():
    """Pools with heads before tokens, K and V interleaved in one tensor, a
    table and queries that are views."""
    lens = [70, 33]
    k, v, table = orc.make_paged(lens, 16, 2, 128, seed=7)
    q = queries(2, 8, 128, k.dtype, 7)
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor(lens), 0.1)
    both = torch.stack((k, v), 1).to(DEV)  # [P, 2, page, Hkv, D]
    hnd = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    wide_q = torch.zeros(2, 16, 256, dtype=q.dtype, device=DEV)[:, ::2, 128:]
    wide_q.copy_(q)
    wide_t = torch.full((2, 50), 99, dtype=torch.int32, device=DEV)[:, 7:7 + table.shape[1]]
    wide_t.copy_(table)
    out = torch.full((2, 8, 256), 5.0, dtype=q.dtype, device=DEV)
    orc.assert_close(run(wide_q, both[:, 0], both[:, 1], wide_t, lens, 0.1, out=out[..., :128]),
                     ref, spread)
    assert (out[..., 128:] == 5).all()
    orc.assert_close(run(q, hnd[0], both[:, 1], table, lens, 0.1), ref, spread)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, the sequence in its last pages."""
    P, page, Hkv, D = 4200, 1024, 8, 128
    pool = torch.empty(P, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    k, v, table = orc.make_paged([1500], page, Hkv, D, seed=8)
    pool[P - k.shape[0]:] = k.to(DEV)
    vp = torch.empty(P, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vp[P - k.shape[0]:] = v.to(DEV)
    q = queries(1, 16, D, k.dtype, 8)
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor([1500]), 0.1)
    got = run(q, pool, vp, table + (P - k.shape[0]), [1500], 0.1)
    orc.assert_close(got, ref, spread)


def test_pages_and_lengths_outside_the_cache():
    k, v, table = orc.make_paged([64, 64], 16, 2, 128, seed=9)
    q = queries(2, 8, 128, k.dtype, 9)
    bad = table.clone()
    bad[0, 1] = k.shape[0]
    bad[1, 2] = -1
    got = run(q, k, v, bad, [64, 64], 0.1)
    assert capi.device_error(0, clear=True) == capi.FRN_DEVERR_BAD_PAGE
    assert torch.isfinite(got.float()).all()
    got = run(q, k, v, table, [1000, -3], 0.1)
    assert capi.device_error(0, clear=True) == capi.FRN_DEVERR_BAD_PAGE
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor([64, 0]), 0.1)
    orc.assert_close(got, ref, spread)


def test_streams_graphs_and_repeats():
    lens = [900, 64, 2000]
    k, v, table = orc.make_paged(lens, 16, 2, 128, seed=10)
    q = queries(3, 8, 128, k.dtype, 10)
    first = run(q, k, v, table, lens, 0.1)
    args = [t.to(DEV) for t in (q, k, v, table)]
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            again = capi.gqa_paged_decode_attention(*args, lens_d, 0.1)
    side.synchronize()
    assert torch.equal(first, again)
    # A captured call serves other lengths: they are read on the device.
    ws = torch.empty(int(capi.lib().frn_gqa_paged_decode_workspace_size(
        capi.FRN_DTYPE_BF16, 3, 8, 2, 128, 16, table.shape[1])), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.gqa_paged_decode_attention(*args, lens_d, 0.1, out=out, workspace=ws)
    for other in ([1, 0, 1999], [900, 64, 2000], [0, 0, 0]):
        lens_d.copy_(torch.tensor(other, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref, spread = orc.paged_decode(q, k, v, table, torch.tensor(other), 0.1)
        orc.assert_close(out, ref, spread)


def test_python_surface():
    from src.gqa_attention_forward import GQAPagedDecodeAttention
    from src.load_gqa_attention import gqa_attention_cuda as ops

    lens = [70, 0, 33]
    k, v, table = orc.make_paged(lens, 16, 2, 128, seed=12)
    q = queries(3, 8, 128, k.dtype, 12)
    qd, kd, vd, td = (t.to(DEV) for t in (q, k, v, table))
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor(lens), 0.1)
    orc.assert_close(ops.gqa_paged_decode(qd, kd, vd, td, ld, 0.1), ref, spread)
    module = GQAPagedDecodeAttention(8, 2, 128, scale=0.1)
    orc.assert_close(module(qd, kd, vd, td, ld), ref, spread)
    orc.assert_close(module(qd.flatten(1), kd, vd, td, ld), ref, spread)
    assert ops.gqa_paged_decode(qd[:0], kd, vd, td[:0], ld[:0], 0.1).shape == (0, 8, 128)
    for args, match in [((qd.half(), kd, vd, td, ld), "dtype"),
                        ((qd[:, :7], kd, vd, td, ld), "multiple of num_kv_heads"),
                        ((qd, kd, vd[:, :8], td, ld), "pools"),
                        ((qd, kd, vd, td[:2], ld), "entry per sequence"),
                        ((qd, kd, vd, td.long(), ld), "int32"),
                        ((qd, kd, vd, td, ld.cpu()), "CUDA"),
                        ((qd.repeat(1, 5, 1), kd, vd, td, ld), "at most 16")]:
        with pytest.raises(RuntimeError, match=match):
            ops.gqa_paged_decode(*args, 0.1)
    with pytest.raises(capi.FrnError, match="workspace"):
        capi.gqa_paged_decode_attention(qd, kd, vd, td, ld, 0.1,
                                        workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    assert capi.device_error(0) == 0
