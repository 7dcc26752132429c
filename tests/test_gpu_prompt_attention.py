"""GPU parity of causal attention over packed prompts (frn_gqa_prompt_attention
and its Python surface) against the fp64 CPU oracle."""
import itertools

import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"


def cumulate(lens):
    return [0] + list(itertools.accumulate(lens))


def make(lens, Hq, Hkv, Dqk, Dv, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q = torch.randn(T, Hq, Dqk, generator=g).to(dtype)
    k = torch.randn(T, Hkv, Dqk, generator=g).to(dtype)
    v = torch.randn(T, Hkv, Dv, generator=g).to(dtype)
    return q, k, v, cumulate(lens)


def run(q, k, v, cu, scale, longest=None, out=None):
    lens = [b - a for a, b in zip(cu[:-1], cu[1:])]
    got = capi.gqa_prompt_attention(
        q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV),
        max(lens + [0]) if longest is None else longest, scale, out=out)
    torch.cuda.synchronize()
    return got


def check(lens, Hq, Hkv, Dqk, Dv, dtype=torch.bfloat16, seed=0, scale=None, change=None):
    q, k, v, cu = make(lens, Hq, Hkv, Dqk, Dv, dtype, seed)
    if change is not None:
        change(q, k, v, cu)
    scale = Dqk ** -0.5 if scale is None else scale
    got = run(q, k, v, cu, scale)
    ref, spread = orc.prompt_attention(q, k, v, cu, scale)
    orc.assert_close(got, ref, spread)
    assert capi.device_error(0) == 0


LENS = [
    [1],
    [2, 1, 5],
    [77],
    [127, 128, 129],
    [64, 0, 0, 65, 31, 1, 32, 33],
    [300],
    [513, 17],
    list(range(1, 40)),
]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:6])))
@pytest.mark.parametrize("heads", [(8, 2, 128, 128), (7, 1, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
def test_lengths(lens, heads):
    check(lens, *heads, seed=sum(lens))


@pytest.mark.parametrize("heads", [(1, 1, 128, 128), (3, 1, 128, 128), (10, 2, 128, 128),
                                   (16, 1, 128, 128), (32, 2, 64, 64), (71, 1, 64, 64),
                                   (128, 1, 64, 64), (6, 3, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_head_layouts(heads, dtype):
    check([130, 3, 45], *heads, dtype=dtype, seed=7)


@pytest.mark.parametrize("heads", [(4, 1, 128, 128), (2, 2, 192, 128), (2, 1, 64, 64)],
                         ids=lambda x: "x".join(map(str, x)))
def test_long_sequence(heads):
    check([1411, 700], *heads, seed=9)


@pytest.mark.parametrize("heads", [(4, 4, 128, 128), (2, 2, 192, 128), (8, 4, 64, 64)],
                         ids=lambda x: "x".join(map(str, x)))
@pytest.mark.parametrize("length", [40, 128, 160, 257, 300, 390])
def test_many_items(heads, length):
    """Several work items for every SM, with one or two row tiles each."""
    lens = [length, max(1, length // 2), length - 3, 0] * 60
    q, k, v, cu = make(lens, *heads, seed=length)
    got = run(q, k, v, cu, 0.1)
    assert capi.device_error(0) == 0
    some = [0, 1, 2, 117, 238]
    for b in some:
        a, e = cu[b], cu[b + 1]
        ref, spread = orc.prompt_attention(q[a:e], k[a:e], v[a:e], [0, e - a], 0.1)
        orc.assert_close(got[a:e], ref, spread)
    # The others against the same sequence run alone (same tiles, same bits).
    for b in range(len(lens)):
        a, e = cu[b], cu[b + 1]
        if b % 7 == 0 and e > a:
            alone = run(q[a:e], k[a:e], v[a:e], [0, e - a], 0.1)
            assert torch.equal(got[a:e], alone)


@pytest.mark.parametrize("Dqk,Dv", [(128, 128), (64, 64), (192, 128)])
def test_running_maximum(Dqk, Dv):
    """Scores that grow along the sequence move the maximum at every step; large
    ones put nearly all weight on one key."""
    def grow(q, k, v, cu):
        q[:, :, 0] = 8.0
        k[:, :, 0] = torch.linspace(-60, 60, k.shape[0])[:, None].to(k.dtype)

    def shrink(q, k, v, cu):
        q[:, :, 0] = 8.0
        k[:, :, 0] = torch.linspace(60, -60, k.shape[0])[:, None].to(k.dtype)

    for change in (grow, shrink):
        check([600], 2, 1, Dqk, Dv, seed=3, change=change)
    check([300], 2, 1, Dqk, Dv, seed=4, scale=4.0)
    check([300], 2, 1, Dqk, Dv, seed=5, scale=0.0)
    check([300], 2, 1, Dqk, Dv, seed=6, scale=-0.1)


@pytest.mark.parametrize("Dqk,Dv", [(128, 128), (64, 64), (192, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_later_tokens_have_no_effect(Dqk, Dv, bad):
    """Row i does not see what lies in k and v after it, whatever it is: not in
    its own sequence, not in the next one."""
    lens = [130, 40, 300]
    q, k, v, cu = make(lens, 4, 2, Dqk, Dv, seed=11)
    scale = Dqk ** -0.5
    ref, spread = orc.prompt_attention(q, k, v, cu, scale)
    for at in (cu[1] - 1, cu[1], cu[2] + 1, cu[2] + 77, cu[3] - 2):
        k2, v2 = k.clone(), v.clone()
        k2[at, :, 3] = bad
        v2[at, :, 5] = bad
        got = run(q, k2, v2, cu, scale).double().cpu()
        rows = torch.arange(cu[-1])
        seq_end = next(e for e in cu[1:] if at < e)
        clean = (rows < at) | (rows >= seq_end)
        orc.assert_close(got[clean].to(q.dtype), ref[clean], spread[clean])


def test_strided_views():
    """q, k and v as views of one QKV projection, V the tail of a [nope | V]
    block, heads before tokens; the output a view too."""
    T, Hq, Hkv, D = 150, 4, 2, 128
    lens, cu = [100, 50], [0, 100, 150]
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    ref, spread = orc.prompt_attention(q.cpu(), k.cpu(), v.cpu(), cu, 0.1)
    out = torch.full((T, Hq, 2 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    run(q, k, v, cu, 0.1, out=out[..., D:])
    orc.assert_close(out[..., D:], ref, spread)
    assert (out[..., :D] == 7).all()
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    orc.assert_close(run(*by_head, cu, 0.1), ref, spread)

    k = torch.randn(T, Hkv, 192, generator=g).to(torch.bfloat16)
    kv = torch.randn(T, Hkv, 256, generator=g).to(torch.bfloat16)
    q = torch.randn(T, Hq, 192, generator=g).to(torch.bfloat16)
    ref, spread = orc.prompt_attention(q, k, kv[..., 128:], cu, 0.07)
    orc.assert_close(run(q, k, kv.to(DEV)[..., 128:], cu, 0.07), ref, spread)


def test_offsets_past_32_bits():
    """More than 2^32 elements of q and out; the first and the last sequence are looked at."""
    n, count, Hq, Hkv, D = 100, 2700, 128, 8, 128
    q = torch.zeros(n * count, Hq, D, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(n * count, Hkv, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(n * count, Hkv, D, dtype=torch.bfloat16, device=DEV)
    assert q.numel() > 2 ** 32
    q1, k1, v1, _ = make([n], Hq, Hkv, D, D, seed=13)
    for rows in (slice(0, n), slice(n * (count - 1), None)):
        q[rows], k[rows], v[rows] = q1.to(DEV), k1.to(DEV), v1.to(DEV)
    cu = torch.arange(count + 1, dtype=torch.int32, device=DEV) * n
    got = capi.gqa_prompt_attention(q, k, v, cu, n, 0.1)
    ref, spread = orc.prompt_attention(q1, k1, v1, [0, n], 0.1)
    orc.assert_close(got[:n], ref, spread)
    orc.assert_close(got[-n:], ref, spread)
    assert (got[n:2 * n] == 0).all() and capi.device_error(0) == 0


def test_rows_of_no_sequence_are_left_alone():
    q, k, v, _ = make([90], 4, 2, 128, 128, seed=5)
    cu = [10, 40, 80]
    out = torch.full((90, 4, 128), 3.0, dtype=q.dtype, device=DEV)
    run(q, k, v, cu, 0.1, out=out)
    ref, spread = orc.prompt_attention(q, k, v, cu, 0.1)
    orc.assert_close(out[10:80], ref[10:80], spread[10:80])
    assert (out[:10] == 3).all() and (out[80:] == 3).all()


def test_limits_are_enforced():
    """A boundary past the tokens or a sequence past max_seqlen is cut and reported."""
    q, k, v, _ = make([300], 4, 2, 128, 128, seed=6)
    for cu, longest, inside in (([0, 100, 400], 300, [0, 100, 300]), ([0, 300], 140, [0, 140])):
        out = torch.full((300, 4, 128), 3.0, dtype=q.dtype, device=DEV)
        run(q, k, v, cu, 0.1, longest=longest, out=out)
        assert capi.device_error(0, clear=True) == capi.FRN_DEVERR_BAD_LENGTH
        ref, spread = orc.prompt_attention(q, k, v, inside, 0.1)
        n = inside[-1]
        orc.assert_close(out[:n], ref[:n], spread[:n])
        assert (out[n:] == 3).all()
    assert capi.device_error(0) == 0


def test_nothing_to_do():
    q, k, v, _ = make([4], 4, 2, 128, 128)
    out = torch.full((4, 4, 128), 3.0, dtype=q.dtype, device=DEV)
    run(q, k, v, [0], 0.1, longest=4, out=out)
    run(q, k, v, [0, 0, 0], 0.1, longest=4, out=out)
    assert (out == 3).all()
    assert run(q[:0], k[:0], v[:0], [0, 0], 0.1, longest=0).shape == (0, 4, 128)


@pytest.mark.parametrize("heads", [(7, 1, 64, 64), (5, 1, 128, 128), (3, 1, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
def test_bits_do_not_depend_on_the_neighbourhood(heads):
    """A row's bits are the same whatever ran on the SM before and whatever lies
    beside it (rows of no token take part in the tiles): with large values, so
    that maxima move."""
    lens = [77, 130, 9]
    q, k, v, cu = make(lens, *heads, dtype=torch.float16, seed=21)
    q = q * 6
    alone = [run(q[a:b], k[a:b], v[a:b], [0, b - a], 0.3) for a, b in zip(cu[:-1], cu[1:])]
    for noise in (0.0, 100.0, -100.0):
        other = torch.full((400, *q.shape[1:]), noise, dtype=q.dtype)
        run(other, torch.ones(400, *k.shape[1:], dtype=k.dtype),
            torch.ones(400, *v.shape[1:], dtype=v.dtype), [0, 400], 0.3)
        got = run(q, k, v, cu, 0.3)
        for a, b, one in zip(cu[:-1], cu[1:], alone):
            assert torch.equal(got[a:b], one)


def test_streams_graphs_and_repeats():
    q, k, v, cu = make([200, 333], 8, 2, 128, 128, seed=8)
    first = run(q, k, v, cu, 0.09)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    cud = torch.tensor(cu, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = capi.gqa_prompt_attention(qd, kd, vd, cud, 333, 0.09)
    side.synchronize()
    assert torch.equal(first, again)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.gqa_prompt_attention(qd, kd, vd, cud, 333, 0.09, out=out)
    qd.copy_(qd.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    ref, spread = orc.prompt_attention(qd.cpu(), k, v, cu, 0.09)
    orc.assert_close(out, ref, spread)


def test_beside_other_work():
    """Bits and answers are the same while another stream keeps the SMs busy."""
    lens = [77, 300, 1, 160]
    q, k, v, cu = (t.to(DEV) if torch.is_tensor(t) else t for t in make(lens, 7, 1, 64, 64, seed=4))
    cud = torch.tensor(cu, dtype=torch.int32, device=DEV)
    busy = [t.to(DEV) for t in make([700] * 8, 16, 4, 128, 128, seed=5)[:3]]
    busy_cu = torch.arange(9, dtype=torch.int32, device=DEV) * 700
    first = capi.gqa_prompt_attention(q, k, v, cud, 300, 0.1)
    busy_first = capi.gqa_prompt_attention(*busy, busy_cu, 700, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got, busy_got = [], []
    for _ in range(20):
        with torch.cuda.stream(side):
            busy_got.append(capi.gqa_prompt_attention(*busy, busy_cu, 700, 0.1))
        got.append(capi.gqa_prompt_attention(q, k, v, cud, 300, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)
    assert all(torch.equal(x, busy_first) for x in busy_got)
    assert capi.device_error(0) == 0


def test_python_surface():
    from src.gqa_attention_forward import GQAPromptAttention
    from src.load_gqa_attention import gqa_attention_cuda as ops

    q, k, v, cu = make([60, 9], 4, 2, 128, 128, seed=1)
    ref, spread = orc.prompt_attention(q, k, v, cu, 0.1)
    cud = torch.tensor(cu, dtype=torch.int32, device=DEV)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    orc.assert_close(ops.gqa_prompt_attention(qd, kd, vd, cud, 60, 0.1), ref, spread)
    module = GQAPromptAttention(4, 2, 128, scale=0.1)
    orc.assert_close(module(qd, kd, vd, cud, 60), ref, spread)
    orc.assert_close(module(qd.flatten(1), kd.flatten(1), vd.flatten(1), cud, 60), ref, spread)
    # Layouts the kernel cannot read are copied first.
    odd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (qd, kd, vd)]
    orc.assert_close(ops.gqa_prompt_attention(*odd, cud, 60, 0.1), ref, spread)
    one = kd[:, :1].expand(-1, 2, -1)
    ref1, spread1 = orc.prompt_attention(q, one.cpu(), v, cu, 0.1)
    orc.assert_close(ops.gqa_prompt_attention(qd, one, vd, cud, 60, 0.1), ref1, spread1)
    shifted = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    shifted.copy_(qd)
    orc.assert_close(ops.gqa_prompt_attention(shifted, kd, vd, cud, 60, 0.1), ref, spread)
    for args, match in [((qd.float(), kd.float(), vd.float(), cud), "bf16 and fp16"),
                        ((qd, kd.half(), vd, cud), "one dtype"),
                        ((qd, kd[:5], vd, cud), "mismatch"),
                        ((qd[:, :3], kd, vd, cud), "multiple of num_kv_heads"),
                        ((qd, kd, vd[..., :64], cud), "head dims"),
                        ((qd, kd, vd, cud.long()), "int32"),
                        ((qd, kd, vd, cud.cpu()), "CUDA")]:
        with pytest.raises(RuntimeError, match=match):
            ops.gqa_prompt_attention(*args, 60, 0.1)
    assert capi.device_error(0) == 0
