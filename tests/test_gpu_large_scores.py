"""Finite inputs whose scores are far beyond 2^24, where a rounding of the score alone is worth
more than one: the weights are still those of the definition (equal keys share, a larger one takes
all), and the results finite."""
import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"
# Largest entries of q and k: their scores stay within fp32, and within reach of the products.
SIZES = {torch.float16: [1500.0, 8000.0, 60000.0], torch.bfloat16: [2.0 ** 13, 2.0 ** 20, 2.0 ** 50],
         torch.float32: [1e4, 1e6, 1e15]}
IDS = {torch.float16: "fp16", torch.bfloat16: "bf16", torch.float32: "fp32"}


def keys(n, Hkv, D, size, pattern, dtype):
    """Keys of +-size, or in steps that make one far larger than another; their scores against
    queries of +size are sums of equal terms, exact ties where the keys are equal."""
    if pattern == "equal":
        value = torch.full((n,), size)
    elif pattern == "negative":
        value = torch.full((n,), -size)
    elif pattern == "blocks":  # a larger value every 23 tokens, ties within
        value = size * (1 + (torch.arange(n) // 23).double()) / (1 + n // 23)
    else:  # one far larger key in the middle
        value = torch.full((n,), size / 2)
        value[n // 2] = size
    return value.to(dtype)[:, None, None].expand(n, Hkv, D).contiguous()


PATTERNS = ["equal", "negative", "blocks", "one"]


@pytest.mark.parametrize("dtype,size", [(d, s) for d in SIZES for s in SIZES[d]],
                         ids=lambda x: IDS.get(x, str(x)))
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("D", [64, 128])
def test_decode(dtype, size, pattern, D):
    decode(dtype, size, pattern, D)


def decode(dtype, size, pattern, D):
    lens = [700, 1, 33]
    k, v, table = orc.make_paged(lens, 16, 2, D, seed=1, dtype=dtype)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        k[table[b].long()[t // 16], t % 16] = keys(n, 2, D, size, pattern, dtype)
    q = torch.full((3, 8, D), size).to(dtype)
    got = capi.gqa_paged_decode_attention(
        *(t.to(DEV) for t in (q, k, v, table)),
        torch.tensor(lens, dtype=torch.int32, device=DEV), D ** -0.5)
    ref, spread = orc.paged_decode(q, k, v, table, torch.tensor(lens), D ** -0.5)
    assert torch.isfinite(got).all()
    orc.assert_same(got, ref, spread)
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("dtype,size", [(d, s) for d in SIZES if d != torch.float32
                                        for s in SIZES[d]], ids=lambda x: IDS.get(x, str(x)))
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("dims", [(4, 2, 128, 128), (7, 1, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
def test_prompt(dtype, size, pattern, dims):
    prompt(dtype, size, pattern, dims)


def prompt(dtype, size, pattern, dims):
    Hq, Hkv, Dqk, Dv = dims
    lens = [300, 1, 45]
    cu = [0, 300, 301, 346]
    q = torch.full((346, Hq, Dqk), size).to(dtype)
    k = torch.cat([keys(n, Hkv, Dqk, size, pattern, dtype) for n in lens])
    v = torch.randn(346, Hkv, Dv, generator=torch.Generator().manual_seed(2)).to(dtype)
    got = capi.gqa_prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV),
                                    torch.tensor(cu, dtype=torch.int32, device=DEV), 300,
                                    Dqk ** -0.5)
    ref, spread = orc.prompt_attention(q, k, v, cu, Dqk ** -0.5)
    assert torch.isfinite(got).all()
    orc.assert_same(got, ref, spread)
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("dims", [(4, 2, 128, 128), (7, 1, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
def test_prompt_of_very_low_scores(dims):
    """Every score far below -1e30."""
    prompt(torch.bfloat16, 2.0 ** 55, "negative", dims)
