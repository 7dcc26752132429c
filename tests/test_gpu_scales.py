"""Scales that are not finite give what the definition gives: NaN in every row of a token."""
import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"
SCALES = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dims", [(4, 2, 128, 128), (7, 1, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
def test_prompt(scale, dims):
    Hq, Hkv, Dqk, Dv = dims
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(140, h, d, generator=g).bfloat16()
               for h, d in ((Hq, Dqk), (Hkv, Dqk), (Hkv, Dv)))
    cu = [0, 3, 130]  # ten rows of no sequence
    out = torch.full((140, Hq, Dv), 3.0, dtype=q.dtype, device=DEV)
    capi.gqa_prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV),
                              torch.tensor(cu, dtype=torch.int32, device=DEV), 127, scale, out=out)
    ref, _ = orc.prompt_attention(q, k, v, cu, scale)
    assert torch.isnan(ref[:130]).all()
    assert torch.isnan(out[:130]).all() and (out[130:] == 3).all()
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32],
                         ids=["bf16", "fp16", "fp32"])
def test_decode(scale, dtype):
    lens = [70, 0, 3000]
    k, v, table = orc.make_paged(lens, 16, 2, 128, seed=2, dtype=dtype)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(3)).to(dtype)
    got = capi.gqa_paged_decode_attention(
        *(t.to(DEV) for t in (q, k, v, table)),
        torch.tensor(lens, dtype=torch.int32, device=DEV), scale)
    assert torch.isnan(got[[0, 2]]).all() and (got[1] == 0).all()
    assert capi.device_error(0) == 0
