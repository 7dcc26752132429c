"""NaN and infinities in the keys and values of packed prompts: rows that see one carry it on as
the definition does, rows that do not are as if it were not there, however long the prompt."""
import os
import subprocess
import sys

import pytest
import torch

from oracle import serving_attention as orc
from src import capi

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAN, INF = float("nan"), float("inf")
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def make(lens, Hq, Hkv, Dqk, Dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q, k = (torch.randn(T, h, Dqk, generator=g).to(dtype) for h in (Hq, Hkv))
    v = torch.randn(T, Hkv, Dv, generator=g).to(dtype)
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    return q, k, v, cu


def check(q, k, v, cu):
    scale = q.shape[2] ** -0.5
    longest = max(b - a for a, b in zip(cu[:-1], cu[1:]))
    got = capi.gqa_prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV),
                                    torch.tensor(cu, dtype=torch.int32, device=DEV), longest, scale)
    ref, spread = orc.prompt_attention(q, k, v, cu, scale)
    orc.assert_same(got, ref, spread)
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("dims", [(4, 2, 128, 128), (6, 2, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("values", [[(500, 5, NAN)], [(301, 5, INF), (310, 5, NAN)],
                                    [(301, 5, INF), (310, 5, -INF), (310, 9, -INF)],
                                    [(260, 60, -INF), (262, 61, NAN), (380, 60, INF)],
                                    [(0, 0, INF), (699, 0, NAN), (640, 1, NAN)],
                                    [(j, 7, INF) for j in range(250, 700, 3)]],
                         ids=["one", "two", "signs", "apart", "ends", "many"])
def test_values(dims, dtype, values):
    """(position, column, value) in V of a prompt of several items, between two others."""
    q, k, v, cu = make([130, 700, 40], *dims, dtype, seed=3)
    for at, column, value in values:
        v[cu[1] + at, :, column] = value
    check(q, k, v, cu)


@pytest.mark.parametrize("dims", [(4, 2, 128, 128), (6, 2, 64, 64), (2, 2, 192, 128)],
                         ids=lambda x: "x".join(map(str, x)))
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_keys_and_values(dims, value):
    """The same token's key and value, and a query's."""
    q, k, v, cu = make([260, 300], *dims, torch.bfloat16, seed=4)
    k[cu[1] + 150, :, 3] = value
    v[cu[1] + 150, :, 5] = value
    v[cu[1] + 160, :, 6] = value
    q[cu[1] + 155, :, 2] = value
    check(q, k, v, cu)


CHILD = r"""
import os, sys
sys.path[:0] = [os.environ["FRN_TEST_REPO"], os.environ["FRN_TEST_PROJECT"]]
import torch
from oracle import serving_attention as orc
from src import capi

T, Hq, D = 65536, 4, 64
g = torch.Generator().manual_seed(1)
q, k, v = (torch.randn(T, h, D, generator=g).bfloat16() for h in (Hq, 1, 1))
args = [t.cuda() for t in (q, k, v)]
cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
clean = capi.gqa_prompt_attention(*args, cu, T, 0.125)
args[2][T - 1, 0, 5] = float("nan")
got = capi.gqa_prompt_attention(*args, cu, T, 0.125)
torch.cuda.synchronize()
assert capi.device_error(0) == 0, "a wait ran out"
assert torch.equal(got[:T - 64], clean[:T - 64])
kd, vd = k[:, 0].double(), v[:, 0].double()
for i in (T - 33, T - 32, T - 20, T - 2):
    p = torch.softmax(q[i].double() @ kd[:i + 1].T * 0.125, 1)
    orc.assert_same(got[i], p @ vd[:i + 1], p @ vd[:i + 1].abs())
last = got[T - 1]
assert torch.isnan(last[:, 5]).all()
others = [c for c in range(D) if c != 5]
assert torch.equal(last[:, others], clean[T - 1][:, others])
print("child ok")
"""


def test_redone_rows_outlast_the_wait_limit():
    """A NaN at the end of 65536 tokens: the rows before it in its tile are computed again, which
    takes longer than the limit on waits (lowered for the child), and nothing is lost by it."""
    env = dict(os.environ, FRN_WAIT_TIMEOUT_MS="5", FRN_TEST_REPO=REPO,
               FRN_TEST_PROJECT=os.path.join(REPO, "kimi26-h100-rmsnorm-swiglu-fusion_b200"))
    out = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "child ok" in out.stdout, out.stderr[-2000:]
