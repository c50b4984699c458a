"""ops.attention on the GPU: rows and keys whose numbers must not reach others (blind rows, padding, hidden keys), and the
exactness of each key's gradients whatever the other rows hold."""
import math

import pytest
import torch

from attention_oracle import check, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _A():
    from masters_thesis_amd.ops import attention as A

    return A


def make(b, tq, tk, h, hk, d, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(b, t, n, d, generator=g, device=DEV).to(dtype) for t, n in ((tq, h), (tk, hk), (tk, hk), (tq, h))]


def run(q, k, v, do, **kw):
    A = _A()
    out, lse = A.attention_forward(q, k, v, **kw)
    dq, dk, dv = A.attention_backward(do, q, k, v, out, lse, **kw)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,tq,tk,h,hk,d", [(2, 9, 4, 2, 2, 32), (1, 150, 40, 4, 2, 64), (1, 257, 63, 2, 2, 40), (70, 150, 40, 4, 4, 32),
                                            (1, 2400, 2300, 1, 1, 128)])
def test_what_blind_rows_hold_reaches_nothing(b, tq, tk, h, hk, d, dtype):
    """Causal, more queries than keys: the first Tq - Tk see no key.  Their q and dout may be anything."""
    q, k, v, do = make(b, tq, tk, h, hk, d, dtype)
    none = tq - tk
    q[:, :none], do[:, :none] = 0, 0
    want = run(q, k, v, do, causal=True)
    check({n: want[n] for n in want}, oracle(q, k, v, do, True))
    for bad in (math.nan, math.inf, -math.inf, float(torch.finfo(dtype).max)):
        q[:, :none:2], do[:, 1:none:3] = bad, bad
        do[:, 0] = bad
        got = run(q, k, v, do, causal=True)
        for name in want:
            assert torch.equal(got[name], want[name]), (name, bad)
        assert not got["dq"][:, :none].any() and not got["out"][:, :none].any()
