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


def _dk_by_rows_that_see_it(q, k, do, want, causal):
    """dk's bound with float16's own step (2^-25 of dS times at least 2 / max |dO|) from the rows that see the key alone,
    instead of from all rows as attention_oracle counts it."""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    see = torch.ones(tq, tk, dtype=torch.bool, device=DEV)
    if causal:
        see &= torch.arange(tk, device=DEV)[None] <= torch.arange(tq, device=DEV)[:, None] + tk - tq
    top = do.double().abs().amax(3).view(b, tq, hk, h // hk).amax(3)  # (b, tq, hk)
    each = torch.where(see[None, :, :, None], top[:, :, None], 0.0).amax(1)  # (b, tk, hk)
    qsum = torch.einsum("tk,bthd->bkhd", see.double(), q.double().abs().view(b, tq, hk, h // hk, d).sum(3))
    per = 2.0 ** -26 * qsum / math.sqrt(d) * (1 + 2.0 ** -11)
    ref, bound = want["dk"]
    return ref, bound - per * (do.double().abs().amax() - each)[..., None]


@pytest.mark.parametrize("b,tq,tk,h,hk,d", [(1, 90, 90, 2, 2, 64), (1, 300, 300, 4, 1, 32), (1, 2200, 2300, 1, 1, 128), (70, 130, 130, 4, 4, 64),
                                            (2, 200, 90, 2, 1, 40)])
def test_float16_keys_are_as_exact_as_the_rows_that_see_them(b, tq, tk, h, hk, d):
    """One row of large output gradients, which sees only the first keys, and small ones over 2^20 of sizes."""
    q, k, v, do = make(b, tq, tk, h, hk, d, F16)
    size = 2.0 ** -torch.randint(2, 13, (b, tq, h, 1), generator=torch.Generator().manual_seed(2)).double()
    size[:, max(0, tq - tk)] = 2.0 ** 8
    do = (do.double() * size.to(DEV)).to(F16)
    want = oracle(q, k, v, do, True)
    want["dk"] = _dk_by_rows_that_see_it(q, k, do, want, True)
    check(run(q, k, v, do, causal=True), want)


@pytest.mark.parametrize("tq,tk,h,hk", [(1, 5000, 4, 1), (1, 1029, 2, 2), (16, 3000, 2, 1), (200, 2100, 1, 1)])
def test_float16_split_keys(tq, tk, h, hk):
    q, k, v, _ = make(2, tq, tk, h, hk, 64, F16)
    lengths = [tk, tk // 9]
    out, lse = _A().attention_forward(q, k, v, key_lengths=torch.tensor(lengths, device=DEV))
    check({"out": out, "lse": lse}, oracle(q, k, v, None, False, lengths))


@pytest.mark.parametrize("b,tq,tk,h,hk,causal", [(1, 700, 700, 2, 1, True), (2, 40, 3000, 1, 1, False), (1, 1500, 130, 4, 2, True),
                                                 (1, 1, 2000, 2, 1, False), (1, 2200, 2300, 1, 1, True), (3, 1, 5000, 2, 1, False)])
def test_float16_split_sums_of_the_backward(b, tq, tk, h, hk, causal):
    """The sums of ranges carry each range's power of two; rows of sizes that differ by 2^20."""
    q, k, v, do = make(b, tq, tk, h, hk, 72, F16)
    lengths = [tk - 5] * b
    size = 2.0 ** -torch.randint(0, 21, (b, tq, h, 1), generator=torch.Generator().manual_seed(3)).double()
    do = (do.double() * size.to(DEV) * 2 ** 6).to(F16)
    check(run(q, k, v, do, causal=causal, key_lengths=torch.tensor(lengths, device=DEV)), oracle(q, k, v, do, causal, lengths))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq,tk,h,hk,causal", [(65, 65, 16, 1, True), (1, 90, 33, 3, False), (7, 300, 64, 2, True), (40, 130, 12, 1, False)])
def test_large_groups(tq, tk, h, hk, causal, dtype):
    """More query heads to a key head than rows of a tile are tokens."""
    q, k, v, do = make(2, tq, tk, h, hk, 32, dtype)
    lengths = [tk, tk - tk // 3]
    check(run(q, k, v, do, causal=causal, key_lengths=torch.tensor(lengths, device=DEV)), oracle(q, k, v, do, causal, lengths))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,tq,tk,h,hk", [(1, 1, 200, 2, 1), (2, 70, 70, 4, 2), (70, 150, 150, 4, 4)])
@pytest.mark.parametrize("d", [8, 24, 32, 40, 56, 64, 72, 120, 128])
def test_infinite_keys_weigh_nothing_at_every_dim(d, b, tq, tk, h, hk, dtype):
    """An infinite element that takes a key's score to -inf gives it the weight 0, whatever the dim; its value may be
    anything finite."""
    q, k, v, _ = make(b, tq, tk, h, hk, d, dtype)
    q[..., 0] = q[..., 0].abs() + 0.5
    shut = torch.arange(tk, device=DEV) % 5 == 2
    k[:, shut, :, 0] = -math.inf
    out, lse = _A().attention_forward(q, k, v)
    want = oracle(q, k[:, ~shut], v[:, ~shut])
    # the keys in between are in other tiles than they would be without the others: the same sums in another order
    check({"out": out, "lse": lse}, want)


@pytest.mark.parametrize("b,tq,tk,h,hk,causal,few", [(16, 200, 200, 1, 1, False, True), (8, 400, 400, 1, 1, True, True), (8, 400, 400, 1, 1, False, False),
                                                     (2, 1000, 1000, 2, 2, True, False), (40, 300, 300, 1, 1, True, False)])
def test_float16_kernels_of_few_problems_past_dim_64(b, tq, tk, h, hk, causal, few):
    """Both kernels of a backward with few problems, on either side of the rule that chooses them."""
    q, k, v, do = make(b, tq, tk, h, hk, 96, F16)
    want = oracle(q, k, v, do, causal)
    check(run(q, k, v, do, causal=causal), want)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        run(q, k, v, do, causal=causal)
        torch.cuda.synchronize()
    names = [e.key for e in prof.key_averages()]
    assert any("mha_dkv_few_kernel" in n for n in names) == few == any("mha_dq_few_kernel" in n for n in names)
    assert any("mha_dkv_kernel" in n for n in names) != few


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales(dtype):
    """The smallest scale (every key weighs the same, hidden ones nothing) and the refusal of those that float32 does not hold."""
    q, k, v, do = make(2, 70, 90, 4, 2, 40, dtype)
    n = torch.tensor([90, 41], device=DEV)
    for scale in (1e-60, 2.0 ** -121, 2.0 ** 121, 1e39, math.nan):
        with pytest.raises(ValueError, match="scale"):
            _A().attention(q, k, v, scale=scale)
    for causal in (False, True):
        check(run(q, k, v, do, causal=causal, key_lengths=n, scale=2.0 ** -120), oracle(q, k, v, do, causal, [90, 41], 2.0 ** -120))
