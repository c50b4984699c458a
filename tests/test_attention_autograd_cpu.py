"""What ops.attention is asked for by autograd beyond first derivatives, on the CPU."""
import math

import pytest
import torch

from masters_thesis_amd.ops.attention import attention, attention_backward, attention_forward


def leaves(b=2, t=9, h=4, hk=2, d=16):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(b, t, n, d, generator=g).requires_grad_() for n in (h, hk, hk)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_derivatives_raise(which):
    """Also where another differentiable term stands beside the gradients, and where only inputs are asked for."""
    x = leaves()
    out = attention(*x, causal=True)
    (g,) = torch.autograd.grad(out.square().sum(), x[which], create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(g.square().sum() + out.sum(), x[which], retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        (g.square().sum() + out.sum()).backward()
    (plain,) = torch.autograd.grad(attention(*x, causal=True).square().sum(), x[which])
    assert torch.equal(g.detach(), plain)


def test_gradients_into_shared_memory_are_refused():
    q, k, v = (x.detach() for x in leaves(2, 8, 2, 2, 32))
    do = torch.randn_like(q)
    out, lse = attention_forward(q, k, v)
    new = lambda: [torch.zeros_like(x) for x in (q, k, v)]  # noqa: E731
    packed = torch.zeros(2, 8, 6, 32)
    for bad in ((packed[:, :, :2], packed[:, :, 1:3], packed[:, :, 4:]), (packed[:, :, :2], packed[:, :, 2:4], packed[:, :, 3:5])):
        with pytest.raises(ValueError, match="memory"):
            attention_backward(do, q, k, v, out, lse, grads=bad)
    for i, bad in ((0, q), (1, do), (2, out), (1, torch.zeros_like(k).as_strided(k.shape, (16 * 32, 32, 32, 1)))):
        grads = new()
        grads[i] = bad
        with pytest.raises(ValueError, match="memory"):
            attention_backward(do, q, k, v, out, lse, grads=tuple(grads))
    for i, bad in ((0, q[:1].clone()), (1, k.double()), (2, torch.zeros(2, 8, 2, 33)[..., :32])):
        grads = new()
        grads[i] = bad
        with pytest.raises(ValueError):
            attention_backward(do, q, k, v, out, lse, grads=tuple(grads))
    attention_backward(do, q, k, v, out, lse, grads=(packed[:, :, :2], packed[:, :, 2:4], packed[:, :, 4:]))
    assert all(torch.equal(a, b) for a, b in zip(packed.split(2, 2), attention_backward(do, q, k, v, out, lse)))


def test_what_blind_rows_hold_reaches_nothing():
    """Causal, more queries than keys: the first ones see no key, and their q and dout may be anything."""
    g = torch.Generator().manual_seed(1)
    q, do = (torch.randn(2, 9, 4, 16, generator=g) for _ in range(2))
    k, v = (torch.randn(2, 4, 2, 16, generator=g) for _ in range(2))
    q[:, :5], do[:, :5] = 0, 0

    def run():
        out, lse = attention_forward(q, k, v, causal=True)
        return out, *attention_backward(do, q, k, v, out, lse, causal=True)

    want = run()
    for bad in (math.nan, math.inf):
        q[:, :5:2], do[:, 1:5], do[:, 0] = bad, bad, bad
        assert all(torch.equal(a, b) for a, b in zip(run(), want))


def test_scales_that_float32_does_not_hold_are_refused():
    q, k, v = (x.detach() for x in leaves())
    for scale in (1e-60, 2.0 ** -121, 2.0 ** 121, 1e39, math.nan):
        with pytest.raises(ValueError, match="scale"):
            attention(q, k, v, scale=scale)
    even = attention(q, k, v, scale=2.0 ** -120)  # every key weighs the same
    assert torch.allclose(even, v.mean(1, keepdim=True).repeat_interleave(2, 2).expand_as(even), atol=1e-6)
