"""What ops.attention is asked for by autograd beyond first derivatives, on the CPU."""
import pytest
import torch

from masters_thesis_amd.ops.attention import attention


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
