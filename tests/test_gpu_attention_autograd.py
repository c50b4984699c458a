"""What ops.attention is asked for by autograd beyond first derivatives: raised where it is not there, never left out."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _A():
    from masters_thesis_amd.ops import attention as A

    return A


def leaves(b=2, t=9, h=4, hk=2, d=16, dtype=torch.float32, grad=True):
    g = torch.Generator(device=DEV).manual_seed(0)
    return [torch.randn(b, t, n, d, generator=g, device=DEV).to(dtype).requires_grad_(grad) for n in (h, hk, hk)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_derivatives_raise(which):
    """Also where another differentiable term stands beside the gradients, and in a penalty on them."""
    x = leaves()
    out = _A().attention(*x, causal=True)
    (g,) = torch.autograd.grad(out.square().sum(), x[which], create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):  # asked for by name: the way to them leads through the gradient
        torch.autograd.grad(g.square().sum() + out.sum(), x[which], retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        (g.square().sum() + out.sum()).backward()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(_penalty(x), x)
    # and first derivatives taken with create_graph are those without it
    (plain,) = torch.autograd.grad(_A().attention(*x, causal=True).square().sum(), x[which])
    assert torch.equal(g.detach(), plain)


def _penalty(x):
    out = _A().attention(*x)
    grads = torch.autograd.grad(out.sum(), x, create_graph=True)
    return out.sum() + sum(g.square().sum() for g in grads)


def test_forward_mode_raises():
    """A tangent is not left behind: every entry point refuses dual tensors, whichever argument carries it."""
    import torch.autograd.forward_ad as fw

    A = _A()
    x = leaves(grad=False)
    out, lse = A.attention_forward(*x)
    with fw.dual_level():
        for i in range(3):
            y = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(x)]
            for fn in (A.attention, A.attention_forward):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*y)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.attention_backward(fw.make_dual(out, out), *x, out, lse)
        z = leaves()
        recorded = A.attention(*z)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(recorded, z, fw.make_dual(out, out))


def test_batched_transforms_raise():
    """torch.func's wrappers, whose tensors have no memory of their own, are refused, not read."""
    A = _A()
    x = leaves(grad=False)
    with pytest.raises(RuntimeError):
        torch.func.vmap(A.attention)(*(t[None] for t in x))
    with pytest.raises(RuntimeError):
        torch.func.jvp(A.attention, tuple(x), tuple(x))
    y = leaves()
    out = A.attention(*y)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, y, torch.stack([out.detach()] * 2), is_grads_batched=True)


def test_rope_is_refused_within_a_graph():
    """It records nothing: the gradients of what it turned would be those of what it did not."""
    import torch.autograd.forward_ad as fw

    A = _A()
    w = torch.randn(6, 24, device=DEV, requires_grad=True)
    x = torch.randn(10, 6, device=DEV)
    for t in (w, x @ w, (x @ w)[:, :16]):
        with pytest.raises(RuntimeError, match="gradient"):
            A.rope_(t, 5, 2, 4)
    with fw.dual_level(), pytest.raises(RuntimeError, match="gradient"):
        A.rope_(fw.make_dual(w.detach(), w.detach()), 5, 2, 4)
    with torch.no_grad():  # as any operation in place
        A.rope_(w, 3, 2, 4)
    with torch.inference_mode():
        A.rope_(torch.randn(6, 24, device=DEV), 3, 2, 4)


def test_rope_of_sequences_past_31_bits():
    """Lengths are 32-bit numbers in the kernel: longer ones are refused, not cut (2^32 would become 0)."""
    A = _A()
    x = torch.randn(6, 24, device=DEV)
    for seq in (2 ** 32, 2 ** 32 + 3, 2 ** 31, 0, -1):
        with pytest.raises(RuntimeError, match="bad sizes"):
            A.rope_(x, seq, 2, 4)
    y = x.clone()
    A.rope_(x, 2 ** 31 - 1, 2, 4)
    A.rope_(y, 6, 2, 4)
    assert torch.equal(x, y)


def test_rope_is_seen_by_a_backward_that_saved_its_tensor():
    A = _A()
    x = torch.randn(10, 24, device=DEV)
    w = torch.randn(24, device=DEV, requires_grad=True)
    y = (x * w).sum()
    A.rope_(x, 5, 2, 4)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradients_that_overlap_are_refused():
    """Views of one buffer a head apart (two kernels would write the same places) are refused, beside each other they are not."""
    A = _A()
    q, k, v = leaves(2, 8, 2, 2, 32, grad=False)
    do = torch.randn_like(q)
    out, lse = A.attention_forward(q, k, v)
    packed = torch.zeros(2, 8, 6, 32, device=DEV)
    for bad in ((packed[:, :, :2], packed[:, :, 1:3], packed[:, :, 4:]), (packed[:, :, :2], packed[:, :, 2:4], packed[:, :, 3:5]),
                (packed[:, :, 3:5], packed[:, :, :2], packed[:, :, 4:])):
        with pytest.raises(ValueError, match="memory"):
            A.attention_backward(do, q, k, v, out, lse, grads=bad)
    turned = torch.zeros(6, 2, 8, 32, device=DEV).permute(1, 2, 0, 3)  # heads first
    for p in (packed, turned):
        A.attention_backward(do, q, k, v, out, lse, grads=(p[:, :, :2], p[:, :, 2:4], p[:, :, 4:]))
        assert all(torch.equal(a, b) for a, b in zip(p.split(2, 2), A.attention_backward(do, q, k, v, out, lse)))


def test_gradients_written_in_place_are_seen_by_a_backward_that_saved_them():
    A = _A()
    q, k, v = leaves(2, 8, 2, 2, 32, grad=False)
    out, lse = A.attention_forward(q, k, v)
    grads = tuple(torch.zeros_like(x) for x in (q, k, v))
    w = torch.ones(3, device=DEV, requires_grad=True)
    y = [(g * w[i]).sum() for i, g in enumerate(grads)]
    A.attention_backward(out, q, k, v, out, lse, grads=grads)
    for x in y:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            x.backward()
