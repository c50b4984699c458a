"""ops.optim.TensorAdam on the GPU: tensors that start late or are left out of steps."""
import pytest
import torch

from test_tensor_adam_steps_cpu import SHAPES, check_skipped, run, tensors

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("adamw", [True, False])
def test_each_tensor_has_its_own_steps(adamw):
    opt, ref, off = run(32, adamw, DEV)
    assert off <= 12 * (32 * 0.1 * 2.0 ** -22 + 4 * 2.0 ** -23)  # as on the CPU
    mine, its = opt.state_dict()["state"], ref.state_dict()["state"]
    assert [float(mine[i]["step"]) for i in range(3)] == [float(its[i]["step"]) for i in range(3)] and float(opt.step_t) == opt.calls


def test_codes_of_left_out_tensors_are_the_cpus():
    a, _, _ = run(8, True, DEV)
    b, _, _ = run(8, True)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(a._state, b._state)) and torch.equal(a.steps.cpu(), b.steps)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_a_launch_takes(bits):
    """Counts and factors of every tensor, in whichever launch it is, with and without clipping; empty tensors between."""
    from masters_thesis_amd.ops.optim import TensorAdam

    n = 300
    shapes = [(0,) if i % 50 == 7 else (1 + 37 * i % 700,) for i in range(n)]
    ps, qs = [p.to(DEV) for p in tensors(shapes)], tensors(shapes)
    a, b = TensorAdam(ps, lr=1e-2, state_bits=bits), TensorAdam(qs, lr=1e-2, state_bits=bits)
    for t in range(4):
        gs = [g if (i + t) % 3 or t == 3 else None for i, g in enumerate(tensors(shapes, seed=t + 1))]
        norm = 1.0 if t % 2 else 0.0
        a.step(max_norm=norm, grads=[None if g is None else g.to(DEV) for g in gs])
        b.step(max_norm=norm, grads=gs)
        assert torch.equal(a.steps.cpu(), b.steps)
    for p, q in zip(ps, qs):
        assert torch.allclose(p.cpu(), q, rtol=1e-5, atol=1e-6)


def test_captured_steps_count_for_the_tensors_they_take():
    from masters_thesis_amd.ops.optim import TensorAdam

    ps, qs = [p.to(DEV) for p in tensors(SHAPES)], [p.to(DEV) for p in tensors(SHAPES)]
    gs = [g.to(DEV) for g in tensors(SHAPES, seed=1)]
    a, b = (TensorAdam(x, lr=1e-2, state_bits=8) for x in (ps, qs))
    for o in (a, b):
        o.step(1.0, grads=gs)
    part = [gs[0], None, gs[2]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(1.0, grads=part)
    for t in range(3):
        graph.replay()
        b.step(1.0, grads=part)
        if t == 1:
            for o in (a, b):
                o.step(grads=gs)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ps + a._state, qs + b._state)) and torch.equal(a.steps, b.steps)
    assert a.steps.tolist() == [5.0, 2.0, 5.0]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_loaded_state_replaces_all_moments(bits):
    a, _, _ = run(bits, True, DEV)
    full = a.state_dict()
    a.load_state_dict({"state": {1: full["state"][1]}, "param_groups": full["param_groups"]})
    m, v = a.moments()
    o, n = a.offsets[1], a.params[1].numel()
    assert torch.equal(m[o:o + n].cpu(), full["state"][1]["exp_avg"].view(-1)) and m[o:o + n].any()
    m[o:o + n] = v[o:o + n] = 0
    assert not m.any() and not v.any() and a.steps.tolist() == [0.0, float(full["state"][1]["step"]), 0.0]


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("bits", [8, 32])
def test_steps_that_are_not_finite_are_skipped(bits, max_norm):
    check_skipped(bits, max_norm, DEV)


def test_a_captured_step_skips_too():
    from masters_thesis_amd.ops.optim import TensorAdam

    ps, gs = [p.to(DEV) for p in tensors(SHAPES)], [g.to(DEV) for g in tensors(SHAPES, seed=1)]
    opt = TensorAdam(ps, lr=1e-2, state_bits=8, skip_nonfinite=True)
    opt.step(1.0, grads=gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(1.0, zero_grad=True, grads=gs)
    for t in range(4):
        for g, x in zip(gs, tensors(SHAPES, seed=t)):
            g.copy_(x)
        if t % 2:
            gs[1][3, 2] = float("nan")
        was = [x.clone() for x in ps + opt._state]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(was, ps + opt._state)) == bool(t % 2) and not any(g.any() for g in gs)
    assert opt.steps.tolist() == [3.0] * 3 and float(opt.nonfinite) == 2


def test_a_backward_that_saved_what_a_step_changed_sees_it():
    """Parameters, and gradients that are zeroed; not those that are left as they were."""
    from masters_thesis_amd.ops.optim import TensorAdam

    ps = [torch.nn.Parameter(p.to(DEV)) for p in tensors(SHAPES)]
    gs = [g.to(DEV) for g in tensors(SHAPES, seed=1)]
    opt = TensorAdam(ps, lr=1e-2)
    x = torch.ones(2, device=DEV, requires_grad=True)
    late = [(x[0] * p).square().sum() for p in ps] + [(x[1] * g).sum() for g in gs]
    opt.step(grads=[None, *gs[1:]])
    late[0].backward(), late[4].backward()
    for y in late[1:3]:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    opt.step(grads=[None, *gs[1:]], zero_grad=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late[5].backward()
    late[3].backward()


@pytest.mark.parametrize("bits", [8, 32])
def test_the_smallest_eps(bits):
    """Elements without a gradient stay where they are."""
    from masters_thesis_amd.ops.optim import TensorAdam

    ps = [p.to(DEV) for p in tensors(SHAPES)]
    was = [p.clone() for p in ps]
    opt = TensorAdam(ps, lr=1e-2, eps=2.0 ** -126, state_bits=bits, weight_decay=0.0)
    for _ in range(2):
        opt.step(grads=[torch.zeros_like(p) for p in ps])
    assert all(torch.equal(p, w) for p, w in zip(ps, was))
