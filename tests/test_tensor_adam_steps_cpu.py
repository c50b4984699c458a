"""ops.optim.TensorAdam: tensors that start late or are left out, and states of part of the tensors, as torch.optim has them."""
import ctypes

import pytest
import torch

from masters_thesis_amd.ops.optim import TensorAdam


def tensors(shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) for s in shapes]


SHAPES = [(300,), (7, 5), (260,)]


def run(state_bits, adamw, device="cpu", steps=12):
    """The optimizer and torch's on the same gradients, some left out: the largest difference of the parameters."""
    ps = [p.to(device) for p in tensors(SHAPES)]
    qs = [torch.nn.Parameter(p.clone()) for p in tensors(SHAPES)]
    opt = TensorAdam(ps, lr=0.1, betas=(0.9, 0.99), weight_decay=0.01, adamw=adamw, state_bits=state_bits)
    ref = (torch.optim.AdamW if adamw else torch.optim.Adam)(qs, lr=0.1, betas=(0.9, 0.99), weight_decay=0.01)
    opt.calls = 0
    for t in range(steps):
        gs = [g if (t + i) % (i + 2) == 0 or t > 8 else None for i, g in enumerate(tensors(SHAPES, seed=t + 1))]
        if t < 5:
            gs[2] = None  # starts late
        for q, g in zip(qs, gs):
            q.grad = g
        ref.step()
        opt.calls += any(g is not None for g in gs)
        opt.step(grads=[None if g is None else g.to(device) for g in gs])
    return opt, ref, max(float((p.cpu() - q.detach()).abs().max()) for p, q in zip(ps, qs))


@pytest.mark.parametrize("adamw", [True, False])
def test_each_tensor_has_its_own_steps(adamw):
    opt, ref, off = run(32, adamw)
    # 12 updates of at most about lr * 3.2 of some 20 fp32 operations each, on parameters up to 4
    assert off <= 12 * (32 * 0.1 * 2.0 ** -22 + 4 * 2.0 ** -23)
    mine, its = opt.state_dict()["state"], ref.state_dict()["state"]
    assert [float(mine[i]["step"]) for i in range(3)] == [float(its[i]["step"]) for i in range(3)] and float(opt.step_t) == opt.calls


def test_a_late_tensor_moves_as_a_first_step():
    ps = [torch.zeros(4), torch.zeros(4)]
    opt = TensorAdam(ps, lr=1.0, weight_decay=0.0)
    for _ in range(50):
        opt.step(grads=[torch.ones(4), None])
    opt.step(grads=[None, torch.ones(4)])
    assert torch.allclose(ps[1], torch.full((4,), -1.0), rtol=1e-6)


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_of_a_state_load_tensor_by_tensor(bits):
    a, _, _ = run(bits, True)
    b = TensorAdam([p.clone() for p in a.params], lr=0.3, state_bits=bits)
    b.load_state_dict(a.state_dict())
    assert torch.equal(a.steps, b.steps) and len(set(a.steps.tolist())) > 1
    for t in range(3):
        for o in (a, b):
            o.step(grads=tensors(SHAPES, seed=90 + t))
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    assert all(torch.equal(x, y) for x, y in zip(a._state, b._state))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_loaded_state_replaces_all_moments(bits):
    """Tensors without an entry start anew, as in torch.optim: an empty state, then one of a single tensor."""
    a, _, _ = run(bits, True)
    full = a.state_dict()
    for keep in ([], [1]):
        b, _, _ = run(bits, True)
        b.load_state_dict({"state": {i: full["state"][i] for i in keep}, "param_groups": full["param_groups"]})
        m, v = b.moments()
        for i, (o, p) in enumerate(zip(b.offsets, b.params)):
            if i in keep:
                assert torch.equal(m[o:o + p.numel()].view(p.shape), full["state"][i]["exp_avg"]) and b.steps[i] == full["state"][i]["step"]
            else:
                assert not m[o:o + p.numel()].any() and not v[o:o + p.numel()].any() and b.steps[i] == 0
        fresh = TensorAdam([p.clone() for p in b.params], lr=b.lr, betas=b.betas, weight_decay=b.weight_decay, state_bits=bits)
        gs = tensors(SHAPES, seed=70)
        b.step(grads=gs), fresh.step(grads=gs)
        assert all(torch.equal(x, y) for i, (x, y) in enumerate(zip(b.params, fresh.params)) if i not in keep)


def check_skipped(bits, max_norm, device):
    """A step with a gradient that is not finite changes nothing but the count of such steps (and zeroes the gradients)."""
    shapes = [(300,), (70, 90), (0,), (1,)]
    make = lambda seed: [x.to(device) for x in tensors(shapes, seed)]  # noqa: E731
    a, b = (TensorAdam(make(0), lr=1e-2, state_bits=bits, skip_nonfinite=s) for s in (True, False))
    for o in (a, b):
        o.step(max_norm, grads=make(1))
    state = lambda o: [x.clone() for x in (*o.params, *o._state, o.steps, o.step_t)]  # noqa: E731
    was, seen = state(a), 0
    assert all(torch.equal(x, y) for x, y in zip(was, state(b)))
    for zero in (False, True):
        for bad in (float("nan"), float("inf"), -float("inf")):
            for where in (0, 1, 3):
                gs = make(2)
                gs[where].view(-1)[-1] = bad
                a.step(max_norm, zero_grad=zero, grads=gs)
                seen += 1
                assert all(torch.equal(x, y) for x, y in zip(was, state(a))) and float(a.nonfinite) == seen
                assert not torch.isfinite(a.grad_norm).any()
                assert all(not g.any() for g in gs) if zero else gs[1].any()
    for o in (a, b):
        o.step(max_norm, grads=make(3))
    assert all(torch.equal(x, y) for x, y in zip(state(a), state(b))) and torch.isfinite(a.grad_norm).all()


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("bits", [8, 32])
def test_steps_that_are_not_finite_are_skipped(bits, max_norm):
    check_skipped(bits, max_norm, "cpu")


def test_the_trainer_keeps_its_weights_through_a_bad_gradient():
    """model.optimizer=adam_8bit: one NaN in a gradient loses neither weights nor moments, and is counted."""
    from masters_thesis_amd.engine import Trainer
    from masters_thesis_amd.models import get_model_class

    for clip in (None, 5.0):
        torch.manual_seed(0)
        model = get_model_class("FinancialLstmMse", "lstm")(input_size=3, hidden_size=32, num_layers=1, dropout=0.0, optimizer="adam_8bit")
        tr = Trainer(gradient_clip_val=clip, enable_progress_bar=False, enable_model_summary=False, accelerator="cpu")
        tr._setup_env()
        tr._setup_model(model)
        tr._configure_optimizers(model)
        assert isinstance(tr.optimizer, TensorAdam)
        tr.flat.grad.normal_()
        tr._optimizer_step()
        was = [x.clone() for x in (tr.flat.data, *tr.optimizer._state)]
        tr.flat.grad.normal_()
        tr.flat.params[0].grad.view(-1)[3] = float("nan")
        tr._optimizer_step()
        assert all(torch.equal(x, y) for x, y in zip(was, (tr.flat.data, *tr.optimizer._state)))
        assert float(tr.optimizer.nonfinite) == 1 and not any(p.grad.any() for p in tr.flat.params)
        tr.flat.grad.normal_()
        tr._optimizer_step()
        assert torch.isfinite(tr.flat.data).all() and not torch.equal(tr.flat.data, was[0])


class Table(ctypes.Structure):  # csrc/adam_tensors.h AdamTable
    _fields_ = [("p", ctypes.c_void_p * 112), ("g", ctypes.c_void_p * 112), ("n", ctypes.c_long * 112), ("block", ctypes.c_uint * 112),
                ("first", ctypes.c_uint * 112), ("type", ctypes.c_ubyte * 112), ("count", ctypes.c_int), ("place", ctypes.c_int),
                ("group", ctypes.c_int), ("groups", ctypes.c_uint)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="host checks: a launch would run")
@pytest.mark.parametrize("groups", [0, 2 ** 24, 2 ** 31])
def test_more_workgroups_than_a_launch_holds(groups):
    """Refused before anything is started; and a launch that fails (here: no device) is told."""
    from masters_thesis_amd.ops import build
    from masters_thesis_amd.ops._lib import lib

    if not build.ext_path().exists():
        build.build()
    lib()
    so = ctypes.CDLL(str(build.ext_path()))
    so.mta_adam_tensors.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    t, state = Table(count=1, group=4096, groups=groups), ctypes.create_string_buffer(512)
    assert so.mta_adam_tensors(ctypes.byref(t), 1, state, 1, None) == 2
    t.groups = 5
    assert so.mta_adam_tensors(ctypes.byref(t), 1, state, 1, None) == 4


def test_moments_in_8_bits_against_32_over_many_steps():
    """The same gradients for 600 steps: rounding by chance keeps the mean, and what noise it leaves has a bound.

    A step moves v by (1 - b2) |g^2 - v|, on average 0.97 (1 - b2) v for normal gradients; rounded up or down on a grid of
    steps s <= v / 16, the chance of the nearer end is that part of s, so the variance added is at most s 0.97 (1 - b2) v, and
    what stays of all steps' is 1 / (1 - b2^2) of it: 0.97 / 32 v^2, a deviation of 0.175 v.  m likewise with steps of |m| / 8,
    at most one step's s^2 / 4 a time: (m_max / 8)^2 / 4 / (1 - b1^2) of the block's largest m."""
    n, b1, b2 = 8192, 0.9, 0.99
    ps = [torch.zeros(n), torch.zeros(n)]
    opts = [TensorAdam([p], lr=1e-3, betas=(b1, b2), state_bits=bits, seed=11) for p, bits in zip(ps, (8, 32))]
    size = torch.linspace(0.5, 2.0, n)
    g = torch.Generator().manual_seed(0)
    for _ in range(600):
        x = torch.randn(n, generator=g) * size
        for o in opts:
            o.step(grads=[x])
    (m8, v8), (m, v) = opts[0].moments(), opts[1].moments()
    off = (v8 / v - 1).double()
    assert float(off.std()) <= 0.175 * 1.03 and abs(float(off.mean())) <= 5 * 0.175 / n ** 0.5
    top = m.view(-1, 256).abs().amax(1, keepdim=True).expand(-1, 256).reshape(-1)
    off = ((m8 - m) / top).double()
    noise = 1 / 8 / 2 / (1 - b1 ** 2) ** 0.5
    assert float(off.std()) <= noise and abs(float(off.mean())) <= 5 * noise / n ** 0.5


def test_an_eps_that_is_no_normal_number_is_refused():
    """Also from a state: an element without a gradient would become 0 / 0."""
    for eps in (1e-46, 2.0 ** -127, 0.0):
        with pytest.raises(ValueError, match="eps"):
            TensorAdam(tensors(SHAPES), eps=eps)
    opt = TensorAdam(tensors(SHAPES), eps=2.0 ** -126)
    opt.step(grads=[torch.zeros(s) for s in SHAPES])
    assert all(torch.isfinite(p).all() for p in opt.params)
    sd = opt.state_dict()
    for bad in (dict(eps=0.0), dict(betas=(0.9, 1.0)), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            opt.load_state_dict({**sd, "param_groups": [{**sd["param_groups"][0], **bad}]})
