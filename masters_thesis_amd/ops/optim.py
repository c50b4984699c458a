"""Flat-buffer parameters and the fused clip + Adam/AdamW optimizer.

Reference: ``torch.optim.Adam(params, lr, weight_decay)`` (coupled L2,
`src/model.py:150-154`) preceded by Lightning's ``gradient_clip_val`` norm clipping
(`train.py:171`, `configs/trainer/*.yaml:2`).

MI355X design:

* ``FlatParameters`` moves every parameter (and its gradient) into ONE contiguous
  fp32 buffer, padded to a multiple of 1024 floats.  Each ``param.data`` /
  ``param.grad`` becomes a view, so autograd accumulates straight into the flat
  gradient buffer — which is then the single DDP all-reduce bucket (one RCCL call
  per step for the <= 1 MB gradients of this workload) and the single input of
  the fused optimizer.
* ``FusedAdam.step`` is ONE HIP launch (``csrc/optim.hip:adam_fused_kernel``): per-workgroup
  partial grad norms, an in-launch arrival ticket (write-through partials, no fences), then
  clip + Adam with ``lr`` and the step counter in device memory, i.e. it can be captured once
  in a HIP graph and replayed forever; the plateau scheduler only writes the lr scalar.  With
  ``zero_grad=True`` the kernel leaves the gradient zeroed, which replaces the per-step fill
  (``grads_zeroed`` tells the trainer).  ``single_launch=False`` selects the older
  norm + update pair (slower: profiles/r5_adam_two_launch_ab.jsonl; kept as the test oracle).
"""
from __future__ import annotations

import math
import os
from typing import Dict, Iterable, List, Optional, Sequence

import torch
from torch import Tensor

from ._lib import lib, use_hip

_ALIGN = 1024

# The optimizer whose flat gradient the ops may produce into by OVERWRITING (see FusedAdam.register_producer), or None.
_PRODUCER_OPT: List[Optional["FusedAdam"]] = [None]


def set_producer_optimizer(opt: Optional["FusedAdam"]) -> None:
    """Enable (single-process training) or disable gradient producers for ``opt`` (the trainer calls this)."""
    _PRODUCER_OPT[0] = opt


def register_grad_producer(grad: Tensor) -> Optional[Tensor]:
    """For a weight-gradient op about to write ``grad`` (a view into the active optimizer's flat gradient): the norm
    partials buffer it must fill, with overwrite semantics (``lib().gemm_grad_producer(parts, True)``), or None
    (accumulate as usual)."""
    opt = _PRODUCER_OPT[0]
    return None if opt is None else opt.register_producer(grad)


class FlatParameters:
    def __init__(self, params: Iterable[torch.nn.Parameter], device: Optional[torch.device] = None):
        self.params: List[torch.nn.Parameter] = [p for p in params if p.requires_grad]
        if not self.params:
            raise ValueError("no trainable parameters")
        dev = device or self.params[0].device
        self.offsets: List[int] = []
        off = 0
        for p in self.params:
            self.offsets.append(off)
            # every parameter starts on a 16-byte boundary: its range is whole float4s (the vectorised kernels and
            # the gradient producers' covered ranges); the gaps stay zero in every buffer
            off += -(-p.numel() // 4) * 4
        self.numel = off
        self.padded = -(-off // _ALIGN) * _ALIGN
        self.data = torch.zeros(self.padded, device=dev, dtype=torch.float32)
        self.grad = torch.zeros(self.padded, device=dev, dtype=torch.float32)
        for p, o in zip(self.params, self.offsets):
            n = p.numel()
            self.data[o:o + n].copy_(p.detach().reshape(-1).to(dev, torch.float32))
            p.data = self.data[o:o + n].view_as(p)
            p.grad = self.grad[o:o + n].view_as(p)

    def zero_grad(self) -> None:
        self.grad.zero_()

    def ensure_grad_views(self) -> None:
        """Re-attach grad views if something replaced ``p.grad`` (e.g. set_to_none)."""
        for p, o in zip(self.params, self.offsets):
            n = p.numel()
            if p.grad is None or p.grad.data_ptr() != self.grad[o:o + n].data_ptr():
                if p.grad is not None:
                    self.grad[o:o + n].copy_(p.grad.reshape(-1))
                p.grad = self.grad[o:o + n].view_as(p)

    def views(self, buf: Tensor) -> List[Tensor]:
        return [buf[o:o + p.numel()].view_as(p) for p, o in zip(self.params, self.offsets)]


class FusedAdam:
    """Adam (coupled L2, torch.optim.Adam semantics) or AdamW over a FlatParameters buffer."""

    def __init__(self, flat: FlatParameters, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, adamw: bool = False, single_launch: bool = True):
        self.flat = flat
        dev = flat.data.device
        self.exp_avg = torch.zeros_like(flat.data)
        self.exp_avg_sq = torch.zeros_like(flat.data)
        self.lr_t = torch.tensor([lr], device=dev, dtype=torch.float32)
        self.step_t = torch.zeros(1, device=dev, dtype=torch.float32)
        self.grad_norm = torch.zeros(1, device=dev, dtype=torch.float32)
        # [0] steps with a NaN/Inf grad norm, [1] in-launch arrival waits that gave up (fused kernel)
        self._health = torch.zeros(2, device=dev, dtype=torch.float32)
        self.nonfinite = self._health[0:1]
        self.sync_timeouts = self._health[1:2]
        self.grads_zeroed = False  # True after a step that left the flat gradient zeroed
        self.betas = tuple(float(b) for b in betas)
        self.eps = float(eps)
        self.weight_decay = float(weight_decay)
        self.adamw = bool(adamw)
        self._lr = float(lr)
        self.hip = use_hip(flat.data)
        # gradient producers (register_producer): float4 ranges of the flat gradient a weight-gradient GEMM overwrote
        # this step, and their clip-norm partials; consumed by the next step()
        self._plan: Dict[tuple, tuple] = {}
        self._dropped: set = set()  # ranges produced twice this step: accumulated, not covered
        if self.hip:
            C = lib()
            self.single_launch = bool(single_launch)
            n = C.adam_fused_partials() if self.single_launch else C.optim_num_partials(flat.padded)
            self.partials = torch.zeros(n, device=dev, dtype=torch.float32)
            self.ticket = torch.zeros(1, device=dev, dtype=torch.int64)
            self._nparts = int(C.gemm_norm_parts())
            self.ext_parts = torch.zeros(self.MAX_PRODUCERS * self._nparts, device=dev, dtype=torch.float32)
        # torch.optim-like surface for schedulers / LR monitors / checkpoints
        self.param_groups = [{
            "lr": lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay, "amsgrad": False,
            "maximize": False, "foreach": None, "capturable": True, "differentiable": False, "fused": True,
            "decoupled_weight_decay": self.adamw, "params": list(range(len(flat.params))),
        }]

    MAX_PRODUCERS = 8  # csrc/optim.hip MAX_COVERED

    def register_producer(self, grad: Tensor) -> Optional[Tensor]:
        """A producer that overwrites ``grad`` (contiguous view into the flat gradient, float4-aligned) and writes the
        clip-norm partials of it into the returned buffer; this step's fused update then neither re-reads it for the
        norm nor zeroes it.  None when not applicable (accumulate as usual).  Decided from static properties only
        (alignment, slots), so a producer makes the same choice every step: a range the update left unzeroed is
        always overwritten by the next backward."""
        if not (self.hip and self.single_launch) or os.environ.get("MTA_OPTIM_PRODUCERS", "1") == "0":
            return None
        f = self.flat
        if not grad.is_contiguous() or grad.dtype != torch.float32:
            return None
        off = (grad.data_ptr() - f.grad.data_ptr()) // 4
        n = grad.numel()
        if off < 0 or off + n > f.padded or off % 4 or n % 4:
            return None
        key = (off // 4, (off + n) // 4)
        clash = [k for k in self._plan if k[0] < key[1] and key[0] < k[1]]
        if clash:
            # a second producer of the same range before step() (a weight used twice, two backward calls): the
            # first one overwrote the range, this one must ADD to it, and the range's norm partials would be stale
            # -- drop the range from this step's covered plan (the update re-reads it for the norm and zeroes it)
            # and let this GEMM accumulate
            for k in clash:
                del self._plan[k]
                self._dropped.add(k)
            self._dropped.add(key)
            return None
        if any(k[0] < key[1] and key[0] < k[1] for k in self._dropped):
            return None
        used = {s for _, _, s in self._plan.values()}
        free = [s for s in range(self.MAX_PRODUCERS) if s not in used]
        if not free:
            return None
        self._plan[key] = (key[0], key[1], free[0])
        slot = free[0]
        return self.ext_parts[slot * self._nparts:(slot + 1) * self._nparts]

    # ---- lr (device-resident) --------------------------------------------------
    @property
    def lr(self) -> float:
        return self._lr

    def set_lr(self, lr: float) -> None:
        self._lr = float(lr)
        self.param_groups[0]["lr"] = float(lr)
        self.lr_t.fill_(float(lr))

    def sync_lr_from_groups(self) -> None:
        if self.param_groups[0]["lr"] != self._lr:
            self.set_lr(self.param_groups[0]["lr"])

    # ---- step -------------------------------------------------------------------
    def step(self, max_norm: float = 0.0, grad_scale: float = 1.0, zero_grad: bool = False,
             ext_norm: Optional[Tensor] = None) -> None:
        """Clip (if max_norm > 0) the flat gradient scaled by ``grad_scale`` and apply one Adam step.

        ``zero_grad``: leave the flat gradient zeroed (the fused kernel writes 0 instead of the clipped
        gradient; ``grads_zeroed`` reports whether that happened).  ``ext_norm``: partial sums of squares of the
        WHOLE gradient written by its producer (world > 1: the xGMI all-reduce kernel, ``FlatDDP.norm_parts``): the
        fused kernel takes the clip norm from them instead of re-reading the gradient, and the producers' ranges only
        stay unzeroed."""
        self.sync_lr_from_groups()
        f = self.flat
        b1, b2 = self.betas
        self.grads_zeroed = False
        if self.hip and self.single_launch:
            plan = sorted(self._plan.values(), key=lambda r: r[2])
            self._plan = {}
            self._dropped = set()
            ext = None
            if ext_norm is not None:
                # the producers' own partials are of the local gradient (the all-reduce rewrote their ranges): unused
                lib().adam_fused(f.data, f.grad, self.exp_avg, self.exp_avg_sq, self.partials, self.ticket, self.lr_t,
                                 self.step_t, b1, b2, self.eps, self.weight_decay, float(max_norm or 0.0),
                                 float(grad_scale), self.adamw, bool(zero_grad), self.grad_norm, self._health,
                                 [r[0] for r in plan], [r[1] for r in plan], ext_norm, True)
                self.grads_zeroed = bool(zero_grad)
                return
            if plan:
                # the kernel sums every partial of ext: hand it slots [0, last used] and zero the slots in between
                # that no covered range owns (a range dropped by a double registration left its stale partials there)
                top = plan[-1][2] + 1
                used = {r[2] for r in plan}
                for s in range(top):
                    if s not in used:
                        self.ext_parts[s * self._nparts:(s + 1) * self._nparts].zero_()
                ext = self.ext_parts[:top * self._nparts]
            lib().adam_fused(f.data, f.grad, self.exp_avg, self.exp_avg_sq, self.partials, self.ticket, self.lr_t,
                             self.step_t, b1, b2, self.eps, self.weight_decay, float(max_norm or 0.0),
                             float(grad_scale), self.adamw, bool(zero_grad), self.grad_norm, self._health,
                             [r[0] for r in plan], [r[1] for r in plan], ext, False)
            # covered ranges keep this step's gradient (their producers overwrite them next step)
            self.grads_zeroed = bool(zero_grad)
            return
        if self.hip:
            C = lib()
            C.grad_sqnorm(f.grad, float(grad_scale), self.partials, self.step_t)
            C.adam(f.data, f.grad, self.exp_avg, self.exp_avg_sq, self.partials, self.lr_t, self.step_t, b1, b2,
                   self.eps, self.weight_decay, float(max_norm or 0.0), float(grad_scale), self.adamw,
                   self.grad_norm, self.nonfinite)
            return
        self._step_torch(max_norm, grad_scale)

    @torch.no_grad()
    def _step_torch(self, max_norm: float, grad_scale: float) -> None:
        f = self.flat
        b1, b2 = self.betas
        g = f.grad
        if grad_scale != 1.0:
            g.mul_(grad_scale)
        # clip_grad_norm_ semantics: norm over all grads, coef = max_norm / (norm + 1e-6), clamp 1
        norms = torch.stack([v.norm() for v in f.views(g)])
        total = norms.norm()
        self.grad_norm.copy_(total.reshape(1))
        if not torch.isfinite(total):
            self.nonfinite += 1
        if max_norm and max_norm > 0:
            coef = torch.clamp(max_norm / (total + 1e-6), max=1.0)
            g.mul_(coef)
        self.step_t += 1
        t = float(self.step_t.item())
        lr = self._lr
        p, m, v = f.data, self.exp_avg, self.exp_avg_sq
        if self.adamw:
            p.mul_(1 - lr * self.weight_decay)
            gg = g
        else:
            gg = g.add(p, alpha=self.weight_decay) if self.weight_decay else g
        m.lerp_(gg, 1 - b1)
        v.mul_(b2).addcmul_(gg, gg, value=1 - b2)
        bc1 = 1 - b1 ** t
        bc2 = 1 - b2 ** t
        denom = (v.sqrt() / math.sqrt(bc2)).add_(self.eps)
        p.addcdiv_(m, denom, value=-lr / bc1)

    def zero_grad(self, set_to_none: bool = False) -> None:
        self.flat.zero_grad()

    # ---- torch.optim.Adam-compatible state dict (Lightning 'optimizer_states') -----
    def state_dict(self) -> Dict:
        step = self.step_t.detach().cpu().reshape(())
        state = {}
        for i, (mv, vv) in enumerate(zip(self.flat.views(self.exp_avg), self.flat.views(self.exp_avg_sq))):
            state[i] = {"step": step.clone(), "exp_avg": mv.detach().cpu().clone(),
                        "exp_avg_sq": vv.detach().cpu().clone()}
        groups = [dict(self.param_groups[0])]
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, sd: Dict) -> None:
        g = sd["param_groups"][0]
        self.betas = tuple(g.get("betas", self.betas))
        self.eps = g.get("eps", self.eps)
        self.weight_decay = g.get("weight_decay", self.weight_decay)
        self.set_lr(g["lr"])
        mvs = self.flat.views(self.exp_avg)
        vvs = self.flat.views(self.exp_avg_sq)
        step = 0.0
        for i, st in sd["state"].items():
            i = int(i)
            mvs[i].copy_(st["exp_avg"].to(mvs[i].device))
            vvs[i].copy_(st["exp_avg_sq"].to(vvs[i].device))
            step = float(st["step"])
        self.step_t.fill_(step)


_BLOCK = 256  # csrc/adam_tensors.h ADAM_BLOCK: elements of a tensor that share one power of two (8-bit moments)
_M32 = 0xFFFFFFFF


def _chances(seed: int, step: int, n: int, device, first: int = 0) -> tuple:
    """Two 16-bit random numbers for each of n elements from ``first`` on (csrc/adam_tensors.hip chance_of)."""
    i = torch.arange(first, first + n, device=device)
    x = (seed & _M32) ^ ((step * 0x9E3779B1) & _M32) ^ (((seed >> 32) * 0x85EBCA77) & _M32)
    x = ((i >> 32) * 0x27D4EB2F) & _M32 ^ (i & _M32) ^ x
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & _M32
    x = ((x ^ (x >> 15)) * 0x846CA68B) & _M32
    x = x ^ (x >> 16)
    return x & 0xFFFF, x >> 16


def _encode8(x: Tensor, chance, digits: int, loaded: bool = False) -> tuple:
    """Values (whole blocks) -> codes without sign and block exponents (csrc/adam_tensors.hip encode, load_exp)."""
    x = x.view(-1, _BLOCK)
    top = x.abs().amax(1)
    bad = ~(top < 2.0 ** 128)  # NaN, infinity, or past fp32's
    e = (torch.frexp(torch.where(bad, 0.0, top)).exponent - 1).clamp(-100, 126)
    if loaded:  # a power of two as the grid's top
        e = torch.where((torch.frexp(top).mantissa == 0.5) & (e > -100), e - 1, e)
    e = torch.where(top > 0, e, torch.full_like(e, -100))
    y = x.abs().double() * torch.exp2(-e.double())[:, None]
    ey = (torch.frexp(y).exponent - 1).clamp(min=-13)
    ey = torch.where(y > 0, ey, torch.full_like(ey, -13))
    q = torch.floor(y * torch.exp2(digits - ey.double()) + chance.view(-1, _BLOCK).double() / 65536).nan_to_num(0.0, 0.0)
    code = (((ey.long() + 13) << digits) + q.long()).clamp(0, 15 << digits)
    if digits == 4:
        code = torch.where((y > 0) & (code == 0), torch.ones_like(code), code)
    code = torch.where(bad[:, None], torch.zeros_like(code), code)
    return code.view(-1), torch.where(bad, torch.full_like(e, -128), e).to(torch.int8)


def _decode8(code: Tensor, e: Tensor, digits: int) -> Tensor:
    c = code.view(-1, _BLOCK).long()
    field, part = c >> digits, c & ((1 << digits) - 1)
    y = torch.where(field > 0, part + (1 << digits), part).double() * torch.exp2(field.clamp(min=1).double() - 14 - digits)
    y = (y * torch.exp2(e.double())[:, None]).float()
    return torch.where((e == -128)[:, None], torch.full_like(y, math.nan), y).view(-1)


class TensorAdam:
    """Adam (coupled L2) or AdamW over a list of tensors as they are: no flat buffer, any shapes, float32, bfloat16 or
    float16 parameters (float32 ones also with 16-bit gradients), with the moments in 32 or in 8 bits.

    Beside :class:`FusedAdam`, which needs every parameter and gradient in ONE fp32 buffer: two launches for up to 112
    tensors (``csrc/adam_tensors.hip``: gradient norm, update), two more for each further 112; lr and step live on the
    device, so a captured step replays.

    ``state_bits=8``: 256 elements of a tensor share a power of two; an element keeps 4 bits of exponent and 3 (first
    moment, with sign) or 4 (second) of mantissa, rounded up or down by chance so that the mean is right.  The random
    bits are a hash of ``seed``, the step and the element's place: the same run gives the same bits.  2 bytes a
    parameter instead of 8.

    A NaN or infinite gradient makes its parameter NaN, and in 8 bits the moments of its block; with ``max_norm`` the
    norm and so every parameter, as ``torch.nn.utils.clip_grad_norm_`` would.  ``skip_nonfinite``: a step whose gradient
    norm is not finite changes no parameter, moment or count (gradients are zeroed if asked for) and is counted in
    ``nonfinite``; the norm is then taken without ``max_norm`` too.

    ``step(grads=...)`` takes the gradients in the parameters' order; without it, ``p.grad``.  A parameter whose
    gradient is None is left out of the step: each tensor has its own count of steps (``steps``), as in torch.optim.
    Gradients are not changed unless ``zero_grad`` is set.
    """

    def __init__(self, params: Iterable[Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, adamw: bool = True, state_bits: int = 32, seed: int = 0,
                 skip_nonfinite: bool = False):
        self.params: List[Tensor] = list(params)
        if not self.params:
            raise ValueError("TensorAdam: no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"TensorAdam: state_bits must be 8 or 32, got {state_bits}")
        b1, b2 = self._checked(lr, betas, eps, weight_decay)
        dev = self.params[0].device
        for i, p in enumerate(self.params):
            if p.device != dev or p.dtype not in (torch.float32, torch.bfloat16, torch.float16) or not p.is_contiguous():
                raise ValueError(f"TensorAdam: parameter {i} must be contiguous float32, bfloat16 or float16 on {dev}, got "
                                 f"{p.dtype} on {p.device}")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i) for i, p in enumerate(self.params) if p.numel())
        for (_, end, i), (start, _, j) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f"TensorAdam: parameters {i} and {j} share memory")
        self.betas, self.eps, self.weight_decay = (b1, b2), float(eps), float(weight_decay)
        self.adamw, self.state_bits, self.seed = bool(adamw), int(state_bits), int(seed) & ((1 << 63) - 1)
        self.skip_nonfinite = bool(skip_nonfinite)
        self._lr = float(lr)
        #: where each tensor's moments start in the buffers of ``moments()`` (whole blocks of 256)
        self.offsets: List[int] = []
        at = 0
        for p in self.params:
            self.offsets.append(at)
            at += -(-p.numel() // _BLOCK) * _BLOCK
        self.padded = at
        f32 = dict(device=dev, dtype=torch.float32)
        if self.state_bits == 32:
            self._state = [torch.zeros(at, **f32), torch.zeros(at, **f32)]
        else:
            self._state = [torch.zeros(at, device=dev, dtype=torch.uint8) for _ in range(2)]
            self._state += [torch.full((at // _BLOCK,), -100, device=dev, dtype=torch.int8) for _ in range(2)]
        self.lr_t = torch.tensor([lr], **f32)
        #: steps taken, and by each tensor
        self.step_t = torch.zeros(1, **f32)
        self.steps = torch.zeros(len(self.params), **f32)
        #: norm of the last step's scaled gradient, and the count of steps where it was not finite: with ``max_norm`` or
        #: ``skip_nonfinite`` only
        self.grad_norm = torch.zeros(1, **f32)
        self.nonfinite = torch.zeros(1, **f32)
        self.grads_zeroed = False
        self.hip = use_hip(self.params[0])
        if self.hip:
            C = lib()
            self._blocks = [o // _BLOCK for o in self.offsets]
            # tables of a step: by their tensors, and where their workgroups fill a launch (16 Mi of at least 1024 elements)
            launches = -(-len(self.params) // C.ADAM_TABLE) + sum(1 + (p.numel() >> 33) for p in self.params if p.numel() >> 30)
            self._parts = torch.zeros(launches * C.adam_norm_parts(), device=dev, dtype=torch.float64)
            self._ticket = torch.zeros(1, device=dev, dtype=torch.int32)
            self._ctl = torch.zeros(8 + 4 * len(self.params), **f32)
        self.param_groups = [{
            "lr": lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay, "amsgrad": False,
            "maximize": False, "foreach": None, "capturable": True, "differentiable": False, "fused": True,
            "decoupled_weight_decay": self.adamw, "params": list(range(len(self.params))),
        }]

    @staticmethod
    def _checked(lr, betas, eps, weight_decay) -> tuple:
        b1, b2 = (float(b) for b in betas)
        # eps: a normal number of float32, as the reciprocal of what is not is taken for that of 0
        if not (0 <= b1 < 1 and 0 <= b2 < 1 and lr >= 0 and eps >= 2.0 ** -126 and weight_decay >= 0):
            raise ValueError(f"TensorAdam: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        return b1, b2

    # ---- lr (device-resident) --------------------------------------------------
    @property
    def lr(self) -> float:
        return self._lr

    def set_lr(self, lr: float) -> None:
        self._lr = float(lr)
        self.param_groups[0]["lr"] = float(lr)
        self.lr_t.fill_(float(lr))

    def sync_lr_from_groups(self) -> None:
        if self.param_groups[0]["lr"] != self._lr:
            self.set_lr(self.param_groups[0]["lr"])

    # ---- step -------------------------------------------------------------------
    @torch.no_grad()
    def step(self, max_norm: float = 0.0, grad_scale: float = 1.0, zero_grad: bool = False,
             grads: Optional[Sequence[Optional[Tensor]]] = None) -> None:
        """Scale the gradients by ``grad_scale``, clip their global norm to ``max_norm`` (if positive) and apply one step.
        ``zero_grad``: leave the gradients zeroed."""
        self.sync_lr_from_groups()
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"TensorAdam: {len(grads)} gradients for {len(self.params)} parameters")
        if all(g is None for g in grads):
            return
        if not self.hip:
            self._step_torch(grads, max_norm, grad_scale)
            if zero_grad:
                for g in grads:
                    if g is not None:
                        g.zero_()
        else:
            if not zero_grad:
                grads = [g if g is None or g.is_contiguous() else g.contiguous() for g in grads]
            lib().adam_tensors(self.params, grads, self._blocks, self._state, self.lr_t, self.step_t, self.steps, self._ctl,
                               self.grad_norm, self.nonfinite, self._parts, self._ticket, *self.betas, self.eps, self.weight_decay,
                               float(max_norm or 0.0), float(grad_scale), self.adamw, bool(zero_grad), self.skip_nonfinite,
                               self.seed)
        self.grads_zeroed = bool(zero_grad)

    def _step_torch(self, grads, max_norm, grad_scale) -> None:
        b1, b2 = self.betas
        scale = float(grad_scale)
        if (max_norm and max_norm > 0) or self.skip_nonfinite:
            norm = torch.stack([g.double().square().sum() for g in grads if g is not None]).sum().sqrt() * scale
            self.grad_norm.copy_(norm.float().reshape(1))
            if not torch.isfinite(self.grad_norm):
                self.nonfinite += 1
                if self.skip_nonfinite:
                    return
        if max_norm and max_norm > 0:
            scale = scale * torch.clamp(max_norm / (norm + 1e-6), max=1.0)
        self.step_t += 1
        m, v = self.moments()
        kind = torch.float32
        if self.state_bits == 8:  # up to their rounding in 64 bits, as csrc/adam_tensors.hip
            kind, m, v = torch.float64, m.double(), v.double()
        chances = torch.zeros(2, self.padded if self.state_bits == 8 else 0, dtype=torch.long, device=m.device)
        took = torch.zeros(self.padded // _BLOCK, dtype=torch.bool, device=m.device)
        for place, (p, g, o) in enumerate(zip(self.params, grads, self.offsets)):
            if g is None:
                continue
            if p.shape != g.shape:
                raise ValueError(f"TensorAdam: parameter {tuple(p.shape)} with gradient {tuple(g.shape)}")
            n = p.numel()
            if not n:
                continue
            self.steps[place] += 1
            t = int(self.steps[place].item())
            x, gg, mm, vv = p.float().reshape(-1), g.to(kind).reshape(-1) * scale, m[o:o + n], v[o:o + n]
            if not self.adamw:
                gg = gg + x.to(kind) * self.weight_decay
            mm.mul_(b1).add_(gg * (1 - b1))
            vv.mul_(b2).add_(gg * (1 - b2) * gg)
            x = x * (1 - self._lr * self.weight_decay) if self.adamw else x
            x = x - mm.float() / (vv.float().sqrt() / math.sqrt(1 - b2 ** t) + self.eps) * (self._lr / (1 - b1 ** t))
            p.copy_(x.view(p.shape))
            if self.state_bits == 8:
                end = o + -(-n // _BLOCK) * _BLOCK
                took[o // _BLOCK:end // _BLOCK] = True
                chances[0, o:end], chances[1, o:end] = _chances(self.seed, t, end - o, m.device, o)
        if self.state_bits == 8:
            self._put8(m, v, chances[0], chances[1], took)

    def _put8(self, m, v, low, high, took, loaded: bool = False) -> None:
        mc, me = _encode8(m, low, 3, loaded)
        vc, ve = _encode8(v, high, 4, loaded)
        mc = mc | ((torch.signbit(m).view(-1, _BLOCK) & (me != -128)[:, None]).view(-1).long() << 7)
        each = took.repeat_interleave(_BLOCK)
        for buf, new, mask in zip(self._state, (mc, vc, me, ve), (each, each, took, took)):
            buf.copy_(torch.where(mask, new.to(buf.dtype), buf))

    # ---- moments ------------------------------------------------------------------
    def moments(self, dtype: torch.dtype = torch.float32) -> tuple:
        """``(exp_avg, exp_avg_sq)`` of all tensors, tensor i from ``offsets[i]``.  32 bits: the optimizer's own buffers
        (``dtype`` float32).  8 bits: the values its codes stand for, float32 or bfloat16, which holds each exactly."""
        if self.state_bits == 32:
            if dtype != torch.float32:
                raise ValueError("TensorAdam: 32-bit moments are float32")
            return self._state[0], self._state[1]
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("TensorAdam: moments as float32 or bfloat16")
        if self.hip:
            m, v = (torch.empty(self.padded, device=self.lr_t.device, dtype=dtype) for _ in range(2))
            lib().adam_moments(self._state, m, v, True)
            return m, v
        c = self._state[0].long()
        m = _decode8(c & 127, self._state[2], 3)
        return torch.where(c >= 128, -m, m).to(dtype), _decode8(self._state[1], self._state[3], 4).to(dtype)

    # ---- torch.optim.Adam-compatible state dict -----------------------------------
    def _views(self, buf: Tensor) -> List[Tensor]:
        return [buf[o:o + p.numel()].view(p.shape) for p, o in zip(self.params, self.offsets)]

    def state_dict(self) -> Dict:
        steps = self.steps.detach().cpu()
        m, v = self.moments()
        state = {i: {"step": steps[i].clone(), "exp_avg": a.detach().cpu().clone(), "exp_avg_sq": b.detach().cpu().clone()}
                 for i, (a, b) in enumerate(zip(self._views(m), self._views(v)))}
        return {"state": state, "param_groups": [dict(self.param_groups[0])]}

    @torch.no_grad()
    def load_state_dict(self, sd: Dict) -> None:
        """Moments go to the nearest code in 8 bits (a state of this optimizer's own: to the values it had).  Tensors that
        the state has no entry of start anew."""
        g = sd["param_groups"][0]
        eps, decay = float(g.get("eps", self.eps)), float(g.get("weight_decay", self.weight_decay))
        self.betas = self._checked(g["lr"], g.get("betas", self.betas), eps, decay)
        self.eps, self.weight_decay = eps, decay
        self.param_groups[0].update(betas=self.betas, eps=self.eps, weight_decay=self.weight_decay)
        self.set_lr(g["lr"])
        m, v = self.moments()
        mvs, vvs = self._views(m), self._views(v)
        steps = [0.0] * len(self.params)
        for i in set(range(len(self.params))) - {int(i) for i in sd["state"]}:
            mvs[i].zero_(), vvs[i].zero_()
        for i, st in sd["state"].items():
            mvs[int(i)].copy_(st["exp_avg"].reshape(mvs[int(i)].shape))
            vvs[int(i)].copy_(st["exp_avg_sq"].reshape(vvs[int(i)].shape))
            steps[int(i)] = float(st["step"])
        self.steps.copy_(torch.tensor(steps))
        self.step_t.fill_(max(steps))
        if self.state_bits == 8:
            if self.hip:
                lib().adam_moments(self._state, m, v, False)
            else:
                half = torch.full((self.padded,), 0x8000, device=m.device)
                self._put8(m, v, half, half, torch.ones(self.padded // _BLOCK, dtype=torch.bool, device=m.device), True)
