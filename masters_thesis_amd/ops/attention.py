"""Attention over sequences of any length, with its gradients (``csrc/mha.hip``).

The transformer's fused attention (``ops.extras``) covers windows of at most 64 tokens.  These are the operators for
everything longer -- and for padded batches, causal order, query heads that share key heads and single queries -- in
bfloat16, float16 and float32:

* :func:`attention` -- differentiable, ``softmax(scale * q k^T) v`` over the keys that each query sees;
* :func:`attention_forward` / :func:`attention_backward` -- the two halves, for a caller that keeps its own graph;
* :func:`rope_` -- rotary positions of packed projections, in place.

Shapes are ``(batch, tokens, heads, dim)``.  Nothing of the size ``tokens x tokens`` is stored: the forward leaves each
row's log-sum-exp, the backward recomputes the probabilities from it.  The backward uses no atomics: the same inputs
give the same bits.

On the CPU the same functions compute the plain formula in PyTorch.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from ._lib import lib, use_hip

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_DIM = 128


def _check(q: Tensor, k: Tensor, v: Tensor, key_lengths: Optional[Tensor], scale: Optional[float]) -> float:
    """The arguments' checks on the CPU (on the GPU: csrc/bindings.cpp mha_check); returns the scale."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"attention: {name} must be (batch, tokens, heads, dim), got {tuple(t.shape)}")
        if t.dtype not in _TYPES:
            raise ValueError(f"attention: {name} must be bfloat16, float16 or float32, got {t.dtype}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"attention: q is {q.dtype} on {q.device}, {name} {t.dtype} on {t.device}")
    if k.shape != v.shape:
        raise ValueError(f"attention: k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"attention: q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or dim")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"attention: {q.shape[2]} query heads are not a multiple of {k.shape[2]} key heads")
    if q.shape[3] % 8 or not 8 <= q.shape[3] <= MAX_DIM:
        raise ValueError(f"attention: head dim must be a multiple of 8 up to {MAX_DIM}, got {q.shape[3]}")
    if key_lengths is not None:
        if key_lengths.shape != (q.shape[0],) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"attention: key_lengths must be int32 or int64 ({q.shape[0]},), got {key_lengths.dtype} "
                             f"{tuple(key_lengths.shape)}")
        if key_lengths.device != q.device:
            raise ValueError(f"attention: key_lengths is on {key_lengths.device}, q on {q.device}")
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if not 2.0 ** -120 <= scale <= 2.0 ** 120:  # a number that float32 holds
        raise ValueError(f"attention: scale must be positive, 2^-120 to 2^120, got {scale}")
    return scale


def _seen(q: Tensor, k: Tensor, causal: bool, key_lengths: Optional[Tensor]) -> Tensor:
    """(batch or 1, 1, Tq, Tk): whether query i, at position i + Tk - Tq, sees key j."""
    tq, tk = q.shape[1], k.shape[1]
    j = torch.arange(tk, device=q.device)
    see = torch.ones(1, 1, tq, tk, dtype=torch.bool, device=q.device)
    if causal:
        see = see & (j[None, :] <= torch.arange(tq, device=q.device)[:, None] + (tk - tq))
    if key_lengths is not None:
        see = see & (j < key_lengths[:, None])[:, None, None, :]
    return see


def attention_reference(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, key_lengths: Optional[Tensor] = None,
                        scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """The plain formula (differentiable, in the inputs' type): out and log-sum-exp ``(batch, heads, Tq)``."""
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    group = q.shape[2] // k.shape[2]
    see = _seen(q, k, causal, key_lengths)
    visible = see.any(2).any(1)  # (batch or 1, Tk): a key that no query sees takes no part, whatever it holds
    keep = visible[:, :, None, None]
    kk = torch.where(keep, k, torch.zeros((), dtype=k.dtype, device=k.device)).repeat_interleave(group, 2).transpose(1, 2)
    vv = torch.where(keep, v, torch.zeros((), dtype=v.dtype, device=v.device)).repeat_interleave(group, 2).transpose(1, 2)
    s = (q.transpose(1, 2) @ kk.transpose(-1, -2).contiguous() * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else s.new_full(s.shape[:3], -math.inf)
    empty = ~see.any(-1, keepdim=True)
    p = torch.exp(s - lse.masked_fill(empty[..., 0], 0.0)[..., None])
    return (p @ vv.contiguous()).transpose(1, 2), lse


def attention_forward(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, key_lengths: Optional[Tensor] = None,
                      scale: Optional[float] = None, need_lse: bool = True) -> Tuple[Tensor, Optional[Tensor]]:
    """``(out, lse)`` without recording a graph: see :func:`attention`.  ``lse`` (batch, heads, Tq) float32 is what
    :func:`attention_backward` takes; None with ``need_lse=False``."""
    with torch.no_grad():
        if use_hip(q):
            return lib().mha(q, k, v, key_lengths, causal, scale, need_lse)
        scale = _check(q, k, v, key_lengths, scale)
        out, lse = attention_reference(q.float(), k.float(), v.float(), causal=causal, key_lengths=key_lengths, scale=scale)
        return out.to(q.dtype).contiguous(), (lse if need_lse else None)


def _check_grads(grads, ins, others) -> None:
    """Places to write gradients into, on the CPU (on the GPU: csrc/bindings.cpp mha_backward)."""
    places = []
    for i, (g, x) in enumerate(zip(grads, ins)):
        if g.shape != x.shape or g.dtype != x.dtype or g.device != x.device:
            raise ValueError(f"attention_backward: gradient {i} must be {tuple(x.shape)} {x.dtype} on {x.device}")
        if not g.numel():
            continue
        unit = 16 // g.element_size()
        if g.stride(3) != 1 or g.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % unit) for s, n in zip(g.stride()[:3], g.shape)):
            raise ValueError(f"attention_backward: gradient {i} must have contiguous rows that start on 16 bytes")
        at = torch.full((1,), g.data_ptr() // g.element_size())
        for s, n in zip(g.stride(), g.shape):
            at = (at[:, None] + s * torch.arange(n)).view(-1)
        lo, hi = int(at.min()) * g.element_size(), (int(at.max()) + 1) * g.element_size()
        for t in others:
            if t.numel():
                end = t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
                if lo < end and t.data_ptr() < hi:
                    raise ValueError(f"attention_backward: gradient {i} lies in the memory of an input")
        places.append(at)
    if places and torch.cat(places).unique().numel() < sum(at.numel() for at in places):
        raise ValueError("attention_backward: elements of the gradients share memory")


def attention_backward(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, *, causal: bool = False,
                       key_lengths: Optional[Tensor] = None, scale: Optional[float] = None,
                       grads: Optional[Tuple[Tensor, Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients ``(dq, dk, dv)`` of :func:`attention` from its output and log-sum-exp.  ``grads``: tensors to write
    them into (any strides with 16-byte rows, for instance views of one packed buffer; neither each other's memory nor the
    inputs')."""
    if use_hip(q):
        return lib().mha_backward(dout, q, k, v, out, lse, key_lengths, causal, scale, *(grads or (None, None, None)))
    scale = _check(q, k, v, key_lengths, scale)
    if dout.shape != q.shape or out.shape != q.shape or lse.shape != (q.shape[0], q.shape[2], q.shape[1]):
        raise ValueError(f"attention_backward: dout {tuple(dout.shape)} and out {tuple(out.shape)} must be {tuple(q.shape)}, "
                         f"lse {tuple(lse.shape)} (batch, heads, queries)")
    if grads is not None:
        _check_grads(grads, (q, k, v), (dout, q, k, v, out, lse))
    got = _backward_reference(dout, q, k, v, causal, key_lengths, scale)
    if grads is None:
        return got
    with torch.no_grad():
        for g, x in zip(grads, got):
            g.copy_(x)
    return grads


def _backward_reference(dout, q, k, v, causal, key_lengths, scale):
    f = torch.float32
    sees = _seen(q, k, causal, key_lengths).any(-1)[:, 0, :, None, None]  # (batch or 1, Tq, 1, 1)
    q, dout = (torch.where(sees, t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (q, dout))  # others take no part
    leaves = [t.detach().to(f).requires_grad_() for t in (q, k, v)]
    with torch.enable_grad():
        out, _ = attention_reference(*leaves, causal=causal, key_lengths=key_lengths, scale=scale)
    return tuple(g.to(q.dtype) for g in torch.autograd.grad(out, leaves, dout.to(f)))


class _Once(torch.autograd.Function):
    """Gradients as they are; differentiating them raises.  It takes what they depend on too: without a way to it,
    torch.autograd.grad would leave this node out instead of running it."""

    @staticmethod
    def forward(ctx, dq, dk, dv, *inputs):
        return dq.view_as(dq), dk.view_as(dk), dv.view_as(dv)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("attention: its gradients are not differentiable")


class _AttentionFn(torch.autograd.Function):
    """The CPU's recorded form (on the GPU: csrc/bindings.cpp MhaFn)."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, causal, scale):
        out, lse = attention_forward(q, k, v, causal=causal, key_lengths=key_lengths, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths)
        ctx.causal, ctx.scale = causal, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _):
        q, k, v, out, lse, key_lengths = ctx.saved_tensors
        with torch.no_grad():
            grads = attention_backward(dout, q, k, v, out, lse, causal=ctx.causal, key_lengths=key_lengths, scale=ctx.scale)
        if torch.is_grad_enabled():  # create_graph
            grads = _Once.apply(*grads, q, k, v, dout)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, key_lengths: Optional[Tensor] = None,
              scale: Optional[float] = None, return_lse: bool = False):
    """``softmax(scale * q k^T) v`` over the keys that each query sees.

    ``q`` (batch, Tq, heads, dim); ``k``, ``v`` (batch, Tk, key heads, dim): query head h takes key head
    ``h // (heads // key heads)``.  dim: a multiple of 8 up to 128.  bfloat16, float16 or float32, accumulated in
    float32.  Any strides; rows that do not start on 16 bytes are copied first.

    Query i stands at position ``i + Tk - Tq`` (the queries are the last of the sequence: a single query sees the whole
    cache).  ``causal``: it sees the keys up to its position.  ``key_lengths`` (batch,): the keys of each sequence;
    what lies behind them is never read as a number (it may be NaN) and gets zero gradients; lengths outside 0 .. Tk
    are clamped.  (A NaN or infinity within the lengths may reach queries whose causal order hides its key, and one in a
    query or its output gradient the gradients of keys that are hidden from it.)  A query that sees no key returns 0,
    log-sum-exp -inf, and contributes no gradient, whatever it and its output gradient hold.  ``scale``: positive (2^-120 to
    2^120), default ``1 / sqrt(dim)``.

    ``return_lse``: also the log-sum-exp (batch, heads, Tq), float32, not differentiable.

    First derivatives only: differentiating the gradients raises, on the GPU also forward-mode derivatives.

    Captured into a graph, the backward needs leaves whose earlier graphs are gone: it raises where one is alive on
    another stream.
    """
    if use_hip(q):
        out, lse = lib().mha(q, k, v, key_lengths, causal, scale, return_lse)
    elif torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        out, lse = _AttentionFn.apply(q, k, v, key_lengths, bool(causal), _check(q, k, v, key_lengths, scale))
    else:
        out, lse = attention_forward(q, k, v, causal=causal, key_lengths=key_lengths, scale=scale, need_lse=return_lse)
    return (out, lse) if return_lse else out


def rope_(x: Tensor, seq: int, heads: int, dim: int, base: float = 10000.0, inverse: bool = False) -> Tensor:
    """Turns the first ``heads * dim`` columns of ``x`` (tokens of ``seq``-long sequences, columns) in place: the pair
    (2 i, 2 i + 1) of each head by ``position * base^(-2 i / dim)`` (back with ``inverse``).  bfloat16 or float32.
    Not differentiable: a tensor that a gradient passes through is refused (its gradient is turned with ``inverse`` by
    whoever keeps the graph, as the encoder does)."""
    if not use_hip(x):
        raise ValueError("rope_ is the GPU form: on the CPU use ops.extras.rope_reference")
    lib().rope_(x, int(seq), int(heads), int(dim), float(base), bool(inverse))
    return x
