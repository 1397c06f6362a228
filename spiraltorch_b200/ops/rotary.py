"""Rotary positions of queries and keys (``csrc/serving/rotary.cu``): any positions, half or interleaved pairs, a part of
the head, frequencies scaled for long contexts, forward and backward.

``elementwise.rope_`` remains the in-place form of packed training rows whose positions are their place in the sequence.

Reference parity: RoPE cache util (crates/st-core/src/util/rope_lru.rs); the reference has neither positions per row, interleaved
pairs nor scaling.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import native

launch_count = 0
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@dataclass(frozen=True)
class Scaling:
    """How frequencies change for contexts ``factor`` times longer than trained for.

    ``linear``: every frequency divided by the factor.  ``base``: the base raised by ``factor^(r / (r - 2))``, which divides the lowest
    frequency by the factor and keeps the highest.  ``bands``: a frequency that turns ``high`` times or more over the
    ``original`` length is kept, one that turns ``low`` times or less is divided by the factor, a ramp between them."""
    kind: str
    factor: float
    original: int = 4096
    low: float = 1.0
    high: float = 32.0

    def __post_init__(self):
        if self.kind not in ("linear", "base", "bands"):
            raise ValueError(f"rotary scaling '{self.kind}' is none of 'linear', 'base', 'bands'")
        if not (math.isfinite(self.factor) and self.factor > 0):
            raise ValueError(f"rotary scaling factor must be positive, got {self.factor}")
        if self.kind == "bands" and not (self.original > 0 and self.high > self.low):
            raise ValueError("rotary scaling by bands needs original > 0 and high > low")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Scaling] = None, device="cpu") -> torch.Tensor:
    """Angle per position of each rotated pair, fp64 ``[rotary_dim / 2]``: ``base^(-2 j / rotary_dim)``, scaled."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"rotary base must be positive, got {base}")
    if scaling is not None and scaling.kind == "base" and rotary_dim > 2:
        base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if scaling is not None and scaling.kind == "linear":
        f = f / scaling.factor
    if scaling is not None and scaling.kind == "bands":
        turns = scaling.original * f / (2.0 * math.pi)
        keep = ((turns - scaling.low) / (scaling.high - scaling.low)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / scaling.factor)
    return f.to(device)


def rotary_reference(x: torch.Tensor, positions: torch.Tensor, freq: torch.Tensor, interleaved: bool = False, magnitude: float = 1.0,
                     backward: bool = False) -> torch.Tensor:
    """``x`` ``[..., heads, dim]``, ``positions`` ``[...]``: angles in fp64, products in fp32 (fp64 for fp64 ``x``)."""
    angle = positions.to(torch.float64)[..., None, None] * freq
    t = torch.float64 if x.dtype == torch.float64 else torch.float32
    c, s = (angle.cos() * magnitude).to(t), (angle.sin() * (-magnitude if backward else magnitude)).to(t)
    n, xf = freq.numel(), x.to(t)
    a, b = (xf[..., 0:2 * n:2], xf[..., 1:2 * n:2]) if interleaved else (xf[..., :n], xf[..., n:2 * n])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, xf[..., 2 * n:]], -1).to(x.dtype)


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """``x`` as ``[tokens, heads, dim]`` without a copy of a strided view that has such a form."""
    if x.stride()[-1] != 1 and x.shape[-1] > 1:
        raise ValueError(f"rotary: {name} must have contiguous head elements")
    return x if x.dim() == 3 else x.flatten(0, -3) if x.dim() > 3 else x.unsqueeze(0)


def _check(q, k, positions, freq) -> None:
    if q.dtype not in _TYPES and not (q.dtype == torch.float64 and not q.is_cuda):
        raise ValueError(f"rotary: bf16, fp16 and fp32 tensors, got {q.dtype}")
    if q.dim() < 2 or positions.shape != q.shape[:-2]:
        raise ValueError(f"rotary: positions {tuple(positions.shape)} do not match q {tuple(q.shape)} without heads and head elements")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"rotary: positions must be int32 or int64, got {positions.dtype}")
    if k is not None and (k.dtype != q.dtype or k.shape[:-2] != positions.shape or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"rotary: k {tuple(k.shape)} {k.dtype} does not match q {tuple(q.shape)} {q.dtype}")
    if freq.dtype != torch.float64 or freq.dim() != 1 or not freq.is_contiguous():
        raise ValueError("rotary: freq must be a contiguous fp64 vector, as frequencies() gives")
    if not 0 < 2 * freq.numel() <= q.shape[-1]:
        raise ValueError(f"rotary: {freq.numel()} frequencies rotate {2 * freq.numel()} elements of heads of {q.shape[-1]}")


def _launch(q, k, qo, ko, positions, freq, interleaved, magnitude, backward) -> None:
    """Rotates ``[tokens, heads, dim]`` views q and k (None: no keys) into qo and ko."""
    global launch_count
    index = native.require_cuda("rotary", q, k, positions, freq)
    kk, kko, hk = (q, qo, 0) if k is None else (k, ko, k.shape[1])
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return
    h = q.shape[1]
    if h == 0:
        q, qo, h, kk, kko, hk = k, ko, hk, k, ko, 0
    with native.on_device(index):
        st = native.entry("st_rotary", "pppppipqiiiiqqqqqqqqifiip")(
            q.data_ptr(), kk.data_ptr(), qo.data_ptr(), kko.data_ptr(), positions.data_ptr(), int(positions.dtype == torch.int64),
            freq.data_ptr(), q.shape[0], h, hk, q.shape[2], freq.numel(), *q.stride()[:2], *kk.stride()[:2], *qo.stride()[:2], *kko.stride()[:2],
            int(interleaved), magnitude, int(backward), _TYPES[q.dtype], native.raw_stream(index))
    native.check(st, "st_rotary")
    launch_count += 1


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _apply(q, k, positions, freq, interleaved, magnitude, backward):
    if not native.use_native(q):
        return tuple(None if x is None else rotary_reference(x, positions, freq, interleaved, magnitude, backward) for x in (q, k))
    qo, ko = _like(q), None if k is None else _like(k)
    _launch(_rows(q, "q"), None if k is None else _rows(k, "k"), qo if qo.dim() == 3 else _rows(qo, "q"), ko if ko is None or ko.dim() == 3 else _rows(ko, "k"),
            positions.contiguous(), freq, interleaved, magnitude, backward)
    return qo, ko


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freq, form):
        ctx.save_for_backward(positions, freq)
        ctx.save_for_forward(positions, freq)
        ctx.form, ctx.shapes = form, (q.shape, None if k is None else k.shape)
        ctx.set_materialize_grads(False)
        return _apply(q, k, positions, freq, *form)

    @staticmethod
    def jvp(ctx, tq, tk, *_):      # linear in q and k; None: no tangent, or no k
        tq, tk = (t if t is None or t.stride()[-1] == 1 else t.contiguous() for t in (tq, tk))
        if tq is None:
            return tk.new_zeros(ctx.shapes[0]), _rotate(tk, None, *ctx.saved_tensors, *ctx.form)[0]
        if tk is None and ctx.shapes[1] is not None:
            return _rotate(tq, None, *ctx.saved_tensors, *ctx.form)[0], tq.new_zeros(ctx.shapes[1])
        return _rotate(tq, tk, *ctx.saved_tensors, *ctx.form)

    @staticmethod
    def backward(ctx, dq, dk):
        need_q, need_k, *_ = ctx.needs_input_grad
        dq, dk = (g if need and (g is None or g.stride()[-1] == 1) else g.contiguous() if need and g is not None else None
                  for g, need in ((dq, need_q), (dk, need_k)))
        if dq is None and dk is None:
            return None, None, None, None, None
        interleaved, magnitude, back = ctx.form
        positions, freq = ctx.saved_tensors
        if dq is None:
            return None, _rotate(dk, None, positions, freq, interleaved, magnitude, not back)[0], None, None, None
        return *_rotate(dq, dk, positions, freq, interleaved, magnitude, not back), None, None, None


def _rotate(q, k, positions, freq, interleaved, magnitude, backward):
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or native.has_tangent(q, k):
        return _RotaryFn.apply(q, k, positions, freq, (interleaved, magnitude, backward))
    return _apply(q, k, positions, freq, interleaved, magnitude, backward)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, *, interleaved: bool = False,
           magnitude: float = 1.0):
    """``(q, k)`` rotated, in new contiguous tensors; differentiable in both, in reverse and in forward mode.

    ``q`` ``[..., heads, dim]`` and ``k`` ``[..., kv_heads, dim]`` or None: bf16, fp16 or fp32 with contiguous head elements and any other strides;
    ``positions`` ``[...]`` int32 or int64; ``freq`` from :func:`frequencies`, on the same device: the first ``2 * len(freq)`` elements of a head are
    rotated, the others copied.  Pairs are ``(j, len(freq) + j)``, or ``(2 j, 2 j + 1)`` where ``interleaved``.  ``magnitude`` multiplies what is rotated."""
    _check(q, k, positions, freq)
    return _rotate(q, k, positions, freq, interleaved, float(magnitude), False)


def rotary_(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, *, interleaved: bool = False,
            magnitude: float = 1.0, backward: bool = False):
    """The same in place, for tensors or views of a fused projection (no autograd); ``backward`` turns the other way, as gradients are."""
    _check(q, k, positions, freq)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        raise ValueError("rotary_: in-place form of tensors that require gradients; use rotary()")
    if native.has_tangent(q, k):
        raise ValueError("rotary_: in-place form of tensors with tangents; use rotary()")
    if not native.use_native(q):
        for x in (q, k):
            if x is not None:
                x.copy_(rotary_reference(x, positions, freq, interleaved, magnitude, backward))
        return q, k
    views = []
    for x, n in ((q, "q"), (k, "k")):
        v = None if x is None else _rows(x, n)
        if v is not None and v.data_ptr() != x.data_ptr() or v is not None and v.numel() and x.numel() != v.numel():
            raise ValueError(f"rotary_: {n} has no form of rows and heads to work on in place")
        views.append(v)
    _launch(*views, *views, positions.contiguous(), freq, interleaved, float(magnitude), backward)
    return q, k
