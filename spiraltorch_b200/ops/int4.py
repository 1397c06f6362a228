"""Weights of four bits and products with them (``csrc/serving/int4_weights.cu``, ``csrc/serving/int4_linear.cu``).

A matrix ``[out, in]`` is held as ``q * s``: a code ``-8 <= q <= 7`` per weight and a scale per row and group of 32, 64 or 128 inputs.

    held = quantize(weight, group=64)              # once, and again after an update
    y = linear(x, held, bias, act="gelu")          # any number of rows, from one token's to a prompt's
    weight = dequantize(held, torch.bfloat16)

The scale is minus an eighth of the group's element of largest magnitude (the negative one of two), rounded to 4 significant bits (ties to even), its
magnitude within ``2^-20`` and ``1.875 * 2^12``; the code is the weight over the scale, rounded to the nearest (ties to even) and clamped.  Every ``q * s`` is a
bf16 and an fp16 number, so all kernels, and ``dequantize`` in any type, work with the same weights.  A group with a NaN or an infinity is NaN.

CPU tensors use a plain PyTorch statement of the same (also the test oracle).  The reference has no weights of fewer than 8 bits.
"""
from __future__ import annotations

import struct
from contextlib import nullcontext
from typing import Optional

import torch

from . import native
from .gemm import gelu_tanh

launch_count = 0
GROUPS = (32, 64, 128)
LEAST_SCALE, LARGEST_SCALE = 2.0 ** -20, 1.875 * 2.0 ** 12
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTS = {None: 0, "relu": 1, "gelu": 2}


# StInt4LinearArgs of csrc/serving/int4_linear.cu, in one call: a ctypes object for each of 16 arguments costs as much as the launch
_pack_args = struct.Struct("@6P3q6i").pack
_pack_weights = struct.Struct("@3Pq4i").pack      # StInt4WeightsArgs of int4_weights.cu


class Weights:
    """``codes`` uint8 ``[tiles down, tiles across, 512]`` (16 rows by 64 columns each, in the order of the kernels), ``scales`` bf16 ``[tiles down, groups, 16]``;
    the matrix's ``out_features`` and ``in_features``, and the inputs to a scale."""
    __slots__ = ("codes", "scales", "out_features", "in_features", "group")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, out_features: int, in_features: int, group: int):
        if group not in GROUPS:
            raise ValueError(f"int4: groups of {GROUPS} inputs, got {group}")
        if not (0 < out_features <= 1 << 30 and 0 < in_features <= 1 << 30):
            raise ValueError(f"int4: a matrix of {out_features} x {in_features} is not supported")
        down = -(-out_features // 16)
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.bfloat16 or not codes.is_contiguous() or not scales.is_contiguous() \
                or codes.shape != (down, -(-in_features // 64), 512) or scales.shape != (down, -(-in_features // group), 16) or codes.device != scales.device:
            raise ValueError(f"int4: codes {codes.dtype} {tuple(codes.shape)} and scales {scales.dtype} {tuple(scales.shape)} are no weights of "
                             f"{out_features} x {in_features} in groups of {group}")
        self._set(codes, scales, out_features, in_features, group)

    def _set(self, *values):
        for name, value in zip(self.__slots__, values):
            object.__setattr__(self, name, value)
        return self

    def __setattr__(self, name, value):
        raise AttributeError("int4.Weights: sizes and memory stay as they were checked")

    @classmethod
    def allocate(cls, out_features: int, in_features: int, group: int = 64, device="cuda") -> "Weights":
        """Room for :func:`quantize` to write to."""
        if group not in GROUPS or not (0 < out_features <= 1 << 30 and 0 < in_features <= 1 << 30):
            raise ValueError(f"int4: a matrix of {out_features} x {in_features} in groups of {group} is not supported")
        down = -(-out_features // 16)
        # tensors of inference mode could not be written to outside it, nor be looked at for updates by a gradient
        with torch.inference_mode(False) if torch.is_inference_mode_enabled() else nullcontext():
            codes = torch.empty((down, -(-in_features // 64), 512), dtype=torch.uint8, device=device)
            scales = codes.new_empty((down, -(-in_features // group), 16), dtype=torch.bfloat16)
        return cls.__new__(cls)._set(codes, scales, out_features, in_features, group)

    def __reduce__(self):
        return Weights, tuple(getattr(self, name) for name in self.__slots__)

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def to(self, device) -> "Weights":
        with torch.inference_mode(False) if torch.is_inference_mode_enabled() else nullcontext():
            return Weights(self.codes.to(device), self.scales.to(device), self.out_features, self.in_features, self.group)


# ---- plain statement ------------------------------------------------------------------------------------------------------------
def quantize_reference(weight: torch.Tensor, group: int):
    """Codes ``[out, in]`` int8 and scales ``[out, groups]`` fp32."""
    n, k = weight.shape
    g = torch.nn.functional.pad(weight.double(), (0, -k % group)).unflatten(1, (-1, group))
    low, high = g.amin(-1), g.amax(-1)
    m, e = torch.frexp(torch.where(high > -low, high, low) * -0.125)
    s = torch.ldexp(torch.round(m * 16), e - 4)
    s = torch.where(s < 0, -1.0, 1.0) * s.abs().clamp(LEAST_SCALE, LARGEST_SCALE)
    s = torch.where(g.isfinite().all(-1), s, float("nan"))
    q = torch.round(g / s[..., None]).clamp(-8, 7).nan_to_num(nan=-8.0)
    return q.flatten(1)[:, :k].to(torch.int8), s.float()


def _tiles(q: torch.Tensor) -> torch.Tensor:
    """Codes ``[out, in]`` in the order of the kernels: see ``csrc/serving/int4.cuh``."""
    n, k = q.shape
    v = torch.nn.functional.pad(q.to(torch.int16) + 8, (0, -k % 64, 0, -n % 16), value=8)
    # [down, half of the rows, g, across, word, half of the columns, t, parity]
    v = v.view(-(-n // 16), 2, 8, -(-k // 64), 4, 2, 4, 2)
    v = v.permute(0, 3, 2, 6, 4, 7, 5, 1)      # [down, across, g, t, word, parity (nibbles 0-3, 4-7), column half, row half]
    v = v.flatten(-2)                          # nibble e = 2 * column half + row half
    v = v.flatten(-2).unflatten(-1, (4, 2))    # bytes of two nibbles, the lower first
    return (v[..., 0] | v[..., 1] << 4).to(torch.uint8).reshape(v.shape[0], v.shape[1], 512)


def _untile(codes: torch.Tensor, n: int, k: int) -> torch.Tensor:
    b = codes.to(torch.int16)
    v = torch.stack([b & 15, b >> 4], -1).view(codes.shape[0], codes.shape[1], 8, 4, 4, 2, 2, 2)
    v = v.permute(0, 7, 2, 1, 4, 6, 3, 5)
    return (v.reshape(codes.shape[0] * 16, codes.shape[1] * 64) - 8)[:n, :k].to(torch.int8)


def _row_scales(w: Weights) -> torch.Tensor:
    """``[out, groups]`` fp32."""
    s = w.scales.unflatten(-1, (8, 2)).permute(0, 3, 2, 1)
    return s.reshape(-1, w.scales.shape[1])[:w.out_features].float()


def dequantize_reference(w: Weights, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    s = _row_scales(w).to(torch.float64 if dtype == torch.float64 else torch.float32).repeat_interleave(w.group, 1)[:, :w.in_features]
    return (_untile(w.codes, w.out_features, w.in_features).to(s.dtype) * s).to(dtype)


def _matmul(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """In their type, under autocast too."""
    with torch.autocast(a.device.type, enabled=False):
        return a @ b


def linear_reference(x, weight, bias=None, act=None, residual=None):
    """``weight`` ``[out, in]``: sums in fp32 (fp64 for fp64 ``x``), rounded once."""
    t = torch.float64 if x.dtype == torch.float64 else torch.float32
    y = _matmul(x.to(t), weight.to(t).T)
    if bias is not None:
        y = y + bias.to(t)
    y = torch.relu(y) if act == "relu" else gelu_tanh(y) if act == "gelu" else y
    return (y if residual is None else y + residual.to(t)).to(x.dtype)


# ---- quantising -----------------------------------------------------------------------------------------------------------------
def quantize(weight: torch.Tensor, group: int = 64, *, out: Optional[Weights] = None) -> Weights:
    """``weight`` ``[out, in]`` in bf16, fp16 or fp32 (rows may be strided) in four bits; ``out``: written to instead of new memory, as after
    an update of weights that a captured step holds."""
    on_cuda = weight.is_cuda
    if weight.dim() != 2 or weight.dtype not in _TYPES and not (weight.dtype == torch.float64 and not on_cuda):
        raise ValueError(f"int4.quantize: a bf16, fp16 or fp32 matrix, got {weight.dtype} {tuple(weight.shape)}")
    if group not in GROUPS:
        raise ValueError(f"int4.quantize: groups of {GROUPS} inputs, got {group}")
    n, k = weight.shape
    if out is None:
        out = Weights.allocate(n, k, group, weight.device)
    elif (out.out_features, out.in_features, out.group) != (n, k, group):
        raise ValueError(f"int4.quantize: a {n} x {k} matrix in groups of {group} into weights of {out.out_features} x {out.in_features} in groups of {out.group}")
    else:
        native.same_device("int4.quantize", weight, out.codes)
        torch.autograd.graph.increment_version(out.codes)      # gradients of products with what they held are refused
    if not on_cuda:
        q, s = quantize_reference(weight.detach(), group)
        out.codes.copy_(_tiles(q))
        s = torch.nn.functional.pad(s, (0, 0, 0, -n % 16), value=LEAST_SCALE)
        out.scales.copy_(s.view(-1, 2, 8, s.shape[1]).permute(0, 3, 2, 1).flatten(-2))
        return out
    stride, step = weight.stride()
    if step != 1 and k > 1:
        weight, stride = weight.contiguous(), k
    _weights_call("st_int4_quantize", weight, stride, out)
    return out


def dequantize(w: Weights, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``[out, in]`` in bf16, fp16 or fp32: the same numbers in each."""
    if not w.codes.is_cuda:
        return dequantize_reference(w, dtype)
    if dtype not in _TYPES:
        raise ValueError(f"int4.dequantize: bf16, fp16 or fp32, got {dtype}")
    y = w.codes.new_empty((w.out_features, w.in_features), dtype=dtype)
    _weights_call("st_int4_dequantize", y, w.in_features, w)
    return y


def _weights_call(name: str, matrix: torch.Tensor, stride: int, w: Weights) -> None:
    global launch_count
    index = matrix.get_device()
    args = _pack_weights(matrix.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), stride, w.out_features, w.in_features, w.group, _TYPES[matrix.dtype])
    with native.on_device(index):
        st = native.entry(name, "sp")(args, native.raw_stream(index))
    if st:
        native.check(st, name)
    launch_count += 1


# ---- products -------------------------------------------------------------------------------------------------------------------
def _boundaries(x2: torch.Tensor) -> torch.Tensor:
    """``x2``, or a copy of it, with every row on a 16-byte boundary, as tiled copies need them."""
    rows, cols = x2.shape
    stride, step = x2.stride()
    if step == 1 and stride % 8 == 0 and stride >= cols and x2.data_ptr() % 16 == 0:
        return x2
    return x2.new_empty((rows, -(-cols // 8) * 8))[:, :cols].copy_(x2)


def _product(x2, w, bias, act, residual2):
    """``[rows, in]`` to ``[rows, out]``."""
    global launch_count
    if not x2.is_cuda:
        return linear_reference(x2, dequantize_reference(w, x2.dtype if x2.dtype == torch.float64 else torch.float32), bias, act, residual2)
    index = native.require_cuda("int4.linear", x2, w.codes, w.scales, bias, residual2)
    (rows, cols), n = x2.shape, w.out_features
    y = x2.new_empty((rows, n))
    if rows == 0:
        return y
    if rows > 16 or rows > 8 and native.entry("st_int4_is_wide", "iii")(rows, n, cols):
        x2 = _boundaries(x2)
    x_row, step = x2.stride()
    if step != 1 and cols > 1:
        x2, x_row = x2.contiguous(), cols
    residual_row = 0
    if residual2 is not None:
        residual_row, step = residual2.stride()
        if step != 1 and n > 1:
            residual2, residual_row = residual2.contiguous(), n
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    args = _pack_args(x2.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if residual2 is None else residual2.data_ptr(),
                      y.data_ptr(), x_row, residual_row, n, rows, n, cols, w.group, _ACTS[act], _TYPES[x2.dtype])
    with native.on_device(index):
        st = native.entry("st_int4_linear", "sp")(args, native.raw_stream(index))
    if st:
        native.check(st, "st_int4_linear")
    launch_count += 1
    return y


def _input_gradient(dy2, w):
    """``[rows, out]`` to ``[rows, in]``: ``dy W``."""
    global launch_count
    if not dy2.is_cuda:
        t = torch.float64 if dy2.dtype == torch.float64 else torch.float32
        return _matmul(dy2.to(t), dequantize_reference(w, t)).to(dy2.dtype)
    dy2 = _boundaries(dy2)
    index = native.require_cuda("int4.linear", dy2, w.codes, w.scales)
    rows, k = dy2.shape[0], w.in_features
    dx = dy2.new_empty((rows, k))
    if rows == 0:
        return dx
    with native.on_device(index):
        st = native.entry("st_int4_linear_grad", "ppppiiiqqiip")(dy2.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), dx.data_ptr(), rows, w.out_features, k,
                                                               dy2.stride(0), k, w.group, _TYPES[dy2.dtype], native.raw_stream(index))
    if st:
        native.check(st, "st_int4_linear_grad")
    launch_count += 1
    return dx


def _version(w: Weights) -> tuple:
    return w.codes._version, w.scales._version


def _check_version(w: Weights, version: tuple) -> None:
    if _version(w) != version:
        raise RuntimeError("int4.linear: weights needed for a gradient have been modified by an inplace operation: they were quantised anew")


class _InputGradientFn(torch.autograd.Function):
    """``dy W`` where a graph of the gradient is asked for: linear in ``dy`` as the product is in ``x``."""

    @staticmethod
    def forward(ctx, dy2, w):
        ctx.w, ctx.version = w, _version(w)
        return _input_gradient(dy2, w)

    @staticmethod
    def backward(ctx, d):
        _check_version(ctx.w, ctx.version)
        return linear(d, ctx.w), None


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, residual, w):
        ctx.w, ctx.version = w, _version(w)
        if x.dim() == 2:
            return _product(x, w, bias, None, residual)
        y = _product(x.reshape(-1, x.shape[-1]), w, bias, None, None if residual is None else residual.reshape(-1, w.out_features))
        return y.view(*x.shape[:-1], w.out_features)

    @staticmethod
    def backward(ctx, dy):
        need_x, need_bias, need_residual, _ = ctx.needs_input_grad
        w, dx, db = ctx.w, None, None
        _check_version(w, ctx.version)
        dy2 = dy if dy.dim() == 2 else dy.reshape(-1, w.out_features)
        if need_x:
            dx = _InputGradientFn.apply(dy2, w) if torch.is_grad_enabled() and dy.requires_grad else _input_gradient(dy2, w)
            if dy.dim() != 2:
                dx = dx.view(*dy.shape[:-1], w.in_features)
        if need_bias:
            db = dy2.sum(0, dtype=torch.float64 if dy.dtype == torch.float64 else torch.float32).to(dy.dtype)
        return dx, db, dy if need_residual else None, None


def linear(x: torch.Tensor, w: Weights, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x W^T + bias) + residual``: ``x`` ``[..., in]`` in bf16 or fp16 (2^30 rows at most), ``bias`` ``[out]`` and ``residual`` ``[..., out]`` of the same type, ``act`` None, ``"relu"``
    or ``"gelu"`` (tanh form).  Sums are in fp32; the result, in ``x``'s type, is rounded once.

    Differentiable in ``x``, ``bias`` and ``residual`` (the weights are constants) without ``act``: apply an activation to the result where gradients are needed."""
    if act not in _ACTS:
        raise ValueError(f"int4.linear: act must be None, 'relu' or 'gelu', got {act!r}")
    dtype, shape = x.dtype, x.shape
    if dtype is not torch.bfloat16 and dtype is not torch.float16 and (x.is_cuda or dtype not in (torch.float32, torch.float64)):
        raise ValueError(f"int4.linear: bf16 and fp16 tensors, got {dtype}")
    n = w.out_features
    if len(shape) == 0 or shape[-1] != w.in_features:
        raise ValueError(f"int4.linear: x {tuple(shape)} does not end in the weights' {w.in_features} inputs")
    if x.numel() > w.in_features << 30:
        raise ValueError(f"int4.linear: at most 2^30 rows, got x {tuple(shape)}")
    if bias is not None and (bias.shape != (n,) or bias.dtype is not dtype):
        raise ValueError(f"int4.linear: bias must be {dtype} {(n,)}, got {bias.dtype} {tuple(bias.shape)}")
    if residual is not None and (residual.shape != (*shape[:-1], n) or residual.dtype is not dtype):
        raise ValueError(f"int4.linear: residual must be {dtype} {(*shape[:-1], n)}, got {residual.dtype} {tuple(residual.shape)}")
    if not x.is_cuda:
        native.same_device("int4.linear", x, w.codes, bias, residual)
    if native.has_tangent(x, bias, residual):
        raise ValueError("int4.linear: forward-mode differentiation is not supported")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad)):
        if act is not None:
            raise ValueError("int4.linear: act with tensors that require gradients; apply it to the result")
        if w.codes.is_inference() or w.scales.is_inference():
            raise ValueError("int4.linear: tensors that require gradients by weights whose memory was made in inference mode")
        return _LinearFn.apply(x, bias, residual, w)
    if len(shape) == 2:
        return _product(x, w, bias, act, residual)
    y = _product(x.reshape(-1, w.in_features), w, bias, act, None if residual is None else residual.reshape(-1, n))
    return y.view(*shape[:-1], n)
