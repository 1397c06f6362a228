"""Scores of given tokens (``csrc/elementwise/scores.cu``): their log probabilities, the entropy of the distributions that they were taken from, and the
likeliest tokens beside them, in one pass over the logits; differentiable.

``loss.cross_entropy`` remains the mean loss of training, which writes the gradient over its logits and works on shards of a vocabulary.

Reference parity: none (its losses take probabilities and give one number)."""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import native

launch_count = 0
MOST_TOP = 32
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# StTokenScoresArgs of csrc/elementwise/scores.cu, in one call: a ctypes object for each of a dozen arguments costs as much as the launch
_pack_args = struct.Struct("@7P2q3i").pack
_pack_grad = struct.Struct("@9P3q3i").pack      # StTokenScoresGradArgs


class TokenScores(NamedTuple):
    """``logprob``, ``entropy`` (natural logarithms) fp32 ``[...]``; ``top_ids`` int64 and ``top_logprobs`` fp32 ``[..., top]``, the likeliest first."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def _ordered(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers in the order of the values, NaN last."""
    wide = x.dtype == torch.float64
    b = (x + 0.0).view(torch.int64 if wide else torch.int32).long()
    b = torch.where(b < 0, (b & (0x7FFFFFFFFFFFFFFF if wide else 0x7FFFFFFF)).neg(), b)
    return torch.where(x.isnan(), torch.iinfo(torch.int64).max, b)


def _statement(x: torch.Tensor):
    """``(log probabilities, entropy)`` of rows: all -inf is an empty row, without probability anywhere."""
    m = x.amax(1, keepdim=True)
    empty = m == float("-inf")
    d = x - torch.where(empty, 0.0, m)
    total = d.exp().sum(1, keepdim=True)
    logp = torch.where(empty, x, d - total.log())
    p = logp.exp()
    entropy = torch.where(p == 0, 0.0, -p * logp).sum(1)
    return logp, entropy


def token_scores_reference(logits: torch.Tensor, targets: torch.Tensor, top: int = 0) -> TokenScores:
    """``[rows, vocab]``, ``[rows]``: in fp32 (fp64 for fp64 logits)."""
    x = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    logp, entropy = _statement(x)
    given = (targets >= 0) & (targets < x.shape[1])
    logprob = torch.where(given, logp.gather(1, torch.where(given, targets, 0)[:, None])[:, 0], 0.0)
    ids = _ordered(x).sort(dim=1, descending=True, stable=True).indices[:, :top]
    return TokenScores(logprob, entropy, ids, logp.gather(1, ids))


def _gradient_reference(logits, targets, ids, g_logprob, g_entropy, g_top):
    x = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    logp, entropy = _statement(x)
    p = logp.exp()
    given = (targets >= 0) & (targets < x.shape[1])
    own = torch.zeros_like(x)
    if g_logprob is not None:
        own.scatter_add_(1, torch.where(given, targets, 0)[:, None], torch.where(given, g_logprob, 0.0)[:, None].to(x.dtype))
    if g_top is not None:
        own.scatter_add_(1, ids, g_top.to(x.dtype))
    g = own - p * own.sum(1, keepdim=True)
    if g_entropy is not None:
        g = g - g_entropy[:, None].to(x.dtype) * torch.where(p == 0, 0.0, p * (logp + entropy[:, None]))
    empty = x.amax(1, keepdim=True) == float("-inf")
    return torch.where(empty, 0.0, g).to(logits.dtype)


def _forward(logits, targets, top, keep):
    """Scores of ``[rows, vocab]`` and, where ``keep``, what the gradient needs."""
    global launch_count
    if not logits.is_cuda:
        return token_scores_reference(logits, targets, top), None
    rows, vocab = logits.shape
    index = native.require_cuda("token_scores", logits, targets)
    ids = targets.new_empty((rows, top))
    logprob = torch.empty_like(targets, dtype=torch.float32)
    entropy, top_logprobs = torch.empty_like(logprob), logprob.new_empty((rows, top))
    stats = logprob.new_empty((rows, 2)) if keep else None
    if rows == 0:
        return TokenScores(logprob, entropy, ids, top_logprobs), stats
    args = _pack_args(logits.data_ptr(), targets.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), native.address(stats), ids.data_ptr(), top_logprobs.data_ptr(), rows,
                      logits.stride(0), vocab, top, _TYPES[logits.dtype])
    with native.on_device(index):
        st = native.entry("st_token_scores", "sp")(args, native.raw_stream(index))
    if st:
        native.check(st, "st_token_scores")
    launch_count += 1
    return TokenScores(logprob, entropy, ids, top_logprobs), stats


def _gradient(logits, targets, stats, entropy, ids, g_logprob, g_entropy, g_top):
    global launch_count
    if not logits.is_cuda:
        return _gradient_reference(logits, targets, ids, g_logprob, g_entropy, g_top)
    rows, vocab = logits.shape
    gl, ge, gt = (g if g is None or (g.dtype is torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous() for g in (g_logprob, g_entropy, g_top))
    # rows as far apart as the logits' where that is not much more than they hold: both are then at the same place between 16-byte boundaries
    stride = logits.stride(0)
    room = stride if vocab <= stride <= vocab + vocab // 8 else vocab
    out = logits.new_empty((rows, room))
    if room != vocab:
        out = out[:, :vocab]
    if rows == 0:
        return out
    index = native.require_cuda("token_scores", logits, targets, gl, ge, gt)
    args = _pack_grad(logits.data_ptr(), targets.data_ptr(), stats.data_ptr(), entropy.data_ptr(), ids.data_ptr(), native.address(gl), native.address(ge),
                      native.address(gt), out.data_ptr(), rows, stride, room, vocab, 0 if gt is None else ids.shape[1], _TYPES[logits.dtype])
    with native.on_device(index):
        st = native.entry("st_token_scores_grad", "sp")(args, native.raw_stream(index))
    if st:
        native.check(st, "st_token_scores_grad")
    launch_count += 1
    return out


class _GradientFn(torch.autograd.Function):
    """The gradient where a graph of it is asked for: there is none."""

    @staticmethod
    def forward(ctx, *args):
        return _gradient(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("token_scores: not differentiable twice")


class _TokenScoresFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top):
        scores, stats = _forward(logits, targets, top, True)
        ctx.save_for_backward(logits, targets, stats, scores.entropy, scores.top_ids)
        ctx.mark_non_differentiable(scores.top_ids)
        ctx.set_materialize_grads(False)
        return scores.logprob, scores.entropy, scores.top_ids, scores.top_logprobs

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, _, g_top):
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None
        f = _GradientFn.apply if torch.is_grad_enabled() else _gradient
        return f(*ctx.saved_tensors, g_logprob, g_entropy, g_top), None, None


def token_scores(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0) -> TokenScores:
    """``logits`` ``[..., vocab]`` in bf16, fp16 or fp32 (rows may be strided), ``targets`` int64 ``[...]``; ``top``: how many of the likeliest tokens
    come with them, up to 32 and the vocabulary; of equal ones the lower id first.

    A target outside the vocabulary (``loss.IGNORE_INDEX``) has log probability 0 and no gradient.  ``-inf`` is a token without probability; a row of
    nothing else has entropy 0, log probabilities of -inf and no gradient.  A row with a NaN or ``+inf`` has NaN for all of its scores.

    Differentiable in ``logits`` through ``logprob``, ``entropy`` and ``top_logprobs``; the logits must not change before that."""
    on_cuda, shape = logits.is_cuda, targets.shape
    if logits.dtype not in _TYPES and not (logits.dtype == torch.float64 and not on_cuda):
        raise ValueError(f"token_scores: bf16, fp16 or fp32 logits, got {logits.dtype}")
    if logits.dim() < 1 or shape != logits.shape[:-1] or targets.dtype is not torch.int64:
        raise ValueError(f"token_scores: targets must be int64 {tuple(logits.shape[:-1])}, got {targets.dtype} {tuple(shape)}")
    vocab = logits.shape[-1]
    if not 1 <= vocab <= 1 << 30:
        raise ValueError(f"token_scores: a vocabulary of {vocab}")
    if not 0 <= top <= min(MOST_TOP, vocab):
        raise ValueError(f"token_scores: top must be 0 to {min(MOST_TOP, vocab)}, got {top}")
    if not on_cuda:
        native.same_device("token_scores", logits, targets)
    if native.has_tangent(logits):
        raise ValueError("token_scores: forward-mode differentiation is not supported")
    flat = len(shape) == 1
    rows = logits if flat else logits.reshape(-1, vocab)
    if not flat:
        targets = targets.reshape(-1)
    if not targets.is_contiguous():
        targets = targets.contiguous()
    if vocab > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        scores = _TokenScoresFn.apply(rows, targets, top)
    else:
        scores = _forward(rows, targets, top, False)[0]
    if flat:
        return scores if type(scores) is TokenScores else TokenScores(*scores)
    return TokenScores(scores[0].view(shape), scores[1].view(shape), scores[2].view(*shape, top), scores[3].view(*shape, top))
