"""An 8-bit paged key / value cache and attention over it (``csrc/serving/paged_cache.cu``, ``csrc/serving/paged_attn.cu``).

A page holds the keys and values of ``page`` consecutive tokens of one sequence for all its key heads, as e4m3 codes with one
scale per page and head: the least power of two ``2^e`` with ``amax <= 448 * 2^e``, ``-60 <= e <= 60``.  A step is

    step = plan(lengths, added, table, free, free_count, page_size=..., rows=...)     # pages for the new tokens, and their maps
    q, k = rotary(q, k, step.positions, freq)
    store(k, v, pages, step.slots)
    o = attention(q, pages, table, step.starts, step.lengths, max_queries=...)

with the new tokens of all sequences one after another in the rows of ``q``, ``k`` and ``v``.  All of it runs on the current stream without
a look at the device's values, so a step can be captured into a CUDA graph and replayed while the sequences grow.

CPU tensors use a plain PyTorch statement of the same (also the test oracle).  The reference has no such cache.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch

from . import native

launch_count = 0
LARGEST = 448.0                 # of e4m3
MIN_EXPONENT, MAX_EXPONENT = -60, 60
PAGE_SIZES = (16, 32, 64, 128, 256)
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class Pages(NamedTuple):
    """``k``, ``v``: e4m3 codes ``[pages, kv_heads, page, dim]`` (dim 64 or 128); ``k_scale``, ``v_scale``: fp32 ``[pages, kv_heads]``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, dim: int, device="cuda") -> "Pages":
        """Room for ``pages * page_size`` tokens; a page is written before it is read, so nothing is cleared."""
        if page_size not in PAGE_SIZES:
            raise ValueError(f"paged: page size must be one of {PAGE_SIZES}, got {page_size}")
        if dim not in (64, 128):
            raise ValueError(f"paged: head dimension must be 64 or 128, got {dim}")
        if pages < 0 or kv_heads < 1:
            raise ValueError(f"paged: {pages} pages of {kv_heads} heads")
        shape = (pages, kv_heads, page_size, dim)
        codes = [torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        return cls(*codes, *(torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))


class Step(NamedTuple):
    """What one step's operators read.  ``starts`` int32 ``[B + 1]``: first row of every sequence; ``positions`` int32 and ``slots`` int64
    ``[rows]``: place in the sequence and in the cache (``page * page_size + offset``), 0 and -1 behind the last sequence; ``lengths`` int32 ``[B]`` and
    ``free_count`` int32 ``[1]``: as they are after the step.  A ``free_count`` below 0 says how many pages were missing: their tokens have
    slot -1 and are not stored."""
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    lengths: torch.Tensor
    free_count: torch.Tensor


def _ints(name: str, t: torch.Tensor, dim: int, dtype=torch.int32) -> None:
    if t.dtype is not dtype or t.dim() != dim or (t.stride()[-1] != 1 and t.numel() > 0):
        raise ValueError(f"paged: {name} must be {dtype} with {dim} dimension{'s' if dim > 1 else ''} and contiguous, got {t.dtype} {tuple(t.shape)}")


def _check_pages(p: Pages) -> tuple:
    k, v, ks, vs = p
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError(f"paged: codes {tuple(shape)}, {tuple(v.shape)} and scales {tuple(ks.shape)}, {tuple(vs.shape)} do not belong together")
    if k.dtype is not torch.float8_e4m3fn or v.dtype is not torch.float8_e4m3fn or ks.dtype is not torch.float32 or vs.dtype is not torch.float32:
        raise ValueError("paged: codes must be float8_e4m3fn and scales float32")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("paged: codes and scales must be contiguous")
    if shape[2] not in PAGE_SIZES or shape[3] not in (64, 128) or shape[1] < 1:
        raise ValueError(f"paged: pages of {shape[2]} tokens and heads of {shape[3]} are not supported (sizes {PAGE_SIZES}, 64 or 128)")
    return shape


@functools.cache
def _max_sequences() -> int:
    return native.lib().st_paged_max_sequences()


# ---- block tables and slot maps -------------------------------------------------------------------------------------------------
def plan(lengths: torch.Tensor, added: torch.Tensor, table: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, *, page_size: int,
         rows: int) -> Step:
    """Pages for ``added`` more tokens of every sequence and the maps of the step.

    ``lengths``, ``added`` int32 ``[B]`` (B up to 8192; negative ones count as 0), ``table`` int32 ``[B, width]``: new pages are taken from the end of
    ``free[:free_count]`` in the order of sequences and blocks and written to it.  Nothing else is changed: ``lengths`` and ``free_count`` after the step
    are in the result, and the step takes effect when the caller goes on with those.  ``rows``: rows of the step's tensors, at least the
    sum of ``added`` (tokens beyond are not mapped).  Tokens beyond the table's width get slot -1.  Totals stay below 2^31."""
    global launch_count
    if page_size not in PAGE_SIZES:
        raise ValueError(f"paged: page size must be one of {PAGE_SIZES}, got {page_size}")
    _ints("lengths", lengths, 1)
    _ints("added", added, 1)
    _ints("table", table, 2)
    _ints("free", free, 1)
    _ints("free_count", free_count, 1)
    B, width = table.shape
    if lengths.shape[0] != B or added.shape[0] != B or free_count.shape[0] != 1 or rows < 0:
        raise ValueError(f"paged: lengths {tuple(lengths.shape)}, added {tuple(added.shape)}, table {tuple(table.shape)}, "
                         f"free_count {tuple(free_count.shape)} and {rows} rows do not belong together")
    if not native.use_native(lengths):
        return _plan_reference(lengths, added, table, free, free_count, page_size, rows)
    index = native.require_cuda("paged.plan", lengths, added, table, free, free_count)
    if B > _max_sequences():
        raise ValueError(f"paged.plan: {B} sequences, at most {_max_sequences()}")
    # one allocation for the 32-bit results: five of them take as long as the launch twice
    positions, starts, after, left = free_count.new_empty(rows + 2 * B + 2).split_with_sizes((rows, B + 1, B, 1))
    step = Step(starts, positions, free_count.new_empty(rows, dtype=torch.int64), after, left)
    with native.on_device(index):
        st = native.entry("st_paged_plan", "pppqippiiiqpppppp")(
            lengths.data_ptr(), added.data_ptr(), table.data_ptr(), table.stride(0), width, free.data_ptr(), free_count.data_ptr(), free.shape[0],
            page_size, B, rows, *(t.data_ptr() for t in step), native.raw_stream(index))
    native.check(st, "st_paged_plan")
    launch_count += 1
    return step


def _plan_reference(lengths, added, table, free, free_count, page_size, rows) -> Step:
    B, width = table.shape
    count = left = min(int(free_count), free.shape[0])
    starts, positions, slots, after = [0], [], [], []
    for b in range(B):
        have, n = max(int(lengths[b]), 0), max(int(added[b]), 0)
        for block in range(min(-(-have // page_size), width), min(-(-(have + n) // page_size), width)):
            left -= 1
            table[b, block] = free[left] if left >= 0 else -1
        for pos in range(have, have + n):
            page = int(table[b, pos // page_size]) if pos // page_size < width else -1
            positions.append(pos)
            slots.append(page * page_size + pos % page_size if page >= 0 else -1)
        starts.append(starts[-1] + n)
        after.append(have + n)
    pad = max(0, rows - len(positions))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                                           # noqa: E731
    return Step(i32(starts), i32((positions + [0] * pad)[:rows]), torch.tensor((slots + [-1] * pad)[:rows], dtype=torch.int64), i32(after), i32([left]))


def release(lengths: torch.Tensor, done: torch.Tensor, table: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, *, page_size: int) -> None:
    """Pages of the sequences with ``done`` (bool ``[B]``) back to the end of ``free``, in the order of sequences and blocks; their ``lengths`` become 0,
    their table entries -1, ``free_count`` grows.  All in place."""
    global launch_count
    if page_size not in PAGE_SIZES:
        raise ValueError(f"paged: page size must be one of {PAGE_SIZES}, got {page_size}")
    for n, t, d in (("lengths", lengths, 1), ("table", table, 2), ("free", free, 1), ("free_count", free_count, 1)):
        _ints(n, t, d)
    _ints("done", done, 1, torch.bool)
    B, width = table.shape
    if lengths.shape[0] != B or done.shape[0] != B or free_count.shape[0] != 1:
        raise ValueError(f"paged: lengths {tuple(lengths.shape)}, done {tuple(done.shape)}, table {tuple(table.shape)} and free_count "
                         f"{tuple(free_count.shape)} do not belong together")
    if not native.use_native(lengths):
        at = max(int(free_count), 0)
        for b in range(B):
            if done[b]:
                for block in range(min(-(-max(int(lengths[b]), 0) // page_size), width)):
                    if table[b, block] >= 0:
                        free[at] = table[b, block]
                        at += 1
                    table[b, block] = -1
                lengths[b] = 0
        free_count[0] = at
        return
    index = native.require_cuda("paged.release", lengths, done, table, free, free_count)
    if B > _max_sequences():
        raise ValueError(f"paged.release: {B} sequences, at most {_max_sequences()}")
    with native.on_device(index):
        st = native.entry("st_paged_release", "pppqippiiip")(lengths.data_ptr(), done.data_ptr(), table.data_ptr(), table.stride(0), width, free.data_ptr(),
                                                             free_count.data_ptr(), free.shape[0], page_size, B, native.raw_stream(index))
    native.check(st, "st_paged_release")
    launch_count += 1


# ---- storing and reading --------------------------------------------------------------------------------------------------------
def store(k: torch.Tensor, v: torch.Tensor, pages: Pages, slots: torch.Tensor) -> None:
    """Rows ``k``, ``v`` ``[rows, kv_heads, dim]`` (bf16, fp16 or fp32; dim contiguous, any other strides) into the cache, in place.

    ``slots`` int64 ``[rows]``, from :func:`plan`; below 0: not stored.  Tokens of one page follow one another in the rows, each slot once; a
    page belongs to one sequence.  A group of rows that starts at offset 0 begins its page anew, one behind that keeps the tokens before
    it: where the scale has to grow, their codes are rounded again.  Finite magnitudes above ``448 * 2^60`` and infinities are
    stored as the largest value of the page, NaN as NaN.  Not differentiable: the values alone are stored."""
    global launch_count
    P, H, page, D = _check_pages(pages)
    if k.shape != v.shape or k.dim() != 3 or k.shape[1:] != (H, D) or k.dtype != v.dtype:
        raise ValueError(f"paged.store: k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} do not match pages of {H} heads of {D}")
    if k.dtype not in _TYPES:
        raise ValueError(f"paged.store: bf16, fp16 and fp32 rows, got {k.dtype}")
    if k.stride()[2] != 1 or v.stride()[2] != 1:
        raise ValueError("paged.store: head elements must be contiguous")
    _ints("slots", slots, 1, torch.int64)
    if slots.shape[0] != k.shape[0]:
        raise ValueError(f"paged.store: {slots.shape[0]} slots for {k.shape[0]} rows")
    if not native.use_native(k):
        return _store_reference(k, v, pages, slots)
    index = native.require_cuda("paged.store", k, v, *pages, slots)
    with native.on_device(index):
        st = native.entry("st_paged_store", "pppppppqiiiqqqqqip")(
            k.data_ptr(), v.data_ptr(), pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), slots.data_ptr(),
            k.shape[0], H, D, page, P, *k.stride()[:2], *v.stride()[:2], _TYPES[k.dtype], native.raw_stream(index))
    native.check(st, "st_paged_store")
    launch_count += 1


def page_exponent(amax: torch.Tensor) -> torch.Tensor:
    """The least ``e`` with ``amax <= 448 * 2^e``, kept to the range of scales (int32)."""
    f, x = torch.frexp(amax.float())
    e = x - 9 + (f > 0.875).int()
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT)).clamp(MIN_EXPONENT, MAX_EXPONENT)


def to_codes(x: torch.Tensor) -> torch.Tensor:
    """fp32 values to e4m3 codes: nearest, ties to even, larger magnitudes to the largest, NaN kept."""
    return x.clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)


@torch.no_grad()
def _store_reference(k, v, pages, slots) -> None:
    P, H, page, D = pages.k.shape
    at, rows = slots.tolist(), len(slots)
    if any(s >= P * page for s in at):
        raise ValueError("paged.store: a slot lies behind the last page")
    seen = set()
    r = 0
    while r < rows:
        n = 1
        if at[r] < 0:
            r += 1
            continue
        while r + n < rows and at[r + n] == at[r] + n and at[r + n] % page:
            n += 1
        p, off = at[r] // page, at[r] % page
        if p in seen:
            raise ValueError(f"paged.store: tokens of page {p} do not follow one another")
        seen.add(p)
        for x, codes, scale in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
            new = x[r:r + n].float().transpose(0, 1)                                # [H, n, D]
            mag = new.abs()
            e = page_exponent(torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag)).amax((1, 2)))
            if off:
                old = torch.log2(scale[p]).round().int().clamp(MIN_EXPONENT, MAX_EXPONENT)
                e = torch.maximum(e, old)
                codes[p, :, :off] = to_codes(codes[p, :, :off].float() * torch.exp2((old - e).float())[:, None, None])
            codes[p, :, off:off + n] = to_codes(new * torch.exp2(-e.float())[:, None, None])
            scale[p] = torch.exp2(e.float())
        r += n


def read(pages: Pages, table: torch.Tensor, lengths: torch.Tensor, max_length: int, dtype: torch.dtype = torch.bfloat16):
    """``(k, v)`` ``[B, max_length, kv_heads, dim]``: what the cache holds of the first ``max_length`` tokens of every sequence (exact, in bf16
    or fp32), zeros at and behind its length; the dense form that ``ops.attention`` takes.  A page number that is none: as in :func:`attention`, and zeros."""
    global launch_count
    P, H, page, D = _check_pages(pages)
    _ints("table", table, 2)
    _ints("lengths", lengths, 1)
    B, width = table.shape
    if lengths.shape[0] != B or max_length < 0:
        raise ValueError(f"paged.read: table {tuple(table.shape)}, lengths {tuple(lengths.shape)}, {max_length} tokens")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"paged.read: bf16 or fp32 (fp16 does not hold every scale), got {dtype}")
    if not native.use_native(pages.k):
        return tuple(_dense_reference(c, s, table, lengths, max_length).to(dtype) for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
    index = native.require_cuda("paged.read", *pages, table, lengths)
    k = pages.k_scale.new_empty((B, max_length, H, D), dtype=dtype)
    v = torch.empty_like(k)
    with native.on_device(index):
        st = native.entry("st_paged_read", "ppppppqiiiiiiqppip")(
            pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            table.stride(0), width, B, max_length, H, D, page, P, k.data_ptr(), v.data_ptr(), int(dtype == torch.float32), native.raw_stream(index))
    native.check(st, "st_paged_read")
    launch_count += 1
    return k, v


def _dense_reference(codes, scale, table, lengths, max_length, dtype=torch.float32) -> torch.Tensor:
    P, H, page, D = codes.shape
    B, width = table.shape
    out = torch.zeros((B, max_length, H, D), dtype=dtype)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), max_length, width * page)
        at = table[b, :-(-n // page)].long()
        if bool(((at < 0) | (at >= P)).any()):
            raise ValueError(f"paged: the table of sequence {b} names a page that is none")
        x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).to(dtype) * scale[at].to(dtype)[:, :, None, None]
        out[b, :n] = x.transpose(1, 2).reshape(-1, H, D)[:n]
    return out


# ---- attention ------------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=1024)
def _workspace(max_queries: int, heads: int, kv_heads: int, dim: int, width: int, page: int, index: int) -> int:
    size = native.entry("st_paged_attention_workspace", "iiiiii")
    size.restype = ctypes.c_longlong
    return size(max_queries, heads, kv_heads, dim, width, page)


def attention(q: torch.Tensor, pages: Pages, table: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, *, max_queries: int, causal: bool = True,
              scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of the newest tokens of every sequence over what the cache holds of it (these tokens included).

    ``q`` ``[rows, heads, dim]`` (bf16 or fp16, on the CPU also fp32; dim contiguous, any other strides), ``heads`` a multiple of the cache's key heads: query head ``h`` reads key head
    ``h // (heads / kv_heads)``.  Rows ``starts[b]`` to ``starts[b + 1]`` belong to sequence ``b``, whose ``lengths[b]`` tokens lie in the pages of ``table[b]``; the last
    row is its newest token, and a row sees the keys up to its own place, or all where not ``causal``.  A row that sees none is 0.
    ``max_queries``: the most rows of one sequence; it decides the kernel's tile, not the result.  With more than 32 rows to a key head (tokens times the heads
    that share it) all sequences get tiles of 128, which a single token leaves empty but for its own: 64 sequences of one token at 4096, 16 heads of 128, 172 us, with a
    part of 256 tokens among them 497, in two calls (parts of ``starts``, ``table``, ``lengths``) 209.  ``scale``: ``1 / sqrt(dim)`` if not given.

    Returns ``o`` like ``q`` (contiguous, or ``out``), with ``return_lse`` also the log-sum-exp of every row's scores, fp32 ``[rows, heads]``.  Rows of no
    sequence, before ``starts[0]`` and behind the last one, are 0 (lse -inf); in a given ``out``, which may be ``q`` itself, they stay as they were.  Softmax
    weights are rounded to fp16, sums and products are fp32.  A page number that is none raises on the CPU; the kernels pass its keys over and leave an error record
    (:func:`native.poll`).  Not differentiable.  Whole causal prompts of 2000 tokens and more run faster over :func:`read` and ``ops.attention``."""
    global launch_count
    P, Hk, page, D = _check_pages(pages)
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] < Hk or q.shape[1] % Hk:
        raise ValueError(f"paged.attention: q {tuple(q.shape)} does not fit pages of {Hk} heads of {D}")
    if not (q.dtype in (torch.bfloat16, torch.float16) or q.dtype == torch.float32 and not q.is_cuda) or q.stride()[2] != 1:
        raise ValueError("paged.attention: q must be bf16 or fp16 (on the CPU also fp32) with contiguous head elements")
    _ints("table", table, 2)
    _ints("starts", starts, 1)
    _ints("lengths", lengths, 1)
    rows, H, _ = q.shape
    B, width = table.shape
    if lengths.shape[0] != B or starts.shape[0] != B + 1:
        raise ValueError(f"paged.attention: table {tuple(table.shape)}, starts {tuple(starts.shape)} and lengths {tuple(lengths.shape)} do not belong together")
    if max_queries < 1 or max_queries * H >= 1 << 31:
        raise ValueError(f"paged.attention: max_queries {max_queries}")
    if not 0 < P * Hk * page < 1 << 31:
        raise ValueError(f"paged.attention: {P} pages of {page} tokens and {Hk} heads")
    if torch.is_grad_enabled() and q.requires_grad or native.has_tangent(q):
        raise ValueError("paged.attention: not differentiable; use ops.attention for training")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1):
        raise ValueError(f"paged.attention: out {tuple(out.shape)} {out.dtype} is not like q")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"paged.attention: scale {scale}")
    if not native.use_native(q):
        o, lse = attention_reference(q, pages, table, starts, lengths, causal, scale)
        o = o.to(q.dtype)
        if out is not None:
            first, end = max(int(starts[0]), 0), min(int(starts[-1]), rows)
            out[first:end] = o[first:end]
            o = out
        return (o, lse.float()) if return_lse else o
    index = native.require_cuda("paged.attention", q, *pages, table, starts, lengths, out)
    o = (torch.empty_like(q) if q.is_contiguous() else q.new_empty((rows, H, D))) if out is None else out
    lse = pages.k_scale.new_empty((rows, H)) if return_lse else None
    with native.on_device(index):
        room = _workspace(max_queries, H, Hk, D, width, page, index)
        work = pages.k_scale.new_empty(room) if room else None
        st = native.entry("st_paged_attention", "pppppppppppqqqqqqqiiiiiiifiiip")(
            q.data_ptr(), pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), table.data_ptr(), starts.data_ptr(),
            lengths.data_ptr(), o.data_ptr(), native.address(lse), native.address(work), *q.stride()[:2], *o.stride()[:2], table.stride(0), P, rows,
            width, page, B, H, Hk, D, max_queries, scale, int(causal), int(out is None), int(q.dtype == torch.float16), native.raw_stream(index))
    native.check(st, "st_paged_attention")
    launch_count += 2 if room else 1
    return (o, lse) if return_lse else o


def attention_reference(q, pages, table, starts, lengths, causal=True, scale=None, dtype=torch.float32):
    """The same in ``dtype``: ``(o [rows, heads, dim], lse [rows, heads])``."""
    P, Hk, page, D = pages.k.shape
    rows, H, _ = q.shape
    G, scale = H // Hk, 1.0 / math.sqrt(D) if scale is None else scale
    o, lse = torch.zeros((rows, H, D), dtype=dtype), torch.full((rows, H), float("-inf"), dtype=dtype)
    for b in range(table.shape[0]):
        r0, r1 = max(int(starts[b]), 0), min(int(starts[b + 1]), rows)
        n, length = r1 - r0, min(max(int(lengths[b]), 0), table.shape[1] * page)
        if n <= 0 or length == 0:
            continue
        k, v = (_dense_reference(c, s, table[b:b + 1], lengths[b:b + 1], length, dtype)[0].repeat_interleave(G, 1)
                for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        for i in range(n):
            seen = min(max(length - (n - 1 - i), 0), length) if causal else length
            if seen:
                s = torch.einsum("hd,shd->hs", q[r0 + i].to(dtype), k[:seen]) * scale
                lse[r0 + i] = torch.logsumexp(s, -1)
                o[r0 + i] = torch.einsum("hs,shd->hd", torch.softmax(s, -1), v[:seen])
    return o, lse
