"""Performance cases of the operators that answer from an 8-bit paged key/value cache: rotary positions, block tables and
slot maps, storing and reading the cache, and attention over it.

A cache page holds ``page`` tokens of one sequence: codes ``[pages, kv_heads, page, dim]`` in e4m3 and a scale
``[pages, kv_heads]`` in fp32 that is a power of two, for keys and for values.  ``kind`` selects the operator.  Where ``own`` is
false ``run`` computes the operator from elementary torch operations in 32 bits; where it is true it makes the framework's calls.
``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 448.0          # of e4m3
EXPONENTS = (-60, 60)    # of a page's scale


def listed():
    return [
        # the queries and keys of a training step of the 1.3B model, 8 sequences of 2048, with their gradients
        {"name": "rotary_train", "kind": "rotary", "rows": 16384, "heads": 16, "kv_heads": 16, "dim": 128, "rot": 128,
         "interleaved": False, "scaling": "none", "span": 2048, "type": "bf16", "backward": True},
        # one decoding step of 64 sequences far into a long context, frequencies scaled by bands
        {"name": "rotary_decode", "kind": "rotary", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "scaling": "bands", "span": 131072, "type": "fp16", "backward": False},
        # half of each head rotated in interleaved pairs, an odd number of packed rows, fp32, with gradients
        {"name": "rotary_partial", "kind": "rotary", "rows": 3001, "heads": 12, "kv_heads": 12, "dim": 64, "rot": 32,
         "interleaved": True, "scaling": "linear", "span": 8192, "type": "fp32", "backward": True},
        # one more token for each of 256 running sequences
        {"name": "blocks_decode", "kind": "blocks", "seqs": 256, "most": 1, "held": 8000, "page": 64},
        # many prompts admitted at once, some sequences waiting
        {"name": "blocks_prompts", "kind": "blocks", "seqs": 1500, "most": 2000, "held": 3000, "page": 16},
        # one token of each of 96 sequences stored, and the pages it went to read back
        {"name": "store_decode", "kind": "store", "seqs": 96, "most": 1, "held": 5000, "kv_heads": 8, "dim": 128, "page": 64,
         "type": "bf16"},
        # prompts of the 1.3B model stored and read back for attention among themselves
        {"name": "store_prompts", "kind": "store", "seqs": 7, "most": 4096, "held": 0, "kv_heads": 16, "dim": 128, "page": 16,
         "type": "bf16"},
        # the next token of one short prompt with the 1.3B model
        {"name": "attend_one", "kind": "attend", "seqs": 1, "most": 1, "length": 777, "heads": 16, "kv_heads": 16, "dim": 128,
         "page": 64, "type": "bf16", "causal": True},
        # the next token of 64 sequences of mixed lengths, four query heads to a key head
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "most": 1, "length": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "type": "bf16", "causal": True},
        # the next token of two very long contexts, eight query heads to a key head
        {"name": "attend_long", "kind": "attend", "seqs": 2, "most": 1, "length": 131001, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 128, "type": "bf16", "causal": True},
        # up to five drafted tokens of 12 sequences checked at once with the byte-level model's heads
        {"name": "attend_draft", "kind": "attend", "seqs": 12, "most": 5, "length": 2049, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 16, "type": "fp16", "causal": True},
        # a prompt's next part of 256 tokens behind what the cache holds, for four sequences
        {"name": "attend_chunk", "kind": "attend", "seqs": 4, "most": 256, "length": 4000, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "type": "bf16", "causal": True},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "blocks", "store", "attend", "attend"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 16])
    if kind == "rotary":
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        inter = rng.random() < 0.5
        return {"kind": kind, "rows": _log(rng, 1, 262144 // max(heads, 8)), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4, dim - 12]), "interleaved": inter,
                "scaling": rng.choice(["none", "linear", "base", "bands"]), "span": _log(rng, 100, 1000000),
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "backward": rng.random() < 0.5}
    page = rng.choice([16, 32, 64, 128])
    if kind == "blocks":
        seqs = _log(rng, 1, 1500)
        return {"kind": kind, "seqs": seqs, "most": rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 16, 2000)]),
                "held": _log(rng, 1, 8000), "page": page}
    if kind == "store":
        most = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 16, 4096)])
        seqs = _log(rng, 1, min(256, max(1, 16384 // (most * max(1, kv_heads // 4)))))
        return {"kind": kind, "seqs": seqs, "most": most, "held": rng.choice([0, _log(rng, 1, 5000)]), "kv_heads": kv_heads,
                "dim": dim, "page": page, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    most = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 256)])
    length = _log(rng, max(20, most), 131001 if most < 16 else 4000)
    room = 64 * 8192 * 8 * 128 // 2 if most < 16 else 4 * 4000 * 4 * 128
    seqs = _log(rng, 1, max(1, min(128, room // (length * kv_heads * dim))))
    group = rng.choice([1, 2, 3, 4, 7, 8]) if most < 16 else rng.choice([1, 2, 4])
    return {"kind": "attend", "seqs": seqs, "most": most, "length": length, "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": dim, "page": page, "type": rng.choice(["bf16", "bf16", "fp16"]), "causal": most == 1 or rng.random() < 0.8}


# ---- sizes that follow from a case --------------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens held before, tokens added) of each sequence: mixed lengths, the first the longest, now and then one that waits."""
    rng = random.Random("%(kind)s %(seqs)d %(most)d %(page)d" % case)
    held, added = [], []
    for b in range(case["seqs"]):
        n = case["most"] if b == 0 else rng.randint(max(1, case["most"] // 4), case["most"])
        if b and rng.random() < 0.05:
            n = 0
        if case["kind"] == "attend":
            total = case["length"] if b == 0 else _log(rng, max(n, case["length"] // 16, 1), case["length"])
            h = total - n
        else:
            h = 0 if not case["held"] else case["held"] if b == 0 else rng.randint(0, case["held"])
        held.append(h)
        added.append(n)
    return held, added


def _rows(added):
    """Rows of the step's tensors: its tokens, and a few rows behind the last sequence, as a padded step has them."""
    return -(-(sum(added) + 3) // 8) * 8


def _blocks(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["kind"] == "rotary":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * (2.0 * n * TYPES[case["type"]].itemsize + 4 * case["rows"]), "flops": 3.0 * passes * n}
    held, added = _lengths(case)
    P = case["page"]
    fresh = sum(_blocks(h + n, P) - _blocks(h, P) for h, n in zip(held, added))
    if case["kind"] == "blocks":
        # lengths, added and starts; positions and slots of every row; a page's number from the list to the table
        return {"bytes": 16.0 * len(held) + 12.0 * _rows(added) + 8.0 * fresh, "flops": 1.0 * _rows(added)}
    if case["kind"] == "store":
        el = sum(added) * case["kv_heads"] * case["dim"]
        back = sum(_read_length(h, n, case) for h, n in zip(held, added)) * case["kv_heads"] * case["dim"]
        room = len(held) * _read_room(case) * case["kv_heads"] * case["dim"]
        return {"bytes": 2.0 * el * (TYPES[case["type"]].itemsize + 1) + 2.0 * back + 4.0 * room, "flops": 4.0 * el}
    pairs = 0
    for h, n in zip(held, added):
        pairs += n * h + n * (n + 1) // 2 if case["causal"] else n * (h + n)
    kept = sum(h + n for h, n in zip(held, added) if n)
    pages = sum(_blocks(h + n, P) for h, n in zip(held, added) if n)
    return {"bytes": 2.0 * kept * case["kv_heads"] * case["dim"] + pages * (4 + 8.0 * case["kv_heads"])
            + 4.0 * sum(added) * case["heads"] * case["dim"], "flops": 4.0 * pairs * case["heads"] * case["dim"]}


def _read_room(case):
    """Tokens of each sequence that a store case reads back: the whole prompts, or the one page that a step wrote to."""
    return case["most"] if _whole(case) else case["page"]


def _whole(case):
    return case["held"] == 0


def _read_length(held, added, case):
    if _whole(case):
        return held + added
    return (held + added - 1) % case["page"] + 1 if held + added else 0


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Angle per position of each rotated pair, fp64: base 10000, as it is or scaled for contexts longer than trained for."""
    rot, factor, trained = case["rot"], 8.0, 4096.0
    base = 10000.0 * (factor ** (rot / (rot - 2)) if case["scaling"] == "base" and rot > 2 else 1.0)
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "bands":       # few turns over the trained length: slowed down, many: kept, a ramp between 1 and 32 turns
        keep = ((trained * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f.to(DEV)


def _table(held, case, gen, free_too):
    """Block table with the pages of what is held (and, without a free list, of what is added), -1 elsewhere; the free pages."""
    P, added = case["page"], _lengths(case)[1]
    need = [_blocks(h + n, P) for h, n in zip(held, added)]
    have = [_blocks(h, P) for h in held] if free_too else need
    pages = sum(need) + 5
    order = torch.randperm(pages, generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
    width = max(1, max(need))
    cols = torch.arange(width, device=DEV)
    filled = cols[None, :] < torch.tensor(have, device=DEV)[:, None]
    table = torch.full((len(held), width), -1, dtype=torch.int32, device=DEV)
    table[filled] = order[:sum(have)]
    return table, order[sum(have):].contiguous(), pages


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(case, pages, gen):
    """Codes and scales as a model leaves them: normal values whose size differs between pages and heads."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = []
    for _ in range(2):
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV)
        for i in range(0, pages, 1024):      # in parts: the normal values take four times the room
            part = torch.randn((min(1024, pages - i),) + shape[1:], generator=gen, device=DEV)
            codes[i:i + 1024] = (part * 100.0).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
        out.append(codes)
    for _ in range(2):
        out.append(torch.exp2(torch.randint(-8, -5, shape[:2], generator=gen, device=DEV).float()))
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "rotary":
        t = TYPES[case["type"]]
        shape = lambda h: (case["rows"], h, case["dim"])                                              # noqa: E731
        s = {"case": case, "freq": _frequencies(case),
             "positions": torch.randint(0, case["span"], (case["rows"],), generator=gen, device=DEV, dtype=torch.int32)}
        for name, h in (("q", case["heads"]), ("k", case["kv_heads"]), ("dq", case["heads"]), ("dk", case["kv_heads"])):
            s[name] = torch.randn(shape(h), generator=gen, device=DEV).to(t)
        if case["backward"]:
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        return s
    held, added = _lengths(case)
    rows, total = _rows(added), [h + n for h, n in zip(held, added)]
    table, free, pages = _table(held, case, gen, case["kind"] == "blocks")
    s = {"case": case, "table": table, "held": _i32(held), "added": _i32(added), "lengths": _i32(total), "rows": rows,
         "starts": torch.cat([_i32([0]), _i32(added).cumsum(0, dtype=torch.int32)])}
    if case["kind"] == "blocks":
        s["free"], s["free_count"] = free, _i32([free.numel()])
        return s
    s["cache"] = _cache(case, pages, gen)
    t = TYPES[case["type"]]
    seq, pos = _plain_rows(s["starts"], s["held"], rows)
    if case["kind"] == "store":
        page = table[seq.clamp(min=0), pos // case["page"]].long()
        s["slots"] = torch.where(seq < 0, -1, page * case["page"] + pos % case["page"])
        shape = (rows, case["kv_heads"], case["dim"])
        s["k"], s["v"] = ((torch.randn(shape, generator=gen, device=DEV) * 1.5).to(t) for _ in range(2))
        if _whole(case):
            s["read_table"], s["read_lengths"] = table, s["lengths"]
        else:
            last = ((s["lengths"] - 1) // case["page"]).clamp(min=0).long()
            s["read_table"] = table.gather(1, last[:, None]).contiguous()
            s["read_lengths"] = _i32([_read_length(h, n, case) for h, n in zip(held, added)])
        return s
    # what lies in a page behind its sequence's end is whatever was there: codes that are no number
    blocks = torch.arange(table.shape[1], device=DEV)[:, None] * case["page"] + torch.arange(case["page"], device=DEV)
    b, i, o = (blocks[None] >= s["lengths"][:, None, None]).logical_and(table[:, :, None] >= 0).nonzero(as_tuple=True)
    for codes in s["cache"][:2]:
        codes.view(torch.uint8)[table[b, i].long(), :, o] = 0x7F
    s["q"] = torch.randn((rows, case["heads"], case["dim"]), generator=gen, device=DEV).to(t)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------------
def _plain_rows(starts, held, rows):
    """Sequence (-1 behind the last one) and position of every row."""
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:].long(), r, right=True)
    inside = seq < held.numel()
    at = seq.clamp(max=held.numel() - 1)
    pos = r - starts.long()[at] + held.long()[at]
    return torch.where(inside, seq, -1), torch.where(inside, pos, 0)


def _plain_rotate(x, positions, freq, interleaved, sign):
    angle = positions.double()[:, None] * freq
    c, s = angle.cos().float()[:, None, :], (angle.sin() * sign).float()[:, None, :]
    n, xf = freq.numel(), x.float()
    a, b = (xf[..., 0:2 * n:2], xf[..., 1:2 * n:2]) if interleaved else (xf[..., :n], xf[..., n:2 * n])
    ya, yb = a * c - b * s, b * c + a * s
    turned = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([turned, xf[..., 2 * n:]], -1).to(x.dtype)


def _plain_plan(s):
    P, table, held, added = s["case"]["page"], s["table"], s["held"].long(), s["added"].long()
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), added.cumsum(0)])
    have, need = -(-held // P), -(-(held + added) // P)
    before = (need - have).cumsum(0) - (need - have)
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    nth = s["free_count"].long() - 1 - before[:, None] - (col - have[:, None])
    table.copy_(torch.where(fresh, s["free"][nth.clamp(min=0, max=s["free"].numel() - 1)], table))
    seq, pos = _plain_rows(starts, held, s["rows"])
    page = table[seq.clamp(min=0), pos // P].long()
    slots = torch.where(seq < 0, -1, page * P + pos % P)
    return (table, starts.int(), pos.int(), slots, (held + added).int(), (s["free_count"] - (need - have).sum()).int())


def _plain_exponent(amax):
    """The least e with amax <= 448 * 2^e."""
    f, x = torch.frexp(amax)
    e = x - 9 + (f > 0.875).int()
    return torch.where(amax > 0, e, EXPONENTS[0]).clamp(*EXPONENTS)


def _plain_store(s):
    P, slots = s["case"]["page"], s["slots"]
    rows = (slots >= 0).nonzero(as_tuple=True)[0]
    page, off = slots[rows] // P, slots[rows] % P
    touched, group = torch.unique(page, return_inverse=True)
    first = torch.full_like(touched, P).scatter_reduce(0, group, off, "amin")
    for codes, scale, x in ((s["cache"][0], s["cache"][2], s["k"]), (s["cache"][1], s["cache"][3], s["v"])):
        xf = x[rows].float()
        amax = torch.zeros((touched.numel(), xf.shape[1]), device=DEV)
        amax = amax.scatter_reduce(0, group[:, None].expand(-1, xf.shape[1]), xf.abs().amax(-1), "amax")
        old = torch.where((first > 0)[:, None], torch.log2(scale[touched]).round().int(), EXPONENTS[0])
        new = torch.maximum(old, _plain_exponent(amax))
        kept = codes.view(torch.uint8)[touched].view(torch.float8_e4m3fn).float() * torch.exp2((old - new).float())[:, :, None, None]
        codes.view(torch.uint8)[touched] = kept.to(torch.float8_e4m3fn).view(torch.uint8)
        scale[touched] = torch.exp2(new.float())
        value = (xf * torch.exp2(-new.float())[group][:, :, None]).clamp(-LARGEST, LARGEST)
        codes.view(torch.uint8)[page, :, off] = value.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_dense(codes, scale, table):
    """fp32 ``[seqs, blocks * page, kv_heads, dim]`` of the pages that a table names."""
    at = table.clamp(min=0).long()
    x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None, None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_read(s):
    room, out = _read_room(s["case"]), []
    inside = torch.arange(room, device=DEV)[None, :] < s["read_lengths"][:, None]
    for codes, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1], s["cache"][3])):
        x = _plain_dense(codes, scale, s["read_table"])[:, :room]
        out.append(torch.where(inside[:, :, None, None], x, 0.0).to(torch.bfloat16))
    return tuple(out)


def _plain_attend(s):
    c, q, most = s["case"], s["q"], s["case"]["most"]
    k, v = (_plain_dense(s["cache"][i], s["cache"][i + 2], s["table"]) for i in (0, 1))       # [B, S, Hk, D]
    B, S, Hk, D = k.shape
    lengths, added, starts = s["lengths"].long(), s["added"].long(), s["starts"].long()
    i = torch.arange(most, device=DEV)
    row = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)                                     # [B, n]
    qs = q[row].float().view(B, most, Hk, -1, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)   # [B, Hk, G * n, D]
    key = torch.arange(S, device=DEV)
    last = (lengths - added)[:, None] + i + 1 if c["causal"] else lengths[:, None].expand(B, most)
    seen = (key[None, None] < last[..., None]) & (key < lengths[:, None, None])                 # [B, n, S]
    scores = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(B, Hk, -1, most, S) / math.sqrt(D)
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = torch.where((key < lengths[:, None])[:, :, None, None], v, 0.0)
    o = torch.matmul(p.flatten(2, 3), v.transpose(1, 2)).view(B, Hk, -1, most, D).permute(0, 3, 1, 2, 4).reshape(B, most, -1, D)
    seq, pos = _plain_rows(s["starts"], lengths - added, q.shape[0])
    at = seq.clamp(min=0)
    o = o[at, (pos - (lengths - added)[at]).clamp(min=0, max=most - 1)]
    return torch.where((seq < 0)[:, None, None], 0.0, o).to(q.dtype)


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from spiraltorch_b200.ops import paged, rotary
        if c["kind"] == "rotary":
            q, k = rotary.rotary(s["q"], s["k"], s["positions"], s["freq"], interleaved=c["interleaved"])
            if not c["backward"]:
                return q, k
            return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        if c["kind"] == "blocks":
            step = paged.plan(s["held"], s["added"], s["table"], s["free"], s["free_count"], page_size=c["page"], rows=s["rows"])
            return s["table"], step.starts, step.positions, step.slots, step.lengths, step.free_count
        pages = paged.Pages(*s["cache"])
        if c["kind"] == "store":
            paged.store(s["k"], s["v"], pages, s["slots"])
            return paged.read(pages, s["read_table"], s["read_lengths"], _read_room(c))
        return paged.attention(s["q"], pages, s["table"], s["starts"], s["lengths"], max_queries=c["most"], causal=c["causal"])
    with torch.no_grad():
        if c["kind"] == "rotary":
            out = [_plain_rotate(s[n], s["positions"], s["freq"], c["interleaved"], 1.0) for n in ("q", "k")]
            if c["backward"]:
                out += [_plain_rotate(s[n], s["positions"], s["freq"], c["interleaved"], -1.0) for n in ("dq", "dk")]
            return tuple(out)
        if c["kind"] == "blocks":
            return _plain_plan(s)
        if c["kind"] == "store":
            _plain_store(s)
            return _plain_read(s)
        return _plain_attend(s)


# ---- 64 bits --------------------------------------------------------------------------------------------------------------------
def _exact_e4m3(x):
    """fp64 values rounded to e4m3: four significant bits down to 2^-6, steps of 2^-9 below, ties to the even one."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return (torch.round(x / step) * step).clamp(-LARGEST, LARGEST)


def _exact_unit(amax):
    """The least power of two that is at least amax / 448, on the host: log2 of a power of two need not be whole on the GPU."""
    return torch.tensor([2.0 ** next(e for e in range(-200, 200) if a <= LARGEST * 2.0 ** e) for a in amax.tolist()],
                        dtype=torch.float64, device=DEV)


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["kind"] == "rotary":
            z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * s["freq"])[:, None]
            n, out = s["freq"].numel(), []
            for name, turn in (("q", z), ("k", z)) + ((("dq", z.conj()), ("dk", z.conj())) if case["backward"] else ()):
                x = s[name].detach().double()
                first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
                w = torch.complex(x[..., first], x[..., second]) * turn
                y = x.clone()
                y[..., first], y[..., second] = w.real, w.imag
                out.append(y)
            return tuple(out)
        if case["kind"] == "blocks":
            return None
        held, added = _lengths(case)
        P, table = case["page"], s["table"].tolist()
        if case["kind"] == "store":
            out = []
            for codes, scale, x in ((s["cache"][0], s["cache"][2], s["k"]), (s["cache"][1], s["cache"][3], s["v"])):
                got = torch.zeros((len(held), _read_room(case)) + tuple(x.shape[1:]), dtype=torch.float64, device=DEV)
                row = 0
                for b, (h, n) in enumerate(zip(held, added)):
                    x64, row = x[row:row + n].double(), row + n
                    for j in range(0 if _whole(case) else max(0, (h + n - 1) // P), _blocks(h + n, P)):
                        lo, hi = max(h, j * P), min(h + n, (j + 1) * P)
                        new, old = x64[max(0, lo - h):max(0, hi - h)], max(0, min(h, (j + 1) * P) - j * P)
                        page = table[b][j]
                        unit = torch.full((x.shape[1],), 2.0 ** EXPONENTS[0], dtype=torch.float64, device=DEV)
                        if new.numel():
                            unit = torch.maximum(unit, _exact_unit(new.abs().amax((0, 2))))
                        if old:
                            unit = torch.maximum(unit, scale[page].double())
                        unit = unit[None, :, None]
                        before = (codes[page, :, :old].double() * scale[page].double()[:, None, None]).transpose(0, 1)
                        vals = torch.cat([before, new])
                        vals = _exact_e4m3(vals / unit) * unit
                        at = 0 if not _whole(case) else j * P
                        got[b, at:at + vals.shape[0]] = vals
                out.append(got)
            return tuple(out)
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        group, row = case["heads"] // case["kv_heads"], 0
        for b, (h, n) in enumerate(zip(held, added)):
            if n == 0:
                continue
            at = torch.tensor(table[b][:_blocks(h + n, P)], device=DEV)
            for kh in range(case["kv_heads"]):
                k, v = ((s["cache"][i][at, kh].double() * s["cache"][i + 2][at, kh].double()[:, None, None]).flatten(0, 1)[:h + n] for i in (0, 1))
                q = s["q"][row:row + n, kh * group:(kh + 1) * group].double()
                t = torch.einsum("igd,sd->gis", q, k) * case["dim"] ** -0.5
                if case["causal"]:
                    t += torch.full((n, h + n), float("-inf"), dtype=torch.float64, device=DEV).triu(h + 1)
                o[row:row + n, kh * group:(kh + 1) * group] = torch.einsum("gis,sd->igd", torch.softmax(t, -1), v)
            row += n
        return o
