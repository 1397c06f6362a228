"""Performance cases of the operators that let a language model answer with weights of four bits and judge what it answers: quantising
weights by groups, products with them (and the gradient of their input), and the log probabilities, entropy and likeliest
alternatives of given tokens, with their gradient.

A weight matrix ``[out, in]`` is held as ``q * s``: codes ``-8 <= q <= 7`` and one scale per row and group of ``group`` consecutive
inputs.  The scale is minus an eighth of the group's element of largest magnitude (the negative one of two), rounded to 4
significant bits (ties to even), its magnitude within ``2^-20`` and ``1.875 * 2^12``; the code is the weight over the scale, rounded to the nearest (ties
to even) and clamped.  Every ``q * s`` is a bf16 and an fp16 number.

``kind`` selects the operator.  Where ``own`` is false ``run`` computes it from elementary torch operations in 32 bits; where it is true it makes
the framework's calls.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCALE = (2.0 ** -20, 1.875 * 2.0 ** 12)      # least and largest magnitude of a scale
IGNORED = -100                               # target of a row that is padding
MOST_PRODUCTS = 4096 * 8192 * 2048
MOST_LOGITS = 8192 * 50304


def listed():
    return [
        # one sequence's next token: the projection behind attention in the 1.3B model, added to the residual stream
        {"name": "linear_one", "kind": "linear", "rows": 1, "in": 2048, "out": 2048, "group": 64, "type": "bf16", "bias": False,
         "act": None, "residual": True, "backward": False},
        # the same token's logits over the whole vocabulary
        {"name": "linear_head", "kind": "linear", "rows": 1, "in": 2048, "out": 50304, "group": 128, "type": "bf16", "bias": False,
         "act": None, "residual": False, "backward": False},
        # a small adapter's odd sizes, five rows, with a bias, in fp16
        {"name": "linear_odd", "kind": "linear", "rows": 5, "in": 1000, "out": 777, "group": 32, "type": "fp16", "bias": True,
         "act": None, "residual": False, "backward": False},
        # a decoding step of 16 sequences: the first product of the MLP with its activation
        {"name": "linear_batch", "kind": "linear", "rows": 16, "in": 2048, "out": 8192, "group": 64, "type": "bf16", "bias": False,
         "act": "gelu", "residual": False, "backward": False},
        # a decoding step of 64 sequences: the second product of the MLP
        {"name": "linear_many", "kind": "linear", "rows": 64, "in": 8192, "out": 2048, "group": 64, "type": "bf16", "bias": False,
         "act": None, "residual": True, "backward": False},
        # queries, keys and values of a prompt of ordinary (odd) length
        {"name": "linear_prompt", "kind": "linear", "rows": 777, "in": 2048, "out": 6144, "group": 64, "type": "bf16", "bias": False,
         "act": None, "residual": False, "backward": False},
        # two sequences of 2048 through a frozen layer whose adapters train: the product and the gradient of its input
        {"name": "linear_adapt", "kind": "linear", "rows": 4096, "in": 2048, "out": 8192, "group": 64, "type": "bf16", "bias": False,
         "act": None, "residual": False, "backward": True},
        # a layer's weights quantised again after an update, and read back
        {"name": "weights_layer", "kind": "weights", "in": 2048, "out": 8192, "group": 64, "type": "bf16"},
        # a small fp32 matrix of odd sizes
        {"name": "weights_odd", "kind": "weights", "in": 1001, "out": 777, "group": 32, "type": "fp32"},
        # the token just drawn for one sequence and its alternatives
        {"name": "scores_one", "kind": "scores", "rows": 1, "vocab": 50304, "room": 50304, "top": 5, "type": "bf16", "banned": False,
         "backward": False},
        # four prompts of 2048 tokens scored, with twenty alternatives of every token
        {"name": "scores_prompts", "kind": "scores", "rows": 8192, "vocab": 50304, "room": 50304, "top": 20, "type": "bf16",
         "banned": False, "backward": False},
        # a policy's step: log probabilities and entropy of sampled answers with their gradient; logits in rows of a padded vocabulary, banned tokens
        {"name": "scores_policy", "kind": "scores", "rows": 4001, "vocab": 50001, "room": 50304, "top": 0, "type": "bf16",
         "banned": True, "backward": True},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "weights", "scores", "scores"])
    if kind == "scores":
        vocab = _log(rng, 33, 262144)
        top = rng.choice([0, 1, 5, 20, 32])
        return {"kind": kind, "rows": _log(rng, 1, min(65536, MOST_LOGITS // vocab)), "vocab": vocab,
                "room": vocab + rng.choice([0, 0, 0, 7, 64]), "top": top, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "banned": rng.random() < 0.3, "backward": rng.random() < 0.5}
    n, m = _log(rng, 32, 8192), _log(rng, 32, 16384)
    if rng.random() < 0.5:      # the sizes of models are multiples of 64
        n, m = max(64, n // 64 * 64), max(64, m // 64 * 64)
    group = rng.choice([32, 64, 128])
    if kind == "weights":
        return {"kind": kind, "in": n, "out": m, "group": group, "type": rng.choice(["bf16", "fp16", "fp32"])}
    most = min(4096, MOST_PRODUCTS // (n * m))
    rows = rng.choice([_log(rng, 1, 16), _log(rng, 1, 256), _log(rng, 1, 4096)])
    back = rng.random() < 0.3
    return {"kind": kind, "rows": max(1, min(rows, most)), "in": n, "out": m, "group": group, "type": rng.choice(["bf16", "bf16", "fp16"]),
            "bias": rng.random() < 0.3, "act": None if back else rng.choice([None, "gelu", "relu"]), "residual": rng.random() < 0.3,
            "backward": back}


def work(case):
    if case["kind"] == "scores":
        n, t = case["rows"] * case["vocab"], TYPES[case["type"]].itemsize
        small = case["rows"] * (8 + 4 + 4 + 12 * case["top"])
        if case["backward"]:      # and the logits' gradient
            return {"bytes": 2.0 * n * t + 2 * small, "flops": 12.0 * n}
        return {"bytes": 1.0 * n * t + small, "flops": 6.0 * n}
    n, m = case["in"], case["out"]
    held = m * n / 2 + 2.0 * m * -(-n // case["group"])
    t = TYPES[case["type"]].itemsize
    if case["kind"] == "weights":
        return {"bytes": 2.0 * n * m * t + 2 * held, "flops": 4.0 * n * m}
    r, passes = case["rows"], 2 if case["backward"] else 1
    extra = (r * m if case["residual"] else 0) + (m if case["bias"] else 0)
    return {"bytes": held + passes * t * (r * n + r * m) + t * extra, "flops": 2.0 * passes * r * n * m}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _weight(case, gen):
    """Weights as an initialised or trained layer has them: normal values, some rows larger than others."""
    w = torch.randn((case["out"], case["in"]), generator=gen, device=DEV)
    w *= 0.02 * torch.exp(0.3 * torch.randn((case["out"], 1), generator=gen, device=DEV))
    return w.to(TYPES[case["type"]])


def _scores_inputs(case, gen):
    rows, vocab, t = case["rows"], case["vocab"], TYPES[case["type"]]
    held = torch.empty((rows, case["room"]), dtype=t, device=DEV)
    step = max(1, (1 << 26) // case["room"])
    for i in range(0, rows, step):      # in parts: the normal values take twice the room
        held[i:i + step] = (torch.randn(held[i:i + step].shape, generator=gen, device=DEV) * 2.5).to(t)
    logits = held[:, :vocab]
    targets = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    if case["banned"]:      # the same tokens in every row, by either of the marks in use
        ids = torch.randperm(vocab, generator=gen, device=DEV)[:max(1, vocab // 50)]
        logits[:, ids[0::2]] = -math.inf
        logits[:, ids[1::2]] = torch.finfo(t).min
        allowed = torch.ones(vocab, dtype=torch.bool, device=DEV)
        allowed[ids] = False
        allowed = allowed.nonzero()[:, 0]
        targets = allowed[torch.randint(0, allowed.numel(), (rows,), generator=gen, device=DEV)]
    # the model expects its token, more or less
    at = torch.arange(rows, device=DEV)
    bump = 6.0 + 3.0 * torch.randn(rows, generator=gen, device=DEV)
    logits[at, targets] = (logits[at, targets].float() + bump).to(t)
    targets[torch.rand(rows, generator=gen, device=DEV) < 0.03] = IGNORED
    return logits, targets


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "scores":
        s["logits"], s["targets"] = _scores_inputs(case, gen)
        if case["backward"]:
            rows = case["rows"]
            s["logits"].requires_grad_(True)
            s["grads"] = [torch.randn(rows, generator=gen, device=DEV) / rows, torch.randn(rows, generator=gen, device=DEV) * (0.01 / rows)]
            if case["top"]:
                s["grads"].append(torch.randn((rows, case["top"]), generator=gen, device=DEV) / rows)
        return s
    w = _weight(case, gen)
    if case["kind"] == "weights":
        s["weight"] = w
        return s
    t, rows = TYPES[case["type"]], case["rows"]
    if own:
        from spiraltorch_b200.ops import int4
        s["held"] = int4.quantize(w, group=case["group"])
    else:
        q, scale = _plain_quantize(w, case["group"])
        q = torch.nn.functional.pad(q + 8, (0, q.shape[1] % 2)).to(torch.uint8)
        s["held"] = (q[:, 0::2] | q[:, 1::2] << 4, scale)
    # normalised activations, a few channels much larger than the others
    x = torch.randn((rows, case["in"]), generator=gen, device=DEV)
    x[:, torch.randint(0, case["in"], (max(1, case["in"] // 500),), generator=gen, device=DEV)] *= 12.0
    s["x"] = x.to(t)
    s["bias"] = (torch.randn(case["out"], generator=gen, device=DEV) * 0.1).to(t) if case["bias"] else None
    s["residual"] = torch.randn((rows, case["out"]), generator=gen, device=DEV).to(t) if case["residual"] else None
    if case["backward"]:
        s["x"].requires_grad_(True)
        s["dy"] = torch.randn((rows, case["out"]), generator=gen, device=DEV).to(t)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------------
def _groups(w, group):
    """``[out, groups, group]``: the last group filled up with zeros."""
    return torch.nn.functional.pad(w, (0, -w.shape[1] % group)).unflatten(1, (-1, group))


def _plain_quantize(w, group):
    """Codes ``[out, in]`` and scales ``[out, groups]``, in fp64 next to the borders of rounding."""
    g = _groups(w.float(), group)
    low, high = g.amin(-1), g.amax(-1)
    m, e = torch.frexp(torch.where(high > -low, high, low) * -0.125)
    s = torch.ldexp(torch.round(m * 16), e - 4)
    s = torch.where(s < 0, -1.0, 1.0) * s.abs().clamp(*SCALE)
    q = torch.round(g.double() / s.double()[..., None]).clamp(-8, 7)
    return q.flatten(1)[:, :w.shape[1]].int(), s


def _plain_dequantize(q, scale, group):
    return q.float() * scale.repeat_interleave(group, 1)[:, :q.shape[1]]


def _plain_linear(s):
    case, (codes, scale) = s["case"], s["held"]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :case["in"]].int() - 8
    w = _plain_dequantize(q, scale, case["group"])
    t = s["x"].dtype
    with torch.no_grad():
        y = s["x"].float() @ w.T
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if case["act"] == "gelu":
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        elif case["act"] == "relu":
            y = y.clamp(min=0.0)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        out = [y.to(t)]
        if case["backward"]:
            out.append((s["dy"].float() @ w).to(t))
    return out


def _top_keys(x):
    """Whole numbers in the order of the values and, where these are equal, of the lower index."""
    b = (x + 0.0).view(torch.int32).long()
    b = torch.where(b < 0, (b & 0x7FFFFFFF).neg(), b)
    return (b << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_scores(s):
    case, targets = s["case"], s["targets"]
    with torch.no_grad():
        x = s["logits"].float()
        m = x.amax(1, keepdim=True)
        d = x - m
        e = d.exp()
        total = e.sum(1, keepdim=True)
        logp = d - total.log()
        p = e / total
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
        given = targets >= 0
        at = targets.clamp(min=0)[:, None]
        out = [torch.where(given, logp.gather(1, at)[:, 0], 0.0), entropy]
        ids = None
        if case["top"]:
            keys = _top_keys(x).topk(case["top"], dim=1).values
            ids = x.shape[1] - 1 - (keys & 0xFFFFFFFF)
            out += [ids, logp.gather(1, ids)]
        if case["backward"]:
            gl, gh = torch.where(given, s["grads"][0], 0.0)[:, None], s["grads"][1][:, None]
            all_given = gl + s["grads"][2].sum(1, keepdim=True) if case["top"] else gl
            g = -p * (all_given + gh * torch.where(p > 0, logp + entropy[:, None], 0.0))
            g.scatter_add_(1, at, gl)
            if case["top"]:
                g.scatter_add_(1, ids, s["grads"][2])
            out.append(g.to(s["logits"].dtype))
    return out


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if not own:
        if case["kind"] == "linear":
            return _plain_linear(s)
        if case["kind"] == "scores":
            return _plain_scores(s)
        return _plain_dequantize(*_plain_quantize(s["weight"], case["group"]), case["group"]).to(s["weight"].dtype)
    if case["kind"] == "scores":
        from spiraltorch_b200.ops import scoring
        r = scoring.token_scores(s["logits"], s["targets"], top=case["top"])
        out = [r.logprob, r.entropy] + ([r.top_ids, r.top_logprobs] if case["top"] else [])
        if case["backward"]:
            given = [r.logprob, r.entropy] + ([r.top_logprobs] if case["top"] else [])
            out = [t.detach() for t in out] + list(torch.autograd.grad(given, s["logits"], s["grads"]))
        return out
    from spiraltorch_b200.ops import int4
    if case["kind"] == "weights":
        return int4.dequantize(int4.quantize(s["weight"], group=case["group"]), s["weight"].dtype)
    y = int4.linear(s["x"], s["held"], s["bias"], act=case["act"], residual=s["residual"])
    if case["backward"]:
        return [y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]]
    return [y]


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------
def _exact_weight(w, group):
    """Element by element from the definition: every group's extremum, its scale by bits, the nearest multiple."""
    w = w.double()
    out = torch.zeros_like(w)
    for i in range(0, w.shape[1], group):
        part = w[:, i:i + group]
        low, high = part.min(1).values, part.max(1).values
        far = torch.where(-low >= high, low, high)
        size = (far.abs() / 8).clamp(min=1e-300)
        unit = torch.exp2(torch.floor(torch.log2(size)) - 3)
        unit = torch.where(size / unit >= 16, unit * 2, torch.where(size / unit < 8, unit / 2, unit))
        size = ((size / unit).round() * unit).clamp(*SCALE)
        step = torch.where(far > 0, -size, size)[:, None]
        out[:, i:i + group] = (part / step).round().clamp(-8, 7) * step
    return out


def exact(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "weights":
        return _exact_weight(_weight(case, gen), case["group"])
    if case["kind"] == "linear":
        w = _exact_weight(_weight(case, gen), case["group"])
        s = prepare(case, seed)
        y = torch.nn.functional.linear(s["x"].detach().double(), w, None if s["bias"] is None else s["bias"].double())
        if case["act"] == "gelu":
            y = torch.nn.functional.gelu(y, approximate="tanh")
        elif case["act"] == "relu":
            y = torch.relu(y)
        if s["residual"] is not None:
            y += s["residual"].double()
        return [y] + ([s["dy"].double() @ w] if case["backward"] else [])
    s = prepare(case, seed)
    rows, given = case["rows"], s["targets"] >= 0
    logprob, entropy = (torch.zeros(rows, dtype=torch.float64, device=DEV) for _ in range(2))
    ids = torch.zeros((rows, case["top"]), dtype=torch.int64, device=DEV)
    top = torch.zeros(ids.shape, dtype=torch.float64, device=DEV)
    grad = torch.zeros((rows, case["vocab"]) if case["backward"] else (0, 0), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // case["vocab"])
    for i in range(0, rows, step):
        a = slice(i, i + step)
        x = s["logits"].detach()[a].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        p = lp.exp()
        n = torch.arange(x.shape[0], device=DEV)
        entropy[a] = torch.special.entr(p).sum(1)
        logprob[a] = torch.where(given[a], lp[n, s["targets"][a].clamp(min=0)], 0.0)
        if case["top"]:
            ids[a] = x.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
            top[a] = lp[n[:, None], ids[a]]
        if case["backward"]:
            # d log p_t = onehot - p; d entropy = -p (log p + entropy)
            weight = torch.zeros_like(p)
            weight[n, s["targets"][a].clamp(min=0)] = torch.where(given[a], s["grads"][0][a].double(), 0.0)
            if case["top"]:
                weight = weight.scatter_add(1, ids[a], s["grads"][2][a].double())
            grad[a] = weight - p * weight.sum(1, keepdim=True)
            grad[a] += s["grads"][1][a].double()[:, None] * (torch.special.entr(p) - p * entropy[a][:, None])
    return [logprob, entropy] + ([ids, top] if case["top"] else []) + ([grad] if case["backward"] else [])


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
