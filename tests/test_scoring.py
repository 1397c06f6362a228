"""Scores of given tokens: the CPU statement against torch's log_softmax and differences, the kernels against 64 bits where a row can go wrong (masked,
empty, equal, ordered, non-finite), refusals.

Tolerances.  x - m is off by half a step of fp32, 2^-24 |x - m|; a term of S is off by 2^-22 (exp2 and its argument) plus 2^-24 |x - m| of itself where it counts
(e^d d is below 0.37 at any d, so that part stays below 2^-24 of S / e^d), and up to vocab / 256 + 60 additions (8 per vector of a thread, then the joins) each by 2^-24: S is within
delta = 2^-21 + (vocab / 256 + 60) 2^-24 of itself, log S within delta.  m lies up to 4 below the largest element.  log p = x - m - log S: delta + 2^-23 (|x - m| + |log S| + 4), where |x - m| <= |log p| + log vocab + 4.
Entropy: the same for log S and delta (|T| / S + 4) for the quotient.  A gradient p (a + g (log p + H)): p and the bracket within twice the same, relative
to the sum of magnitudes, then half a step of the type."""
import math

import pytest
import torch

from spiraltorch_b200.ops import scoring

GPU = pytest.mark.gpu
cuda = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = math.inf


def _logits(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * scale).to(dtype), torch.randint(0, vocab, (rows,), generator=g)


def _hard(vocab, dtype, top):
    """Rows that are masked, empty, equal, ordered, far from zero, with one token, with values behind any bound that the first elements give."""
    low, big = torch.finfo(dtype).min, min(torch.finfo(dtype).max / 4, 1e30)
    base = _logits(1, vocab, dtype, 5)[0][0].float()
    ramp = torch.linspace(-20, 20, vocab)
    one = torch.full((vocab,), -INF)
    one[vocab // 2] = -7.0
    some = torch.full((vocab,), -INF)
    some[:: max(1, vocab // (top + 2))] = base[:: max(1, vocab // (top + 2))]
    holes = base.clone()
    holes[1::3] = -INF
    lows = base.clone()
    lows[::2] = low
    rows = [base, torch.full((vocab,), -INF), torch.zeros(vocab), torch.full((vocab,), low), ramp, ramp.flip(0), one, some, holes, lows, base + 1000.0, base - 1000.0,
            torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0), torch.full((vocab,), big), base.round(), torch.where(torch.arange(vocab) == vocab - 1, 50.0, low),
            base * 1e3 + (3e4 if dtype == torch.float16 else 3e6), base - (60000 if dtype == torch.float16 else 1048570), torch.where(base > 0, -INF, low),
            torch.where(torch.arange(vocab) < vocab // 2, -INF, base)]
    x = torch.stack(rows).to(dtype)
    t = torch.randint(0, vocab, (len(rows),), generator=torch.Generator().manual_seed(9))
    t[6], t[0] = vocab // 2, -100
    t[15], t[10] = vocab - 1, vocab
    return x, t


def _exact(x, t, top):
    return scoring.token_scores_reference(x.double(), t, top)


def _check(got, x, t, top):
    """Scores against 64 bits."""
    vocab = x.shape[1]
    want = _exact(x, t, top)
    delta = 2.0 ** -21 + (vocab / 256 + 60) * 2.0 ** -24
    span = math.log(vocab) + 4

    def near(a, b, allowed):
        a = a.double().cpu()
        same = (a == b) | (a.isnan() & b.isnan())
        assert ((a - b).abs() <= allowed)[~same].all(), float(((a - b).abs() / allowed)[~same].max())

    assert got.logprob.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32
    near(got.logprob, want.logprob, delta + 2.0 ** -23 * (want.logprob.abs().nan_to_num(0, 0, 0) + 3 * span))
    near(got.entropy, want.entropy, delta * (2 * span + 5) + 2.0 ** -23 * 3 * span)
    assert got.top_ids.dtype == torch.int64 and torch.equal(got.top_ids.cpu(), want.top_ids)
    near(got.top_logprobs, want.top_logprobs, delta + 2.0 ** -23 * (want.top_logprobs.abs().nan_to_num(0, 0, 0) + 3 * span))


@pytest.mark.parametrize("vocab,top", [(1, 1), (2, 0), (33, 5), (257, 32)])
def test_statement(vocab, top):
    x, t = _logits(6, vocab, torch.float64)
    s = scoring.token_scores(x, t, top=top)
    lp = torch.log_softmax(x, 1)
    assert torch.allclose(s.logprob, lp.gather(1, t[:, None])[:, 0], atol=1e-12)
    assert torch.allclose(s.entropy, -(lp.exp() * lp).sum(1), atol=1e-12)
    assert torch.equal(s.top_ids, lp.topk(top, 1).indices) and torch.allclose(s.top_logprobs, lp.topk(top, 1).values, atol=1e-12)


def test_statement_of_rows_that_are_masked():
    x, t = _hard(64, torch.float32, 5)
    s = scoring.token_scores(x, t, top=5)
    assert s.logprob[0] == 0 and s.logprob[10] == 0                                       # no such token
    assert s.logprob[1] == -INF and s.entropy[1] == 0 and s.top_ids[1].tolist() == [0, 1, 2, 3, 4] and (s.top_logprobs[1] == -INF).all()
    for r in (2, 3, 12, 13):                                                              # all equal
        assert torch.allclose(s.entropy[r], torch.tensor(math.log(64))) and s.top_ids[r].tolist() == [0, 1, 2, 3, 4]
    assert s.entropy[6] == 0 and s.logprob[6] == 0 and s.top_ids[6, 0] == 32
    x[0, 7] = math.nan
    x[1, 9] = INF
    s = scoring.token_scores(x[:2], t[:2].clamp(min=0), top=3)
    assert s.logprob.isnan().all() and s.entropy.isnan().all() and s.top_logprobs.isnan().all()
    assert s.top_ids[0, 0] == 7 and s.top_ids[1].tolist() == [9, 0, 1]


def test_statement_gradients():
    x, t = _logits(4, 9, torch.float64)
    t[2] = -100
    x[1, 3] = -INF
    x.requires_grad_(True)
    ref = x.detach().clone().requires_grad_(True)
    lp = torch.log_softmax(ref, 1)
    s = scoring.token_scores(x, t, top=3)
    gl, ge, gt = torch.randn(4, dtype=torch.float64), torch.randn(4, dtype=torch.float64), torch.randn(4, 3, dtype=torch.float64)
    ent = -torch.where(lp.isinf(), 0.0, lp.exp() * lp.masked_fill(lp.isinf(), 0.0)).sum(1)
    given = torch.where(t >= 0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    want = torch.autograd.grad((given * gl).sum() + (ent * ge).sum() + (lp.gather(1, s.top_ids) * gt).sum(), ref)[0]
    got = torch.autograd.grad((s.logprob, s.entropy, s.top_logprobs), x, (gl, ge, gt))[0]
    assert torch.allclose(got, want, atol=1e-12)
    y = torch.randn(3, 7, dtype=torch.float64, requires_grad=True)
    u = torch.tensor([1, 6, -100])
    assert torch.autograd.gradcheck(lambda y: (lambda s: (s.logprob, s.entropy, s.top_logprobs))(scoring.token_scores(y, u, top=2)), (y,))
    # one output's gradient alone, none at all, and an empty row
    only = torch.autograd.grad(scoring.token_scores(x, t).entropy.sum(), x)[0]
    assert torch.isfinite(only).all()
    e = torch.full((1, 5), -INF, requires_grad=True)
    s = scoring.token_scores(e, torch.tensor([2]), top=2)
    assert (torch.autograd.grad((s.logprob, s.entropy, s.top_logprobs), e, (torch.ones(1), torch.ones(1), torch.ones(1, 2)))[0] == 0).all()


def test_shapes_and_refusals():
    x, t = _logits(6, 11, torch.float32)
    s = scoring.token_scores(x.view(2, 3, 11), t.view(2, 3), top=4)
    assert s.logprob.shape == s.entropy.shape == (2, 3) and s.top_ids.shape == s.top_logprobs.shape == (2, 3, 4)
    s = scoring.token_scores(x[0], t[0])
    assert s.logprob.shape == () and s.top_ids.shape == (0,)
    assert scoring.token_scores(x[:0], t[:0], top=2).top_ids.shape == (0, 2)
    for call in (lambda: scoring.token_scores(x, t[:5]), lambda: scoring.token_scores(x, t.int()), lambda: scoring.token_scores(x, t, top=12),
                 lambda: scoring.token_scores(x, t, top=-1), lambda: scoring.token_scores(x.int(), t), lambda: scoring.token_scores(x[:, :0], t),
                 lambda: scoring.token_scores(torch.randn(2, 100), t[:2], top=33), lambda: scoring.token_scores(torch.tensor(1.0), torch.tensor(0))):
        with pytest.raises(ValueError):
            call()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError):
            scoring.token_scores(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), t)


# ---- kernels --------------------------------------------------------------------------------------------------------------------
VOCABS = [1, 2, 7, 31, 64, 257, 1000, 2048, 2049, 4099, 8192, 20011, 50304, 140001]


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_kernel(vocab, dtype):
    for rows, top in ((1, min(5, vocab)), (3, 0), (40, min(20, vocab)), (130, min(1, vocab)), (11, min(32, vocab))):
        x, t = _logits(rows, vocab, dtype, rows)
        t[0] = -100 if rows > 1 else t[0]
        _check(scoring.token_scores(x.to(cuda), t.to(cuda), top=top), x, t, top)


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [33, 300, 2048, 3001, 33000, 140001])
@pytest.mark.parametrize("rows", [20, 320])
def test_kernel_on_hard_rows(rows, vocab, dtype):
    for top in (0, 1, 32):
        x, t = _hard(vocab, dtype, top)
        x, t = x.repeat(rows // 20, 1), t.repeat(rows // 20)
        _check(scoring.token_scores(x.to(cuda), t.to(cuda), top=top), x, t, top)


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [2100, 5001])
def test_kernel_on_many_rows(vocab, dtype):
    for top in (0, 20):
        x, t = _hard(vocab, dtype, top)
        x, t = x.repeat(125, 1), t.repeat(125)
        _check(scoring.token_scores(x.to(cuda), t.to(cuda), top=top), x, t, top)


@GPU
@pytest.mark.parametrize("vocab,rows", [(1500, 3000), (2100, 3000), (5001, 3000), (5001, 5), (20011, 1000), (140001, 40), (263000, 3)])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_kernel_on_coarse_values_row_after_row(vocab, rows, top):
    """More elements than there is room for reach the bound in every second row, whose warps must agree that it is looked through with care."""
    g = torch.Generator().manual_seed(8)
    x = torch.where(torch.rand(rows, vocab, generator=g) < 0.999 - 0.9 * torch.rand(rows, 1, generator=g), 2.0, 1.0)
    x[1::2] = torch.randn(x[1::2].shape, generator=g)
    t = torch.randint(0, vocab, (rows,), generator=g)
    at = torch.arange(vocab)
    want = torch.where(x[0::2] == 2.0, at, at + vocab).topk(top, dim=1, largest=False).values % vocab
    x, t = x.bfloat16().to(cuda), t.to(cuda)
    _check(scoring.token_scores(x[:6], t[:6], top=top), x[:6].cpu(), t[:6].cpu(), top)
    first = scoring.token_scores(x, t, top=top)
    assert torch.equal(first.top_ids[0::2].cpu(), want)
    for _ in range(5):
        again = scoring.token_scores(x, t, top=top)
        assert all(torch.equal(a, b) for a, b in zip(again, first))


def _huge(vocab, dtype):
    """Different finite logits whose multiple log2 e is infinite (from 2.36e38 on): in one vector, in one thread's, in those of other lanes, warps and blocks."""
    base, t = _logits(11, vocab, torch.float32, 6)
    at = torch.arange(vocab)
    base[0, 1], base[0, 2] = 2.5e38, 3.3e38
    base[1, 1], base[1, 2] = 3.3e38, 2.5e38
    base[2], base[3] = torch.linspace(2.4e38, 3.38e38, vocab), torch.linspace(3.38e38, 2.4e38, vocab)
    base[4, 0], base[4, -1] = 2.5e38, 3.3e38
    base[5, ::8] = 2.3e38 + 1e38 * torch.rand(base[5, ::8].shape, generator=torch.Generator().manual_seed(7))
    base[6] = torch.where(at % 3 == 0, 3.3e38, 2.5e38)
    base[7] = torch.where(at % 2 == 0, -INF, torch.where(at % 5 == 0, 3e38, 2.4e38))
    base[8, -3:] = torch.tensor([2.35e38, 2.36e38, 2.37e38])
    base[9, vocab // 2], base[9, vocab // 2 + 1] = torch.finfo(dtype).max, 2.5e38
    base[10, :3] = torch.tensor([3.3e38, 2.5e38, math.nan])
    return base.to(dtype), t


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [9, 300, 2048, 5001, 50304, 140001, 263000])
def test_kernel_and_gradient_on_huge_rows(vocab, dtype):
    x, t = _huge(vocab, dtype)
    top = min(5, vocab)
    for k in (0, top):
        got = scoring.token_scores(x.to(cuda), t.to(cuda), top=k)
        _check(got, x, t, k)
        assert got.logprob[:10].isfinite().sum() >= 9 and got.entropy[:10].isfinite().all() and got.entropy[10].isnan()
    g = torch.Generator().manual_seed(2)
    _check_gradient(x[:10], t[:10], top, (torch.randn(10, generator=g), torch.randn(10, generator=g), torch.randn(10, top, generator=g)))


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [7, 300, 5001, 50304])
@pytest.mark.parametrize("scale", [30.0, 1000.0, 1e5])
def test_kernel_on_logits_far_apart(scale, vocab, dtype):
    """Log probabilities of thousands: as near as their difference from the largest logit allows."""
    if dtype == torch.float16 and scale > 1000:
        scale = 1e4
    x, t = _logits(400 if vocab < 50304 else 40, vocab, dtype, 3, scale)
    top = min(32, vocab)
    _check(scoring.token_scores(x.to(cuda), t.to(cuda), top=top), x, t, top)


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9, 300, 5000, 40000, 70001, 263000])
def test_kernel_non_finite(vocab, dtype):
    x, t = _logits(8, vocab, dtype, 3)
    x[0, 0], x[1, vocab - 1], x[2, vocab // 2], x[3, 1], x[3, 5], x[4, 2], x[4, 3] = math.nan, math.nan, INF, INF, math.nan, INF, -INF
    x[5] = math.nan
    x[6] = INF
    top = min(5, vocab)
    _check(scoring.token_scores(x.to(cuda), t.to(cuda), top=top), x, t, top)


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,pad,at", [(300, 7, 3), (300, 20, 4), (5001, 0, 0), (5001, 7, 1), (50001, 303, 0), (20011, 0, 0)])
def test_kernel_views(vocab, pad, at, dtype):
    x, t = _logits(5, vocab, dtype, 1)
    wide = torch.full((5, vocab + pad), math.nan, dtype=dtype, device=cuda)
    view = wide[:, at:at + vocab]
    view.copy_(x)
    _check(scoring.token_scores(view, t.to(cuda), top=7), x, t, 7)
    y = scoring.token_scores(x.to(cuda).T.contiguous().T, t.to(cuda), top=7)
    _check(y, x, t, 7)
    _check(scoring.token_scores(x[:1].to(cuda).expand(5, vocab), t.to(cuda), top=7), x[:1].expand(5, vocab), t, 7)


def _check_gradient(x, t, top, grads, layout=lambda x: x):
    leaf = layout(x.to(cuda)).requires_grad_(True)
    s = scoring.token_scores(leaf, t.to(cuda), top=top)
    outs = [(o, g) for o, g in zip((s.logprob, s.entropy, s.top_logprobs), grads) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], leaf, [g.to(cuda) for _, g in outs])[0]
    assert got.dtype == x.dtype and got.shape == x.shape
    gl, ge, gt = grads
    want = scoring._gradient_reference(x.double(), t, s.top_ids.cpu(), gl, ge, gt)
    vocab = x.shape[1]
    logp, entropy = scoring._statement(x.double())
    p = logp.exp()
    given = (t >= 0) & (t < vocab)
    own = torch.zeros_like(p)
    if gl is not None:
        own.scatter_add_(1, torch.where(given, t, 0)[:, None], torch.where(given, gl.abs(), 0.0)[:, None].double())
    if gt is not None:
        own.scatter_add_(1, s.top_ids.cpu(), gt.abs().double())
    size = own.sum(1, keepdim=True) + (0 if ge is None else ge.abs()[:, None] * (logp.abs().nan_to_num(0, 0, 0) + entropy.abs()[:, None] + 1))
    delta = 2.0 ** -21 + (vocab / 256 + 60) * 2.0 ** -24
    off = 2 * (delta + 2.0 ** -23 * (logp.abs().nan_to_num(0, 0, 0) + 3 * (math.log(vocab) + 4))) + 34 * 2.0 ** -24
    eps = torch.finfo(x.dtype).eps / 2
    allowed = p * size * off * (2 * math.log(vocab) + 13) + own * 34 * 2.0 ** -24 + eps * (want.abs() + torch.finfo(x.dtype).smallest_normal)
    d = (got.double().cpu() - want).abs()
    assert (d <= allowed).all(), float((d / allowed).max())


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 33, 300, 2048, 2049, 8192, 50001])
def test_gradient_kernel(vocab, dtype):
    for rows, top in ((1, min(5, vocab)), (19, 0), (150, min(32, vocab))):
        x, t = _logits(rows, vocab, dtype, rows)
        t[0] = -100 if rows > 1 else t[0]
        g = torch.Generator().manual_seed(2)
        gl, ge, gt = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, top, generator=g)
        for grads in ((gl, ge, gt if top else None), (gl, None, None), (None, ge, None)):
            _check_gradient(x, t, top, grads)


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [33, 300, 3001, 70000])
def test_gradient_kernel_on_hard_rows_and_views(vocab, dtype):
    x, t = _hard(vocab, dtype, 5)
    g = torch.Generator().manual_seed(2)
    grads = (torch.randn(20, generator=g), torch.randn(20, generator=g), torch.randn(20, 5, generator=g))
    _check_gradient(x, t, 5, grads)
    for pad, at in ((7, 3), (8, 8), (vocab, 0)):
        def layout(x):
            wide = torch.zeros((20, vocab + pad), dtype=dtype, device=cuda)
            wide[:, at:at + vocab] = x
            return wide.detach()[:, at:at + vocab]
        _check_gradient(x, t, 5, grads, layout)
    _check_gradient(x, t, 5, (grads[0][:1].expand(20), None, grads[2][:, :1].expand(20, 5)))


@GPU
def test_offsets_beyond_32_bits():
    x, t = _logits(3, 3001, torch.bfloat16)
    far = torch.empty((2 << 30) + 3008, dtype=torch.bfloat16, device=cuda).as_strided((3, 3001), (1 << 30, 1))
    far.copy_(x)
    far.requires_grad_(True)
    s = scoring.token_scores(far, t.to(cuda), top=3)
    _check(scoring.TokenScores(*(v.detach() for v in s)), x, t, 3)
    near = x.to(cuda).requires_grad_(True)
    want = torch.autograd.grad(scoring.token_scores(near, t.to(cuda)).logprob.sum(), near)[0]
    assert torch.equal(torch.autograd.grad(s.logprob.sum(), far)[0], want)


@GPU
def test_gradient_accumulates_and_non_finite_rows():
    x, t = _logits(6, 5000, torch.bfloat16)
    x[2, 9] = math.nan
    leaf = x.to(cuda).requires_grad_(True)
    for _ in range(2):
        scoring.token_scores(leaf, t.to(cuda)).logprob.sum().backward()
    assert leaf.grad[2].isnan().all() and not leaf.grad[[0, 1, 3, 4, 5]].isnan().any()
    one = torch.autograd.grad(scoring.token_scores(leaf, t.to(cuda)).logprob.sum(), leaf)[0]
    assert torch.equal((one + one)[0], leaf.grad[0])


@GPU
def test_streams_and_graphs():
    x, t = _logits(20, 9000, torch.bfloat16)
    x, t = x.to(cuda), t.to(cuda)
    want = scoring.token_scores(x, t, top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = scoring.token_scores(x, t, top=5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = x.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = scoring.token_scores(leaf, t, top=5)
        d = torch.autograd.grad((s.logprob, s.entropy), leaf, (torch.ones(20, device=cuda), torch.ones(20, device=cuda)))[0]
    with torch.no_grad():
        leaf.mul_(0.5)
    graph.replay()
    want = scoring.token_scores(leaf.detach(), t, top=5)
    assert all(torch.equal(a, b) for a, b in zip(s, want))
    y = leaf.detach().clone().requires_grad_(True)
    w = scoring.token_scores(y, t)
    assert torch.equal(d, torch.autograd.grad((w.logprob, w.entropy), y, (torch.ones(20, device=cuda), torch.ones(20, device=cuda)))[0])


@GPU
def test_kernel_refusals():
    x, t = _logits(3, 50, torch.float32)
    for call in (lambda: scoring.token_scores(x.to(cuda), t), lambda: scoring.token_scores(x, t.to(cuda)), lambda: scoring.token_scores(x.to(cuda).double(), t.to(cuda))):
        with pytest.raises(ValueError):
            call()


# ---- where the framework uses them ------------------------------------------------------------------------------------------------
def _model(device="cpu", dtype=torch.float32):
    from spiraltorch_b200.models.gpt import GPTConfig, GPTModel
    return GPTModel(GPTConfig(vocab_size=96, d_model=128, n_layers=2, n_heads=2, ffn=256, seq_len=256, init_std=0.08), device=device, dtype=dtype)


def _check_model_scores(model):
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 96, (3, 17), generator=g).to(model.flat_w.device)
    tokens[1, 9:] = -1
    got = model.score(tokens, top=4)
    logits = model(tokens.clamp(min=0)).view(3, 17, 96).float()
    lp = torch.log_softmax(logits.double(), -1)
    assert got.logprob.shape == got.entropy.shape == (3, 16) and got.top_ids.shape == got.top_logprobs.shape == (3, 16, 4)
    want = lp[:, :-1].gather(2, tokens[:, 1:].clamp(min=0)[..., None])[..., 0]
    want = torch.where(tokens[:, 1:] >= 0, want, 0.0)
    assert torch.allclose(got.logprob.double(), want, atol=2e-5) and (got.logprob[1, 8:] == 0).all()
    assert torch.allclose(got.entropy.double(), -(lp.exp() * lp).sum(-1)[:, :-1], atol=2e-5)
    assert torch.allclose(got.top_logprobs.double(), lp[:, :-1].topk(4).values, atol=2e-5)
    # minus the mean of the log probabilities is the loss
    whole = tokens.clamp(min=0)
    s = model.score(whole)
    targets = torch.cat([whole[:, 1:], whole.new_full((3, 1), -100)], 1)
    with torch.no_grad():
        assert torch.allclose(-s.logprob.mean(), model(whole, targets), atol=2e-5)


def test_scores_of_a_model():
    model = _model()
    _check_model_scores(model)
    with pytest.raises(ValueError):
        model.score(torch.zeros(3, 1, dtype=torch.int64))
    with pytest.raises(ValueError):
        model.score(torch.zeros(5, dtype=torch.int64))


def test_scores_of_no_sequence_are_refused():
    with pytest.raises(ValueError, match="with a sequence"):
        _model().score(torch.zeros(0, 5, dtype=torch.int64))
    with pytest.raises(ValueError, match="top must be 0 to 32"):
        _model().score(torch.zeros(1, 5, dtype=torch.int64), top=33)


def test_generated_tokens_with_scores():
    model = _model()
    prompts = [[1, 2, 3], [7], list(range(30))]
    plain = model.generate(prompts, 6)
    tokens, scores = model.generate(prompts, 6, scores=5)
    assert tokens == plain
    for p, t, s in zip(prompts, tokens, scores):
        assert len(s.logprob) == len(s.entropy) == len(s.top_ids) == len(s.top_logprobs) == 6
        assert [row[0] for row in s.top_ids] == t and [row[0] for row in s.top_logprobs] == s.logprob
        # the first of them is what the model says of the prompt
        got = model.score(torch.tensor([p + t[:1]]), top=5)
        assert abs(float(got.logprob[0, -1]) - s.logprob[0]) < 0.1 and abs(float(got.entropy[0, -1]) - s.entropy[0]) < 0.1      # the cache holds 8 bits
    stop = tokens[0][2]
    cut, judged = model.generate(prompts, 6, stop=stop, scores=0)
    assert [len(t) for t in cut] == [len(s.logprob) for s in judged] and all(row == [] for s in judged for row in s.top_ids)
    assert model.generate(prompts, 0, scores=2) == ([[], [], []], [([], [], [], [])] * 3)
    with pytest.raises(ValueError, match="alternatives"):
        model.generate(prompts, 1, scores=33)


@GPU
def test_scores_of_a_model_on_the_gpu():
    _check_model_scores(_model("cuda", torch.bfloat16))


def test_gradients_are_not_differentiated_twice():
    x, t = _logits(3, 11, torch.float32)
    x.requires_grad_(True)
    g = torch.autograd.grad(scoring.token_scores(x, t).logprob.sum(), x, create_graph=True)[0]
    assert torch.equal(g, torch.autograd.grad(scoring.token_scores(x, t).logprob.sum(), x)[0])
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.pow(2).sum(), x)


def _check_longer_than_learned_positions(device, dtype):
    from spiraltorch_b200.models.gpt import GPTConfig, GPTModel
    model = GPTModel(GPTConfig(vocab_size=96, d_model=128, n_layers=1, n_heads=2, ffn=256, seq_len=16, norm="layer", positional="learned"), device=device, dtype=dtype)
    tokens = torch.zeros(2, 17, dtype=torch.int64, device=device)
    for call in (lambda: model.score(tokens), lambda: model(tokens), lambda: model(tokens, tokens), lambda: model.forward_backward(tokens, tokens)):
        with pytest.raises(ValueError, match="learned positions for 16"):
            call()
    assert model.score(tokens[:, :16]).logprob.isfinite().all()


def test_sequences_longer_than_the_learned_positions():
    _check_longer_than_learned_positions("cpu", torch.float32)


@GPU
def test_sequences_longer_than_the_learned_positions_on_the_gpu():
    _check_longer_than_learned_positions("cuda", torch.bfloat16)
