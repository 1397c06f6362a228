"""Decoding with the cache: logits against the plain network whose keys and values pass the cache's rounding, prompts in parts, places that
wait, end and start again, refusals; on the GPU against the same decoder on the CPU."""
import pytest
import torch

from spiraltorch_b200.models.gpt import GPTConfig, GPTModel
from spiraltorch_b200.ops import paged as P
from spiraltorch_b200.ops import rotary as R

CONFIGS = [dict(), dict(norm="layer", positional="learned"), dict(rope_dim=32, rope_interleaved=True),
           dict(rope_scaling=R.Scaling("bands", 4.0, original=64))]


def _model(device="cpu", dtype=torch.float32, **kw):
    cfg = GPTConfig(vocab_size=96, d_model=128, n_layers=2, n_heads=2, ffn=256, seq_len=256, init_std=0.08, **kw)
    return GPTModel(cfg, device=device, dtype=dtype)


def _rounded(x, page):
    """fp64 keys or values [S, H, D] as the cache holds them when a sequence is stored at once."""
    y = x.clone()
    for i in range(0, x.shape[0], page):
        unit = torch.exp2(P.page_exponent(x[i:i + page].abs().amax((0, 2))).double())[None, :, None]
        y[i:i + page] = P.to_codes((x[i:i + page] / unit).float()).double() * unit
    return y


def _plain(model, tokens, page):
    """Logits of every position."""
    cfg, w = model.cfg, {k: v.detach().double() for k, v in model.p.items()}
    S, H, D = len(tokens), cfg.n_heads, cfg.head_dim

    def norm(x, name):
        if cfg.norm == "rms":
            return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.norm_eps) * w[name + ".gamma"]
        return torch.nn.functional.layer_norm(x, (cfg.d_model,), w[name + ".gamma"], w[name + ".beta"], cfg.norm_eps)

    h = w["embed.weight"][tokens]
    if cfg.positional == "learned":
        h = h + w["pos.weight"][:S]
    for l in range(cfg.n_layers):
        q, k, v = (norm(h, f"h{l}.norm1") @ w[f"h{l}.qkv.weight"].T).view(S, 3, H, D).unbind(1)
        if cfg.positional == "rope":
            q, k = (R.rotary_reference(t, torch.arange(S), model.rope_freq, cfg.rope_interleaved) for t in (q, k))
        k, v = _rounded(k, page), _rounded(v, page)
        s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5 + torch.full((S, S), float("-inf"), dtype=torch.float64).triu(1)
        h = h + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(S, H * D) @ w[f"h{l}.proj.weight"].T
        h = h + torch.nn.functional.gelu(norm(h, f"h{l}.norm2") @ w[f"h{l}.fc1.weight"].T, approximate="tanh") @ w[f"h{l}.fc2.weight"].T
    return norm(h, "norm_f") @ w["embed.weight"].T


@pytest.mark.parametrize("kw", CONFIGS)
def test_prompt_logits_against_the_plain_network(kw):
    """The decoder computes in fp32, the plain network in fp64.  A key or value that stands within fp32's error of a border between two codes may
    fall to the other one, 2^-4 of it away at most: seeds are as they are, such elements are few, and one moves a logit by its share of one head
    element in one key.  Allowed: 2 % of the logits' spread, which one code in 16 and a key in 5 would reach only if all of a head's 64 elements moved."""
    model = _model(**kw)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 96, (n,), generator=g) for n in (5, 33, 70)]
    for page in (16, 64):
        got = model.decoder(3, 128, page_size=page).extend(prompts)
        for p, row in zip(prompts, got):
            want = _plain(model, p, page)[-1]
            assert (row.double() - want).abs().max() <= 0.02 * want.std()


def test_parts_waiting_and_places_that_start_again():
    model = _model()
    g = torch.Generator().manual_seed(5)
    a, b, c = (torch.randint(0, 96, (n,), generator=g).tolist() for n in (40, 23, 9))
    d = model.decoder(2, 64, pages=5, page_size=16)
    whole = model.decoder(1, 64, page_size=64).extend([a])[0]
    assert d.extend([a[:17], []]).shape == (1, 96) and d.held == [17, 0]
    assert d.extend([a[17:39], b[:20]]).shape == (2, 96) and d.pages_left == 0
    last = d.step(torch.tensor([a[39], b[20]]))
    # the same tokens in parts: scales grow as tokens come, which re-rounds what becomes subnormal, and pages have other sizes
    assert torch.nn.functional.cosine_similarity(last[0], whole, dim=0) > 0.99
    with pytest.raises(ValueError, match="pages"):
        d.extend([c * 2, []])
    with pytest.raises(ValueError, match="tokens, at most"):
        d.extend([[], [1] * 60])
    assert d.held == [40, 21]
    d.release([1])
    assert d.pages_left == 2 and d.lengths.tolist() == [40, 0] and int(d.free_count) == 2
    again = d.extend([[], c])[0]
    fresh = model.decoder(1, 64, page_size=16).extend([c])[0]
    assert torch.equal(again, fresh)


def test_generate():
    model = _model()
    prompts = [[1, 2, 3], [7], list(range(30))]
    got = model.generate(prompts, 6, page_size=16)
    assert [len(t) for t in got] == [6, 6, 6]
    for p, t in zip(prompts, got):                        # alone, as in company
        d = model.decoder(1, 40, page_size=16)
        row = d.extend([p])
        for want in t:
            assert int(row.argmax()) == want
            row = d.step(torch.tensor([want]))
    stop = got[0][2]
    cut = model.generate(prompts, 6, stop=stop, page_size=16)
    for full, t in zip(got, cut):
        assert t == (full[:full.index(stop)] if stop in full else full)
    assert model.generate(prompts, 0) == [[], [], []]


def test_generate_up_to_the_last_learned_position():
    """The last new token is never appended."""
    model = _model(norm="layer", positional="learned")
    prompt = [i % 96 for i in range(250)]
    got = model.generate([prompt], 7)
    assert len(got[0]) == 7 and got == model.decoder(1, 256).generate([prompt], 7)
    assert [len(t) for t in model.generate([prompt + [1] * 6, [5]], 1)] == [1, 1] and model.generate([prompt + [1] * 6], 0) == [[]]
    with pytest.raises(ValueError, match="learned positions"):
        model.generate([prompt], 8)


def test_training_with_other_rotary_forms_matches_autograd():
    for kw in CONFIGS[2:]:
        cfg = GPTConfig(vocab_size=64, d_model=128, n_layers=1, n_heads=2, ffn=128, seq_len=8, init_std=0.05, **kw)
        model = GPTModel(cfg, device="cpu", dtype=torch.float32)
        tokens, targets = torch.randint(0, 64, (2, 8)), torch.randint(0, 64, (2, 8))
        w = model.p["h0.qkv.weight"]
        model.forward_backward(tokens, targets)
        grad = w.main_grad.clone()
        for at in ((3, 5), (70, 1), (130, 100), (300, 7)):      # q, q, k and v rows against differences
            with torch.no_grad():
                keep, loss = float(w[at]), []
                for step in (1e-2, -1e-2):
                    w[at] = keep + step
                    loss.append(float(model(tokens, targets)))
                w[at] = keep
            # fp32 losses near 4.2: 2^-22 each over 2e-2, and the third derivative's 1e-4 of a gradient
            assert abs((loss[0] - loss[1]) / 2e-2 - float(grad[at])) <= 2 * 4.2 * 2 ** -22 / 2e-2 + 0.01 * float(grad.abs().max())


def test_steps_past_the_end_as_replays_do_them():
    """Replays do not pass through the host's count: what lies beyond the last position is computed at it, not read from behind the table."""
    model = _model(norm="layer", positional="learned")
    d = model.decoder(1, 256)
    d.extend([[3] * 255])
    for _ in range(3):
        d._admit = lambda counts: None
        assert torch.isfinite(d.step(torch.tensor([5]))).all()
    assert d.lengths.tolist() == [258]


def _replay(d, tokens):
    """What the replay of a captured step does: the device's part of it, past the host's count."""
    held, admit = list(d.held), d._admit
    d._admit, d._capturing = lambda counts: None, lambda: True
    row = d.step(tokens)
    d._admit, d.held = admit, held
    del d._capturing
    return row


def test_calls_behind_replays_go_by_what_the_device_holds():
    model = _model()
    d, e = model.decoder(2, 64, pages=6, page_size=16), model.decoder(2, 64, pages=6, page_size=16)
    for x in (d, e):
        x.extend([[7] * 10, [8] * 10])
    for t in range(20):
        tokens = torch.tensor([t, 90 - t])
        assert torch.equal(_replay(d, tokens), e.step(tokens))
    assert d.pages_left == e.pages_left == 2 and d.held == e.held == [30, 30]
    with pytest.raises(ValueError, match="2 are left"):
        d.extend([[3] * 20, [1] * 20])
    for x in (d, e):
        x.release([1])
    assert d.pages_left == e.pages_left == 4
    for t in range(4):            # a released place waits: it takes neither tokens nor pages
        row, tokens = _replay(d, torch.tensor([t, 5])), torch.tensor([t, 6])
        assert torch.equal(row, e.step(tokens)) and (row[1] == 0).all() and (row[0] != 0).any()
    assert d.lengths.tolist() == [34, 0] and d.pages_left == 3 == int(d.free_count)
    with pytest.raises(ValueError, match="pages"):
        d.extend([[], [2] * 49])
    again = d.extend([[], list(range(40))])[0]
    assert torch.equal(again, model.decoder(1, 64, page_size=16).extend([list(range(40))])[0])
    assert d.held == [34, 40] and d.pages_left == 0 == int(d.free_count)
    e.extend([[], list(range(40))])
    row = d.step(torch.tensor([3, 4]))
    assert torch.equal(row, e.step(torch.tensor([3, 4]))) and (row[1] != 0).any() and d.held == [35, 41] == d.lengths.tolist()


def test_released_places_wait_in_steps():
    model = _model()
    d, e = model.decoder(3, 64, page_size=16), model.decoder(3, 64, page_size=16)
    for x in (d, e):
        x.extend([[1, 2], [3], [4, 5, 6]])
    d.release([1])
    for t in range(3):
        a, b = d.step(torch.tensor([t, 9, t + 1])), e.step(torch.tensor([t, 9, t + 1]))
        assert torch.equal(a[[0, 2]], b[[0, 2]]) and (a[1] == 0).all()
    assert d.held == [5, 0, 6] == d.lengths.tolist() and d.pages_left == 10
    d.release([0, 2])
    with pytest.raises(ValueError, match="released"):
        d.step(torch.tensor([1, 1, 1]))
    assert torch.equal(d.extend([[], [3], []])[0], model.decoder(1, 64, page_size=16).extend([[3]])[0])


def test_a_prompt_behind_a_replayed_token_sees_its_own_keys(monkeypatch):
    from spiraltorch_b200.models import gpt_decoder
    model = _model()
    prompt, rows = list(range(50, 80)), []
    for dense_from in (20, 1 << 30):
        monkeypatch.setattr(gpt_decoder, "DENSE_FROM", dense_from)
        d = model.decoder(1, 64, page_size=16)
        _replay(d, torch.tensor([3]))
        rows.append(d.extend([prompt])[0])
    # the same keys, values and products in another order at most
    assert torch.allclose(*rows, atol=1e-5)


def test_a_pass_that_fails_appends_nothing(monkeypatch):
    model = _model()
    d, e = (model.decoder(2, 64, pages=4, page_size=16) for _ in range(2))
    for x in (d, e):
        x.extend([[1, 2, 3], [4]])
    store, calls = P.store, []

    def failing(*args):
        calls.append(args)
        if len(calls) % 2 == 0:                  # the second layer's
            raise RuntimeError("no memory")
        store(*args)
    for call in (lambda x: x.extend([[5] * 20, []]), lambda x: x.step(torch.tensor([6, 7])), lambda x: x.extend([[], list(range(30))])):
        state = list(d.held), d.pages_left, d.lengths.tolist(), int(d.free_count)
        monkeypatch.setattr(P, "store", failing)
        with pytest.raises(RuntimeError, match="no memory"):
            call(d)
        monkeypatch.setattr(P, "store", store)
        assert (d.held, d.pages_left, d.lengths.tolist(), int(d.free_count)) == state
        assert torch.equal(call(d), call(e))


def test_an_error_record_of_the_kernels_ends_a_call(monkeypatch):
    from spiraltorch_b200.ops import native
    model, polls = _model(), []

    def poll(limit):
        polls.append(1)
        if len(polls) == limit:
            raise native.NativeError("device error")
    for limit in (1, 2, 3, 5):                  # while tokens are generated: at a call's beginning and where the host has read its tokens
        polls.clear()
        monkeypatch.setattr(native, "poll", lambda: poll(limit))
        with pytest.raises(native.NativeError):
            model.generate([[1, 2], [3]], 4)
    d = model.decoder(1, 64)
    for call in (lambda: d.extend([[1]]), lambda: d.step(torch.tensor([2]))):
        polls.clear()
        monkeypatch.setattr(native, "poll", lambda: poll(1))
        with pytest.raises(native.NativeError):
            call()
        assert d.held == [0] == d.lengths.tolist()


def test_refusals():
    model = _model(norm="layer", positional="learned")
    for bad in (lambda: model.decoder(0, 8), lambda: model.decoder(1, 0), lambda: model.decoder(1, 257), lambda: model.decoder(1, 8, page_size=24),
                lambda: model.decoder(2, 8).extend([[1]]), lambda: model.decoder(1, 8).extend([[96]]), lambda: model.decoder(1, 8).extend([[]]),
                lambda: model.decoder(1, 8).extend([[-1]]), lambda: model.decoder(2, 8).step(torch.zeros(1, dtype=torch.int64)),
                lambda: model.decoder(2, 8).step(torch.zeros(2)), lambda: model.decoder(1, 8).release([1]), lambda: model.generate([[]], 2),
                lambda: GPTModel(GPTConfig(vocab_size=64, d_model=128, n_layers=1, n_heads=2, ffn=128, rope_dim=66), device="cpu")):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", CONFIGS)
def test_gpu_decoder_follows_the_cpu_one(kw):
    gpu = _model("cuda", torch.bfloat16, **kw)
    cpu = _model(**kw)
    cpu.flat_w.copy_(gpu.flat_w.float().cpu())
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 96, (n,), generator=g) for n in (3, 100, 17)]
    a, b = gpu.decoder(3, 256, page_size=32), cpu.decoder(3, 256, page_size=32)
    rows = [(a.extend(prompts), b.extend(prompts))]
    rows.append((a.extend([p[:9] for p in prompts]), b.extend([p[:9] for p in prompts])))
    for _ in range(3):
        t = torch.randint(0, 96, (3,), generator=g)
        rows.append((a.step(t.cuda()), b.step(t)))
    for x, y in rows:
        # bf16 activations through two layers: 2^-8 a rounding, about ten of them in a row, and codes that fall to their neighbours (2^-4)
        assert torch.nn.functional.cosine_similarity(x.float().cpu(), y, dim=-1).min() > 0.99


@pytest.mark.gpu
@pytest.mark.parametrize("dense_from", [1, 80, 2048])
def test_gpu_parts_of_prompts_and_whole_ones(dense_from, monkeypatch):
    """Prompts read back and not, and long parts behind what the cache holds, which never are."""
    from spiraltorch_b200.models import gpt_decoder
    gpu = _model("cuda", torch.bfloat16)
    cpu = _model()
    cpu.flat_w.copy_(gpu.flat_w.float().cpu())
    g = torch.Generator().manual_seed(7)
    a, b = gpu.decoder(2, 256, page_size=16), cpu.decoder(2, 256, page_size=16)
    for parts in ((80, 90), (100, 70), (1, 65), (70, 0)):
        ids = [torch.randint(0, 96, (n,), generator=g) for n in parts]
        monkeypatch.setattr(gpt_decoder, "DENSE_FROM", dense_from)
        x = a.extend(ids)
        monkeypatch.setattr(gpt_decoder, "DENSE_FROM", 1 << 30)
        assert torch.nn.functional.cosine_similarity(x.float().cpu(), b.extend(ids), dim=-1).min() > 0.99


@pytest.mark.gpu
def test_gpu_step_captured():
    model = _model("cuda", torch.bfloat16)
    d, e = model.decoder(2, 200, page_size=16), model.decoder(2, 200, page_size=16)
    tokens = torch.tensor([3, 5], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in (d, e):
            x.extend([[1, 2, 3], [4]])
            x.step(tokens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = d.step(tokens)
    for i in range(60):
        tokens.copy_(torch.tensor([i, 95 - i]))
        graph.replay()
        assert torch.equal(out, e.step(tokens))


@pytest.mark.gpu
def test_gpu_calls_behind_replays():
    """Replays, a release between them and prompts behind them, against the same in eager calls: the same bits."""
    model = _model("cuda", torch.bfloat16)
    d, e = (model.decoder(3, 200, pages=30, page_size=16) for _ in range(2))
    tokens = torch.tensor([3, 5, 7], device="cuda")
    for x in (d, e):
        x.extend([[1, 2, 3], [4], [5] * 20])
        x.step(tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = d.step(tokens)
    assert d.held == [4, 2, 21]              # the capture itself appends nothing

    def turns(n):
        for i in range(n):
            tokens.copy_(torch.tensor([i, 95 - i, 2 * i]))
            graph.replay()
            assert torch.equal(out, e.step(tokens))
    turns(20)
    for x in (d, e):
        x.release([1])
    turns(17)
    assert (out[1] == 0).all() and d.pages_left == e.pages_left == int(d.free_count) and d.held == e.held == [41, 0, 58]
    prompt = list(range(40))
    assert torch.equal(d.extend([[9], prompt, []]), e.extend([[9], prompt, []]))
    turns(5)
    assert torch.equal(d.step(tokens), e.step(tokens)) and d.held == e.held == [48, 46, 64] == d.lengths.tolist()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        tokens + 1
        for call in (lambda: d.extend([[9], [], []]), lambda: d.release([0])):
            with pytest.raises(ValueError, match="captured"):
                call()
    torch.cuda.synchronize()
    assert d.held == [48, 46, 64]


@pytest.mark.gpu
def test_gpu_replays_without_pages():
    """A place whose tokens found no page is refused until it is released; the others go on."""
    from spiraltorch_b200.ops import native
    model = _model("cuda", torch.bfloat16)
    d, e = model.decoder(2, 64, pages=3, page_size=16), model.decoder(2, 64, page_size=16)
    tokens = torch.tensor([3, 5], device="cuda")
    for x in (d, e):
        x.extend([[1] * 15, [2] * 15])
        x.step(tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.step(tokens)
    graph.replay()                           # one page, two places that need one: the first gets it
    e.step(tokens)
    torch.cuda.synchronize()
    assert native.read_error_word()[0] == 3 and d.pages_left == 0
    with pytest.raises(ValueError, match="place 1 .* released"):
        d.step(tokens)
    for x in (d, e):
        x.release([1])
    assert d.pages_left == 1
    assert torch.equal(d.step(tokens), e.step(tokens)) and d.held == [18, 0]
    assert torch.equal(d.extend([[], [7] * 9])[0], model.decoder(1, 64, page_size=16).extend([[7] * 9])[0])


@pytest.mark.gpu
def test_gpu_error_records_surface_in_the_decoder():
    from spiraltorch_b200.ops import native
    d = _model("cuda", torch.bfloat16).decoder(1, 64, page_size=16)
    tokens = torch.tensor([3], device="cuda")
    d.extend([[1] * 20])
    page = int(d.table[0, 0])
    d.table[0, 0] = -1                       # the kernel's own check finds it
    d.step(tokens)
    torch.cuda.synchronize()
    with pytest.raises(native.NativeError, match="0x7004"):
        d.step(tokens)
    assert d.held == [21] and native.read_error_word()[0] == 0
    d.table[0, 0] = page
    d.step(tokens)
    torch.cuda.synchronize()
    assert native.read_error_word()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[300, 0, 129], [64, 1, 500]])
def test_gpu_whole_prompts_read_back_see_their_own_keys(counts):
    """Attention over what the cache gives back, by its own tolerance: scores are fp32 sums of D exact products, weights are rounded to bf16 (2^-8) and
    come from an exp2 of no more error than that, sums stay below 2^-16, and the result is rounded (2^-8): (2^-7 + 2^-16 + 2 D 2^-24 S) sum p |v| + 2^-8 |o|, S
    the largest sum |q_d k_d| / 8.  A mask that is one key off would take a row's own key from it."""
    d = _model("cuda", torch.bfloat16).decoder(3, 512, page_size=64)
    g = torch.Generator().manual_seed(9)
    rows, H, D = sum(counts), 2, 64
    q, k, v = (torch.randn(rows, H, D, generator=g).bfloat16() for _ in range(3))
    added = torch.tensor(counts, dtype=torch.int32, device="cuda")
    step = P.plan(d.lengths, added, d.table, d.free, d.free_count, page_size=64, rows=rows)
    P.store(k.cuda(), v.cuda(), d.cache[1], step.slots)
    got, r = d._dense(q.cuda(), 1, counts, step.lengths).cpu().double(), 0
    k, v = (t.cpu().double() for t in P.read(d.cache[1], d.table, step.lengths, max(counts), torch.float32))
    for b, n in enumerate(counts):
        s = torch.einsum("ihd,jhd->hij", q[r:r + n].double(), k[b, :n]) / 8 + torch.full((n, n), float("-inf"), dtype=torch.float64).triu(1)
        size = torch.einsum("ihd,jhd->hij", q[r:r + n].double().abs(), k[b, :n].abs()).tril().amax(-1) if n else torch.zeros(H, 0)
        p = torch.softmax(s, -1)
        want, A = torch.einsum("hij,jhd->ihd", p, v[b, :n]), torch.einsum("hij,jhd->ihd", p, v[b, :n].abs())
        off = (got[r:r + n] - want).abs()
        assert (off <= (2.0 ** -7 + 2.0 ** -16 + 2 * D * 2.0 ** -24 * size.T[..., None] / 8) * A + 2.0 ** -8 * want.abs()).all()
        r += n
