"""The paged 8-bit cache: CPU statements against independent ones, refusals; kernels against the CPU statements (whole numbers and codes: equal)
and, for attention, against the formula in 64 bits.

Tolerance of attention.  With p the softmax weights of a row, A = sum p |v|, S = the largest sum_d |q_d k_d| * scale and n keys:
- scores are fp32 sums of D exact products: D 2^-24 S off at most, so a weight is that much off relatively, numerator and sum alike: 2 D 2^-24 S A;
- weights are rounded to fp16 relative to a reference that is 9 below one of the row's scores and never above the largest less 9, 2^-11 relatively, and what is
  below 2^-16 of that, 2^-25 of the largest, may be dropped: 2^-11 A + n 2^-25 max |v|;
- exp2 and the fp32 sums of weights and of products: 2^-20 A is more than their few units in the last place per step of 16 keys, for n up to 4096;
- the result is rounded once: half a step of the type times |o|."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from spiraltorch_b200.ops import paged as P

GPU = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


# ---- block tables -----------------------------------------------------------------------------------------------------------------
def _request(lengths, added, page, width, spare=0, device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [min(-(-(a + b) // page), width) for a, b in zip(lengths, added)]
    have = [min(-(-a // page), width) for a in lengths]
    order = torch.randperm(sum(need) + spare, generator=g).int()
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(have):
        table[b, :n] = order[at:at + n]
        at += n
    free = order[at:].clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)                            # noqa: E731
    return i32(lengths), i32(added), table.to(device), free.to(device), i32([free.numel()])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths,added,page,width,extra", [
    ([0], [1], 16, 1, 0), ([15, 16, 17], [1, 1, 1], 16, 3, 2), ([0, 0, 5, 0], [0, 40, 0, 3], 16, 4, 7), ([64], [0], 64, 1, 5), ([], [], 32, 2, 3),
    ([100, 3], [29, 0], 128, 2, 1), ([30, 0], [10, 70], 16, 4, 4), ([7] * 600, [2] * 600, 16, 2, 0), ([250, 0, 9], [1000, 777, 0], 64, 20, 9)])
def test_plan(device, lengths, added, page, width, extra):
    ln, ad, table, free, count = _request(lengths, added, page, width, 3, device)
    before, rows = table.clone(), sum(added) + extra
    step = P.plan(ln, ad, table, free, count, page_size=page, rows=rows)
    assert ln.tolist() == lengths and count.tolist() == [free.numel()]                            # inputs stay
    assert step.starts.tolist() == [sum(added[:b]) for b in range(len(added) + 1)]
    assert step.lengths.tolist() == [a + b for a, b in zip(lengths, added)]
    taken, r = [], 0
    got = table.tolist()
    for b, (have, n) in enumerate(zip(lengths, added)):
        old, new = min(-(-have // page), width), min(-(-(have + n) // page), width)
        assert got[b][:old] == before[b, :old].tolist() and got[b][new:] == before[b, new:].tolist()
        taken += got[b][old:new]
        for pos in range(have, have + n):
            assert step.positions[r] == pos
            assert step.slots[r] == (got[b][pos // page] * page + pos % page if pos // page < width else -1)
            r += 1
    assert taken == free.tolist()[::-1][:len(taken)] and step.free_count.tolist() == [free.numel() - len(taken)]
    assert step.positions[r:].tolist() == [0] * extra and step.slots[r:].tolist() == [-1] * extra


@pytest.mark.parametrize("device", DEVICES)
def test_plan_without_enough_pages(device):
    ln, ad, table, free, count = _request([0, 0], [40, 20], 16, 3, 0, device)
    count.fill_(4)
    step = P.plan(ln, ad, table, free, count, page_size=16, rows=60)
    assert step.free_count.tolist() == [-1] and table.tolist()[1][1] == -1
    assert (step.slots[:56] >= 0).all() and step.slots[56:].tolist() == [-1] * 4


@pytest.mark.parametrize("device", DEVICES)
def test_release_and_plan_again(device):
    ln, ad, table, free, count = _request([33, 5, 64], [0, 0, 0], 16, 4, 2, device)
    room = torch.full((free.numel() + 8,), -7, dtype=torch.int32, device=device)
    room[:free.numel()] = free
    before = table.clone()
    done = torch.tensor([True, False, True], device=device)
    P.release(ln, done, table, room, count, page_size=16)
    back = before[0, :3].tolist() + before[2, :4].tolist()
    assert ln.tolist() == [0, 5, 0] and count.tolist() == [9] and room.tolist() == free.tolist() + back + [-7]
    assert table.tolist() == [[-1] * 4, before[1].tolist(), [-1] * 4]
    P.release(ln, done, table, room, count, page_size=16)                                         # nothing left to give back
    assert count.tolist() == [9]
    step = P.plan(ln, torch.tensor([20, 0, 0], dtype=torch.int32, device=device), table, room, count, page_size=16, rows=20)
    assert table[0, :2].tolist() == back[::-1][:2] and step.free_count.tolist() == [7]


@GPU
def test_plan_of_many_sequences_and_strided_table():
    g = torch.Generator().manual_seed(3)
    lengths, added = torch.randint(0, 300, (8192,), generator=g).tolist(), torch.randint(0, 30, (8192,), generator=g).tolist()
    ln, ad, table, free, count = _request(lengths, added, 32, 11, 1)
    rows = sum(added) + 5
    wide = torch.full((8192, 16), -9, dtype=torch.int32, device="cuda")
    wide[:, :11] = table.cuda()
    got = P.plan(ln.cuda(), ad.cuda(), wide[:, :11], free.cuda(), count.cuda(), page_size=32, rows=rows)
    want = P.plan(ln, ad, table, free, count, page_size=32, rows=rows)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(wide[:, :11].cpu(), table) and (wide[:, 11:] == -9).all()
    with pytest.raises(ValueError, match="8193"):
        P.plan(*(t.cuda() for t in (torch.zeros(8193).int(), torch.zeros(8193).int(), torch.zeros(8193, 1).int(), free, count)), page_size=32, rows=4)


@GPU
def test_plan_of_many_sequences_in_a_process_of_its_own():
    """The prefix sums pass 48 KB of shared memory: launches that no larger one went before."""
    code = """
import torch
from spiraltorch_b200.ops import paged as P
i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
for B in (6100, 6126, 6127, 6143, 6144, 8192, 3):
    free = torch.arange(B, dtype=torch.int32, device="cuda")
    step = P.plan(i32(B), i32(B) + 1, i32(B, 1), free, i32(1) + B, page_size=16, rows=B)
    assert torch.equal(step.slots, 16 * free.flip(0).long()) and int(step.free_count) == 0, B
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0, done.stderr[-2000:]


# ---- storing and reading ----------------------------------------------------------------------------------------------------------
def _e4m3(x):
    """fp64 values to the nearest e4m3 value, by arithmetic."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _unit(amax):
    return next(2.0 ** e for e in range(-60, 61) if amax <= 448 * 2.0 ** e or e == 60)


def test_store_against_arithmetic():
    pages = P.Pages.allocate(4, 2, 16, 64, device="cpu")
    for t in pages[:2]:
        t.view(torch.uint8).fill_(0x7F)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 2, 64, generator=g) * torch.logspace(-3, 3, 40)[:, None, None]
    slots = torch.tensor(list(range(48, 64)) + list(range(0, 16)) + list(range(16, 24)))
    P.store(x[:20], -x[:20], pages, slots[:20])
    assert pages.k_scale[3, 0] == _unit(float(x[:16, 0].abs().max()))
    P.store(x[20:], -x[20:], pages, slots[20:])                                                   # the second page's scale grows
    table, lengths = torch.tensor([[3, 0, 1]], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    k, v = P.read(pages, table, lengths, 45, torch.float32)
    want = torch.zeros(45, 2, 64, dtype=torch.float64)
    for lo, hi, parts in ((0, 16, [16]), (16, 32, [20, 32]), (32, 40, [40])):
        for h in range(2):
            held, at = torch.zeros(0, 64, dtype=torch.float64), lo
            for end in parts:                                                                     # as stored, call by call
                unit = _unit(float(x[lo:end, h].abs().max()))
                held = torch.cat([_e4m3(held / unit) * unit, _e4m3(x[at:end, h].double() / unit) * unit])
                at = end
            want[lo:hi, h] = held
    assert torch.equal(k[0].double(), want) and torch.equal(v[0].double(), -want)
    assert torch.equal(P.read(pages, table, lengths, 45)[0].float(), k)                           # exact in bf16 too


@pytest.mark.parametrize("device", DEVICES)
def test_store_of_what_is_not_finite(device):
    pages = P.Pages.allocate(2, 1, 16, 64, device=device)
    x = torch.ones(6, 1, 64, device=device)
    x[1, 0, 3], x[2, 0, 5], x[3, 0, 7], x[4], x[5] = float("inf"), float("-inf"), float("nan"), 0.0, 3.0e38
    P.store(x[:5], x[:5] * 0, pages, torch.arange(5, device=device))
    P.store(x[4:], x[4:], pages, torch.tensor([16, -1], device=device))
    table, n = torch.tensor([[0, 1]], dtype=torch.int32, device=device), torch.tensor([17], dtype=torch.int32, device=device)
    k, v = (t[0, :, 0].cpu() for t in P.read(pages, table, n, 17, torch.float32))
    assert k[1, 3] == 448 * 2.0 ** -8 and k[2, 5] == -448 * 2.0 ** -8 and k[3, 7].isnan() and (k[0] == 1).all() and (k[4] == 0).all() and (k[16] == 0).all()
    assert v[0, 0] == 0 and v[1, 3].isnan() and pages.v_scale[0, 0] == 2.0 ** -60 and pages.k_scale[0, 0] == 2.0 ** -8
    P.store(x[5:], x[5:], pages, torch.tensor([5], device=device))                                # beyond what the largest scale holds
    assert pages.k_scale[0, 0] == 2.0 ** 60 and P.read(pages, table, n, 17, torch.float32)[0][0, 5, 0, 0] == 448 * 2.0 ** 60


@pytest.mark.parametrize("device", DEVICES)
def test_store_holds_values_alone(device):
    """Rows that require gradients: the cache takes their values and no part in the graph."""
    pages, k = P.Pages.allocate(2, 1, 16, 64, device=device), torch.randn(3, 1, 64, device=device, requires_grad=True)
    P.store(k * 2, k * 3, pages, torch.arange(3, device=device))
    assert not any(t.requires_grad for t in pages)
    table, n = torch.tensor([[0]], dtype=torch.int32, device=device), torch.tensor([3], dtype=torch.int32, device=device)
    assert not any(t.requires_grad for t in P.read(pages, table, n, 3))


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,page", [(64, 1, 16), (128, 3, 16), (128, 8, 64), (64, 12, 128), (128, 2, 256)])
def test_store_and_read_kernels(dtype, D, H, page):
    g = torch.Generator().manual_seed(D + H + page)
    cpu = P.Pages.allocate(40, H, page, D, device="cpu")
    for t in cpu[:2]:
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    gpu = P.Pages(*(t.cuda() for t in cpu))
    lengths, width = torch.zeros(9, dtype=torch.int32), 4
    table, free, count = torch.full((9, width), -1, dtype=torch.int32), torch.randperm(40, generator=g).int(), torch.tensor([36], dtype=torch.int32)
    for turn, added in enumerate([[1, 0, page, page + 1, 3, 2 * page - 1, 5, 1, 15], [1] * 9, [page - 1, 1, 1, 0, 14, 1, page, 7, 1], [2, 0, 1, 1, 1, 1, 1, 1, 1]]):
        added = [min(a, width * page - int(n)) for a, n in zip(added, lengths)]
        step = P.plan(lengths, torch.tensor(added, dtype=torch.int32), table, free, count, page_size=page, rows=sum(added) + 3)
        fused = (torch.randn(sum(added) + 3, 2 * H * D + 8, generator=g) * 10.0 ** (turn - 1)).to(dtype)
        k, v = (fused[:, i * H * D:(i + 1) * H * D].unflatten(1, (H, D)) for i in (0, 1))
        P.store(k, v, cpu, step.slots)
        fused = fused.cuda()
        k, v = (fused[:, i * H * D:(i + 1) * H * D].unflatten(1, (H, D)) for i in (0, 1))
        P.store(k, v, gpu, step.slots.cuda())
        lengths, count = step.lengths, step.free_count
        for out in (torch.bfloat16, torch.float32):
            for a, b in zip(P.read(gpu, table.cuda(), lengths.cuda(), width * page - 3, out), P.read(cpu, table, lengths, width * page - 3, out)):
                assert torch.equal(a.cpu(), b)
    for a, b in zip(gpu, cpu):                                                                    # and nothing else was written
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@GPU
def test_store_rows_off_a_16_byte_boundary_and_many_rows():
    H, D, page = 2, 64, 32
    x = torch.randn(2000 * H * D + 1, device="cuda").bfloat16()[1:].view(2000, H, D)
    a, b = (P.Pages(*(t.zero_() for t in P.Pages.allocate(70, H, page, D))) for _ in range(2))
    slots = torch.randperm(63, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
    slots = slots.flatten()[:2000]
    P.store(x, x * 2, a, slots)
    cpu = P.Pages(*(t.cpu() for t in b))
    P.store(x.cpu(), x.cpu() * 2, cpu, slots.cpu())
    for s, t in zip(a, cpu):
        assert torch.equal(s.cpu().view(torch.uint8), t.view(torch.uint8))


# ---- attention --------------------------------------------------------------------------------------------------------------------
def _cache(lengths, H, page, D, seed, spread=2):
    """Pages in a shuffled order, scales that differ by up to 2^spread; behind the lengths codes that are no number, and a table of -1."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    pages = P.Pages.allocate(sum(blocks) + 2, H, page, D, device="cpu")
    order, width = torch.randperm(sum(blocks) + 2, generator=g).int(), max(blocks + [0]) + 1
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        codes.copy_(P.to_codes(torch.randn(codes.shape, generator=g) * 100))
        scale.copy_(torch.exp2(torch.randint(-7, spread - 6, scale.shape, generator=g).float()))
    inside = torch.zeros(pages.k.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        for i in range(n):
            inside[table[b, i], :max(0, min(page, lengths[b] - i * page))] = True
        at += n
    for codes in pages[:2]:
        codes.view(torch.uint8).transpose(1, 2)[~inside] = 0x7F
    return pages, table


def _check_attention(lengths, added, H, G, page, D, dtype, causal=True, max_queries=None, extra=3, seed=0, scale=None, spread=2, edit=None):
    pages, table = _cache(lengths, H, page, D, seed, spread)
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(added) + extra
    fused = torch.randn(rows, H * G * D + 8, generator=g).to(dtype)
    if edit is not None:
        edit(pages, table, fused)
    starts, ln = torch.tensor([sum(added[:b]) for b in range(len(added) + 1)], dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
    q = fused[:, :H * G * D].unflatten(1, (H * G, D))
    want, lse = P.attention_reference(q, pages, table, starts, ln, causal, scale, torch.float64)
    size = P.Pages(pages.k, pages.v.float().abs().to(torch.float8_e4m3fn), pages.k_scale, pages.v_scale)
    weight = P.attention_reference(q, size, table, starts, ln, causal, scale, torch.float64)[0]
    sc = D ** -0.5 if scale is None else abs(scale)
    kmax = (pages.k.float().nan_to_num(0).abs() * pages.k_scale[..., None, None]).amax((0, 2)).double()       # [H, D]
    vmax = float((pages.v.float().nan_to_num(0).abs() * pages.v_scale[..., None, None]).max())
    top = (q.double().abs() * kmax.repeat_interleave(G, 0)).sum(-1, keepdim=True) * sc                        # no less than S
    cuda = [t.cuda() for t in (table, starts, ln)]
    fused = fused.cuda()
    q = fused[:, :H * G * D].unflatten(1, (H * G, D))
    dev = P.Pages(*(t.cuda() for t in pages))
    got, got_lse = P.attention(q, dev, *cuda, max_queries=max_queries or max(added + [1]), causal=causal, scale=scale, return_lse=True)
    n = max(lengths + [1])
    allowed = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -20 + 2 * D * 2.0 ** -24 * top) * weight + n * 2.0 ** -25 * vmax
    same = (got.cpu().double() == want) | (got.cpu().isnan() & want.isnan())                                  # zeros, NaN
    off = (got.cpu().double() - want).abs()
    assert (same | (off <= allowed)).all(), (off - allowed).nan_to_num(-1).max()
    same = (got_lse.cpu().double() == lse) | (got_lse.cpu().isnan() & lse.isnan())
    assert (same | ((got_lse.cpu().double() - lse).abs() <= D * 2.0 ** -24 * top[..., 0] + 2.0 ** -20 * (1 + lse.abs()))).all()
    out = torch.full_like(got, 7.0)
    assert P.attention(q, dev, *cuda, max_queries=max_queries or max(added + [1]), causal=causal, scale=scale, out=out) is out
    end = sum(added)
    assert (out[end:] == 7).all() and torch.equal(out[:end].nan_to_num(5), got[:end].nan_to_num(5)) and (got[end:] == 0).all()
    return got


LENGTHS = [1, 15, 16, 17, 63, 64, 65, 130, 333]


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G,page", [(64, 1, 1, 16), (128, 2, 1, 64), (128, 1, 4, 128), (64, 3, 8, 32), (128, 2, 5, 16), (128, 1, 16, 64), (64, 1, 27, 256), (128, 2, 71, 16)])
def test_attention_of_one_token(dtype, D, H, G, page):
    _check_attention(LENGTHS, [1] * len(LENGTHS), H, G, page, D, dtype, seed=G)


@GPU
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,H,G,page,dtype", [(64, 2, 1, 16, torch.float16), (128, 1, 2, 64, torch.bfloat16), (128, 2, 4, 32, torch.float16), (64, 1, 3, 128, torch.bfloat16)])
def test_attention_of_several_tokens(causal, D, H, G, page, dtype):
    lengths, added = [5, 70, 64, 1, 40, 129, 300, 16], [5, 3, 64, 1, 0, 2, 100, 16]
    _check_attention(lengths, added, H, G, page, D, dtype, causal)
    _check_attention(lengths, added, H, G, page, D, dtype, causal, max_queries=1)       # the tile may be too small, not wrong
    _check_attention([9, 33], [4, 5], H, G, page, D, dtype, causal, max_queries=100)


@GPU
def test_attention_rows_that_see_nothing():
    # more rows than tokens: the first rows lie before the sequence; no tokens at all; no sequences; no rows
    got = _check_attention([3, 0, 0, 20], [5, 2, 0, 1], 2, 4, 16, 64, torch.bfloat16)
    assert (got[:2] == 0).all() and (got[5:7] == 0).all() and (got[2] != 0).any()
    _check_attention([0], [1], 1, 1, 16, 128, torch.float16, causal=False)
    _check_attention([], [], 1, 2, 16, 64, torch.float16)
    pages = P.Pages.allocate(1, 1, 16, 64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")                            # noqa: E731
    assert P.attention(torch.zeros(0, 2, 64, device="cuda").half(), pages, i32(1, 1), i32(2), i32(1), max_queries=1).shape == (0, 2, 64)


@GPU
def test_attention_over_many_blocks_of_one_sequence():
    _check_attention([4096], [1], 1, 2, 64, 128, torch.bfloat16)
    _check_attention([3001, 7, 4095], [3, 2, 1], 2, 3, 16, 64, torch.float16)
    _check_attention([1024] * 150, [1] * 150, 1, 1, 64, 64, torch.float16)
    _check_attention([9] * 700, [1] * 700, 1, 2, 16, 64, torch.bfloat16)                # more sequences than a block scans at once
    _check_attention([9] * 700, [1] * 700, 1, 2, 16, 64, torch.bfloat16, max_queries=40)


@GPU
@pytest.mark.parametrize("D,H,G,page,dtype,lengths,added,causal", [
    (64, 2, 4, 256, torch.float16, [2500, 1, 900], [1, 1, 1], True), (128, 1, 4, 32, torch.bfloat16, [3000, 130], [4, 1], True),
    (64, 1, 16, 16, torch.bfloat16, [5000], [1], True), (128, 2, 4, 64, torch.float16, [4100, 3000], [20, 9], True),
    (64, 1, 3, 128, torch.bfloat16, [3000, 2400, 0, 700], [33, 3, 1, 17], False), (128, 1, 8, 16, torch.bfloat16, [2600, 2599], [64, 65], True),
    (64, 2, 2, 16, torch.float16, [2305, 2600], [40, 5], True)])
def test_attention_of_items_that_several_blocks_share(D, H, G, page, dtype, lengths, added, causal):
    _check_attention(lengths, added, H, G, page, D, dtype, causal, seed=D + G)


@GPU
@pytest.mark.parametrize("D,n,G,page", [(64, 1, 8, 16), (128, 2, 8, 64), (64, 9, 4, 16), (128, 9, 4, 256)])
def test_attention_of_long_sequences_whose_pages_are_none_or_hold_no_numbers(D, n, G, page):
    from spiraltorch_b200.ops import native
    lengths, added = [2600, 3000], [n, n]
    pages, table = _cache(lengths, 1, page, D, 4)
    starts, ln = torch.tensor([0, n, 2 * n], dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
    q = torch.randn(2 * n, G, D, generator=torch.Generator().manual_seed(4)).bfloat16()
    pages.v.view(torch.uint8)[table[1, 2999 // page], 0, 2999 % page, 7] = 0xFF       # seen by the last token's rows alone
    sees = torch.zeros(2 * n, dtype=torch.bool)
    sees[-1] = True
    want = P.attention_reference(q, pages, table, starts, ln, True, None, torch.float64)[0]
    dev = P.Pages(*(t.cuda() for t in pages))
    call = lambda table: P.attention(q.cuda(), dev, table.cuda(), starts.cuda(), ln.cuda(), max_queries=n)                      # noqa: E731
    good = call(table)
    assert torch.equal(good.isnan().any(-1).any(-1).cpu(), sees) and torch.allclose(good.cpu().double(), want, atol=0.1, rtol=0.01, equal_nan=True)
    holes = table.clone()                   # sequence 0: the first 256 keys, and some in the middle; they count as keys that no row sees
    holes[0, :256 // page] = -1
    holes[0, 1024 // page:1280 // page] = pages.k.shape[0]
    got = call(holes)
    torch.cuda.synchronize()
    assert native.read_error_word()[0] == 3
    assert torch.equal(got[n:].nan_to_num(5), good[n:].nan_to_num(5))
    seen = torch.cat([torch.arange(256, 1024), torch.arange(1280, 2600)])
    at = table[0, seen // page].long(), seen % page
    k, v = (c[at[0], 0, at[1]].double() * s[at[0], 0, None].double() for c, s in ((pages.k.float(), pages.k_scale), (pages.v.float(), pages.v_scale)))
    s = torch.einsum("ihd,kd->ihk", q[:n].double(), k) * D ** -0.5
    s.masked_fill_(seen[None, None] >= (2600 - n + 1 + torch.arange(n))[:, None, None], float("-inf"))
    assert torch.allclose(got[:n].cpu().double(), s.softmax(-1) @ v, atol=0.1, rtol=0.01)


@GPU
def test_attention_of_long_tables_captured_twice():
    """Items are split; two graphs and an eager call in turn have workspaces of their own."""
    lengths, H, G, D, page = [1, 40], 2, 4, 64, 16
    pages, table = _cache([3000, 1500], H, page, D, 6)
    pages.k.view(torch.uint8).bitwise_and_(0x77)                # numbers everywhere
    pages.v.view(torch.uint8).bitwise_and_(0x77)
    dev, table_gpu, starts = P.Pages(*(t.cuda() for t in pages)), table.cuda(), torch.arange(3, dtype=torch.int32, device="cuda")
    ln, q = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.randn(2, H * G, D, device="cuda").bfloat16()
    call = lambda: P.attention(q, dev, table_gpu, starts, ln, max_queries=1)                     # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for now in ([1, 40], [129, 1], [0, 1500], [3000, 1111], [2047, 1025]):
        ln.copy_(torch.tensor(now))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = call()
        torch.cuda.synchronize()
        want = P.attention_reference(q.cpu(), pages, table, starts.cpu(), ln.cpu(), True, None, torch.float64)[0]
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        assert torch.allclose(eager.cpu().double(), want, atol=0.1, rtol=0.01)


@GPU
@pytest.mark.parametrize("D,H,G,page,dtype,causal", [(128, 2, 1, 16, torch.bfloat16, True), (64, 1, 2, 64, torch.float16, True), (128, 1, 3, 256, torch.float16, False), (64, 2, 1, 128, torch.bfloat16, False)])
def test_attention_of_parts_of_prompts(D, H, G, page, dtype, causal):
    """Items of 128 rows: of one unit, two, an odd number; whole prompts and their ends; rows that fill no item."""
    _check_attention([1, 127, 128, 129, 256, 257, 385, 500], [1, 127, 128, 129, 100, 257, 385, 33], H, G, page, D, dtype, causal, seed=G, max_queries=400)
    _check_attention([3000, 40, 2500, 0], [200, 40, 129, 3], H, G, page, D, dtype, causal, seed=G)
    _check_attention([200, 130], [130, 130], H, G, page, D, dtype, causal, scale=-0.3)
    _check_attention([200, 130], [130, 130], H, G, page, D, dtype, causal, scale=0.0, spread=7)


@GPU
@pytest.mark.parametrize("D,dtype,page", [(64, torch.bfloat16, 16), (128, torch.bfloat16, 64), (64, torch.float16, 64), (128, torch.float16, 16)])
def test_attention_of_many_items_to_a_block(D, dtype, page):
    """Hundreds of items of one unit, two, three, four, in whole and shared ones."""
    lengths, added = [20 + 37 * (b % 13) for b in range(200)], [18 + b % 3 for b in range(200)]
    _check_attention(lengths, added, 2, 2, page, D, dtype, seed=D)
    _check_attention(lengths[:60] + [1700], added[:60] + [150], 4, 3, page, D, dtype, seed=D)


@GPU
def test_attention_of_parts_of_prompts_with_numbers_that_are_none():
    def values(pages, table, fused):       # hidden from the rows before them
        pages.v.view(torch.uint8)[table[0, 20], 0, 1, 5] = 0xFF
        pages.v.view(torch.uint8)[table[0, 3], 0, 13, 63] = 0x7F
        pages.k.view(torch.uint8)[table[0, 30], 0, 2, 9] = 0x7F
    got = _check_attention([500, 70], [460, 60], 1, 1, 16, 64, torch.bfloat16, edit=values)
    assert not got[:21, 0, 63].isnan().any() and got[21:460, 0, 63].isnan().all() and not got[:281, 0, 5].isnan().any() and got[281:460, 0, 5].isnan().all()
    assert got[442:460].isnan().all() and not got[460:].isnan().any() and not got[:442, 0, 6].isnan().any()
    def queries(pages, table, fused):      # one row's
        fused[7, 3] = float("nan")
    got = _check_attention([300], [200], 1, 1, 64, 128, torch.float16, edit=queries)
    assert got[7].isnan().all() and got.isnan().any(-1).sum() == 1


@GPU
def test_attention_scales_far_apart_and_large_scores():
    _check_attention(LENGTHS, [1] * 9, 2, 2, 16, 64, torch.bfloat16, spread=7)
    # value scales 2^40 apart: the codes of the small ones must not be lost in front of the large ones' masked or light keys
    def edit(pages, table, fused):
        pages.v_scale.copy_(torch.exp2(torch.arange(pages.v_scale.numel()).remainder(5).mul(10.0).sub(20)).view_as(pages.v_scale))
    _check_attention([16, 40, 5], [1, 1, 1], 1, 1, 16, 64, torch.bfloat16, edit=edit)
    _check_attention([100, 64], [1, 2], 1, 2, 16, 128, torch.bfloat16, scale=0.0)
    _check_attention([100, 64], [1, 2], 1, 2, 16, 128, torch.bfloat16, scale=-0.3)
    def tiny(pages, table, fused):      # queries of bf16's whole range keep their bits
        fused.mul_(2.0 ** -40)
        pages.k_scale.mul_(2.0 ** 40)
    _check_attention([100, 64], [1, 2], 1, 2, 16, 128, torch.bfloat16, edit=tiny)


@GPU
def test_attention_numbers_that_are_none():
    def queries(pages, table, fused):      # one row's query; other rows keep their results
        fused[1, 3] = float("nan")
    got = _check_attention([50, 60, 70], [1, 1, 1], 1, 1, 16, 64, torch.bfloat16, edit=queries)
    assert got[1].isnan().all() and not got[0].isnan().any() and not got[2].isnan().any()
    def values(pages, table, fused):       # a value of the last token: hidden from the rows before it
        pages.v.view(torch.uint8)[table[0, 3], 0, 1, 5] = 0xFF
        pages.v.view(torch.uint8)[table[0, 2], 0, 13, 63] = 0x7F
    got = _check_attention([50], [7], 1, 2, 16, 64, torch.bfloat16, edit=values)
    assert got[6, :, 5].isnan().all() and not got[:6, :, 5].isnan().any()
    assert got[1:, :, 63].isnan().sum() == 2 * 5 and not got[:, :, :5].isnan().any()
    def keys(pages, table, fused):
        pages.k.view(torch.uint8)[table[0, 3], 0, 1, 5] = 0x7F
    got = _check_attention([50], [3], 1, 1, 16, 128, torch.float16, edit=keys)
    assert got[2].isnan().all() and not got[:2].isnan().any()


@GPU
def test_attention_captured_while_sequences_grow():
    H, G, D, page, B = 2, 4, 64, 16, 3
    pages = P.Pages.allocate(60, H, page, D)
    table, free, count = torch.full((B, 18), -1, dtype=torch.int32, device="cuda"), torch.randperm(60, device="cuda").int(), torch.tensor([60], dtype=torch.int32, device="cuda")
    lengths, added = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.tensor([3, 1, 2], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(8, h, D, device="cuda").bfloat16() for h in (H * G, H, H))

    def one():
        step = P.plan(lengths, added, table, free, count, page_size=page, rows=8)
        P.store(k, v, pages, step.slots)
        o = P.attention(q, pages, table, step.starts, step.lengths, max_queries=3)
        lengths.copy_(step.lengths)
        count.copy_(step.free_count)
        return o

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        one()
    torch.cuda.default_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:                    # two graphs with workspaces of their own
        with torch.cuda.graph(graph):
            outs.append(one())
    lengths.zero_()
    count.fill_(60)
    table.fill_(-1)
    cpu = P.Pages(*(t.cpu() for t in pages))
    ct, cl, cc, cf = table.cpu(), lengths.cpu(), count.cpu(), free.cpu()
    for turn in range(40):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        graphs[turn % 2].replay()
        step = P.plan(cl, added.cpu(), ct, cf, cc, page_size=page, rows=8)
        P.store(k.cpu(), v.cpu(), cpu, step.slots)
        want = P.attention_reference(q.cpu(), cpu, ct, step.starts, step.lengths)[0]
        cl, cc = step.lengths, step.free_count
        assert torch.equal(table.cpu(), ct) and torch.equal(lengths.cpu(), cl) and torch.equal(count.cpu(), cc)
        assert torch.allclose(outs[turn % 2].cpu().float(), want, atol=0.02, rtol=0.01)


@GPU
def test_attention_repeats_its_bits_and_keeps_streams_apart():
    lengths, H, G, D, page = [700, 31, 2000], 2, 4, 128, 64
    pages, table = _cache(lengths, H, page, D, 5)
    dev, table = P.Pages(*(t.cuda() for t in pages)), table.cuda()
    starts, ln = torch.arange(4, dtype=torch.int32, device="cuda"), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(3, H * G, D, device="cuda").bfloat16() for _ in range(2)]
    want = [P.attention(q, dev, table, starts, ln, max_queries=1) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(P.attention(qs[i], dev, table, starts, ln, max_queries=1))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


@GPU
@pytest.mark.parametrize("D,G,n", [(128, 4, 1), (64, 3, 5), (128, 4, 8), (64, 8, 20), (128, 2, 70)])
def test_attention_of_rows_at_odd_places_and_in_place(D, G, n):
    """Rows, heads and results off a 16-byte boundary, and results over the queries: the same bits."""
    lengths, H, page = [1700, 3000], 2, 64
    pages, table = _cache(lengths, H, page, D, 8)
    dev, table = P.Pages(*(t.cuda() for t in pages)), table.cuda()
    starts, ln = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda"), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(2 * n + 1, H * G, D, device="cuda").half()
    want = P.attention(q, dev, table, starts, ln, max_queries=n)
    room = torch.zeros(2, 2 * n + 1, H * G, D + 1, device="cuda").half()
    odd, out = room[0, ..., 1:], room[1, ..., 1:]
    odd.copy_(q)
    assert torch.equal(P.attention(odd, dev, table, starts, ln, max_queries=n), want)
    P.attention(q, dev, table, starts, ln, max_queries=n, out=out)
    assert torch.equal(out[:2 * n], want[:2 * n]) and (room[1, ..., 0] == 0).all() and (out[2 * n:] == 0).all()
    P.attention(odd, dev, table, starts, ln, max_queries=n, out=odd)
    assert torch.equal(odd[:2 * n], want[:2 * n]) and torch.equal(odd[2 * n:], q[2 * n:])


@GPU
@pytest.mark.parametrize("lengths", [[700, 90, 1100], [700, 2500, 4000]])
def test_attention_of_parts_of_prompts_on_two_streams_and_captured(lengths):
    n, H, G, D, page = 60, 2, 2, 128, 64
    pages, table = _cache(lengths, H, page, D, 9)
    dev, table = P.Pages(*(t.cuda() for t in pages)), table.cuda()
    starts, ln = torch.arange(4, dtype=torch.int32, device="cuda") * n, torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(3 * n, H * G, D, device="cuda").bfloat16() for _ in range(2)]
    call = lambda i: P.attention(qs[i], dev, table, starts, ln, max_queries=n)                   # noqa: E731
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams, graphs, got, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [[], []], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs.append(call(i))
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


@GPU
def test_pages_that_are_none_are_refused_by_the_kernels():
    from spiraltorch_b200.ops import native
    pages = P.Pages(*(t.zero_() for t in P.Pages.allocate(3, 1, 16, 64)))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")                           # noqa: E731
    q = torch.randn(1, 1, 64, device="cuda").bfloat16()
    for table in (i32(0, -1).view(1, 2), i32(0, 3).view(1, 2)):
        P.attention(q, pages, table, i32(0, 1), i32(20), max_queries=1)
        torch.cuda.synchronize()
        assert native.read_error_word()[0] == 3
        k, v = P.read(pages, table, i32(20), 20)
        torch.cuda.synchronize()
        assert native.read_error_word()[0] == 3 and (k[0, 16:] == 0).all()
    P.store(q, q, pages, torch.tensor([48], device="cuda"))
    torch.cuda.synchronize()
    assert native.read_error_word()[0] == 3 and all((t.view(torch.uint8) == 0).all() for t in pages)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attention_log_sums_of_rows_of_no_sequence(device, n):
    """In a given output such rows stay as they were; their log-sum-exp, which the call makes, is that of no keys."""
    pages, table = _cache([50, 64], 2, 16, 64, 3)
    pages, table = P.Pages(*(t.to(device) for t in pages)), table.to(device)
    starts, ln = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([0, n, 2 * n], [50, 64]))
    rows = 2 * n + 6
    q, out = torch.randn(rows, 4, 64).bfloat16().to(device), torch.full((rows, 4, 64), 7.0, device=device).bfloat16()
    want = P.attention(q, pages, table, starts, ln, max_queries=n, return_lse=True)
    junk = [torch.full((rows, 4), 3.0, device=device) for _ in range(4)]        # what the call's own memory may have held
    del junk
    got = P.attention(q, pages, table, starts, ln, max_queries=n, return_lse=True, out=out)
    assert torch.equal(got[1], want[1]) and (got[1][2 * n:] == float("-inf")).all()
    assert got[0] is out and (out[2 * n:] == 7).all() and torch.equal(out[:2 * n], want[0][:2 * n])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attention_of_some_of_the_sequences(device, n):
    """A part of starts, table and lengths: rows before the first sequence are no sequence's either, and are 0."""
    pages, table = _cache([70, 50, 64, 90], 2, 16, 64, 3)
    pages, table = P.Pages(*(t.to(device) for t in pages)), table.to(device)
    starts, ln = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([0, n, 2 * n, 3 * n, 4 * n], [70, 50, 64, 90]))
    q = torch.randn(4 * n + 3, 4, 64).bfloat16().to(device)
    o, lse = P.attention(q, pages, table, starts, ln, max_queries=n, return_lse=True)
    for first, last in ((1, 3), (2, 4), (3, 3), (4, 4), (0, 4)):
        junk = [torch.full_like(q, 3.0) for _ in range(4)], [torch.full_like(lse, 3.0) for _ in range(4)]
        del junk
        part = table[first:last], starts[first:last + 1], ln[first:last]
        got, got_lse = P.attention(q, pages, *part, max_queries=n, return_lse=True)
        mine = slice(first * n, last * n)
        assert torch.equal(got[mine], o[mine]) and torch.equal(got_lse[mine], lse[mine])
        for rest in (slice(0, first * n), slice(last * n, None)):
            assert (got[rest] == 0).all() and (got_lse[rest] == float("-inf")).all()
        out = torch.full_like(q, 7.0)
        got_lse = P.attention(q, pages, *part, max_queries=n, return_lse=True, out=out)[1]
        assert torch.equal(out[mine], o[mine]) and torch.equal(got_lse[mine], lse[mine])
        for rest in (slice(0, first * n), slice(last * n, None)):
            assert (out[rest] == 7).all() and (got_lse[rest] == float("-inf")).all()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refuses_tangents(device):
    import torch.autograd.forward_ad as fw
    pages = P.Pages(*(t.zero_() for t in P.Pages.allocate(2, 1, 16, 64, device=device)))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)                           # noqa: E731
    q = torch.randn(1, 2, 64, device=device).bfloat16()
    call = lambda q: P.attention(q, pages, i32(0).view(1, 1), i32(0, 1), i32(3), max_queries=1)  # noqa: E731
    with fw.dual_level():
        with pytest.raises(ValueError, match="not differentiable"):
            call(fw.make_dual(q, torch.ones_like(q)))
        assert (call(q) == 0).all()


def _rows_and_limits(q, pages, table, lengths, added, causal=True, weight=2.0 ** -11):
    """Per row, in 64 bits: results, log-sum-exp, whether it sees a key, and how far off results and log-sum-exp may be by the keys that it sees itself (the module's
    terms; ``weight``: half a step of the type that weights are rounded to).  n keys: sums in steps of 32 products, each step off by a unit of fp32, 2^-23 (n / 32 + 16) A
    with exp2's and the last sums' own; x + b in fp32 with b up to 60: 2^-22 (64 + S) A; of the weights times 2^b, which are what is rounded, 2^-25 of the largest
    may be dropped for each key: 2^-25 max(p 2^b) sum |code|.  Below the type's smallest normal number N its steps are eps N apart, so half a step is eps / 2 max(|o|, N);
    a result that may lie half a step above its largest number may be infinite (both in fp16 only: N = 2^-14, 65504 + 16).  The log-sum-exp is formed from the logarithm of the sum and a reference that both hold b."""
    rows, heads, D = q.shape
    H, page = pages.k.shape[1:3]
    G, at = heads // H, 0
    want, limit = torch.zeros(rows, heads, D, dtype=torch.float64), torch.zeros(rows, heads, D, dtype=torch.float64)
    lse, sees = torch.full((rows, heads), float("-inf"), dtype=torch.float64), torch.zeros(rows, dtype=torch.bool)
    lse_limit = torch.zeros(rows, heads, dtype=torch.float64)
    for b, (length, n) in enumerate(zip(lengths, added)):
        of, off = table[b, torch.arange(length) // page].long(), torch.arange(length) % page
        seen = torch.arange(length) < (length - n + 1 + torch.arange(n) if causal else torch.full((n,), length))[:, None]        # [n, length]
        some = seen.any(1)
        sees[at:at + n] = some
        for h in range(H):
            k, v = pages.k[of, h, off].double() * pages.k_scale[of, h, None], pages.v[of, h, off].double() * pages.v_scale[of, h, None]
            unit = pages.v_scale[of, h].double()
            x = q[at:at + n, h * G:(h + 1) * G].double() * D ** -0.5
            s = (x @ k.T).masked_fill(~seen[:, None], float("-inf"))
            size = (x.abs() @ k.abs().T).masked_fill(~seen[:, None], 0.0).amax(-1, keepdim=True) if length else torch.zeros(n, G, 1)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            cols, A = slice(h * G, (h + 1) * G), p @ v.abs()
            want[at:at + n, cols], lse[at:at + n, cols] = p @ v, torch.logsumexp(s, -1) if length else float("-inf")
            drop = 2.0 ** -25 * (p * unit).amax(-1, keepdim=True) * (seen.double() @ (v.abs() / unit[:, None]))[:, None] if length else 0.0
            sums = 2.0 ** -23 * (length / 32 + 16) + 2.0 ** -22 * (64 + size)
            limit[at:at + n, cols] = torch.finfo(q.dtype).eps / 2 * (p @ v).abs().clamp(min=torch.finfo(q.dtype).smallest_normal) + (weight + sums + 2 * D * 2.0 ** -24 * size) * A + drop
            lse_limit[at:at + n, cols] = (sums + D * 2.0 ** -24 * size)[..., 0] + 2.0 ** -22 * (64 + lse[at:at + n, cols].abs())
        at += n
    return want, lse, sees, limit, lse_limit


def _check_rows(pages, table, lengths, added, H, G, D, dtype, causal=True, max_queries=None, seed=0):
    q = torch.randn(sum(added), H * G, D, generator=torch.Generator().manual_seed(seed)).to(dtype)
    want, lse, sees, limit, lse_limit = _rows_and_limits(q, pages, table, lengths, added, causal)
    starts = torch.tensor([sum(added[:b]) for b in range(len(added) + 1)], dtype=torch.int32)
    got, got_lse = P.attention(q.cuda(), P.Pages(*(t.cuda() for t in pages)), table.cuda(), starts.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                               max_queries=max_queries or max(added), causal=causal, return_lse=True)
    got, off = got.cpu(), (got.cpu().double() - want).abs()
    beyond = got.isinf() & (got.sign() * want + limit >= torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4))
    bad = ~beyond & ~(off <= limit)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), got[bad][:4], want[bad][:4], limit[bad][:4])
    assert ((got_lse.cpu().double() - lse)[sees].abs() <= lse_limit[sees]).all() and (got_lse.cpu()[~sees] == float("-inf")).all()
    held = want.abs().amax(-1) >= torch.finfo(dtype).smallest_normal * 16
    assert (limit < want.abs()).any(-1)[sees[:, None] & held].all() and (got[~sees] == 0).all()        # zeros would not pass for a row that sees a key and whose results the type holds
    assert dtype != torch.bfloat16 or held[sees].all()


@GPU
@pytest.mark.parametrize("D,G,n,page,lengths,causal", [
    (64, 1, 8, 16, [50, 34, 8], True), (128, 2, 8, 16, [50, 35, 16], True), (64, 4, 8, 32, [66, 36, 9], True), (128, 2, 64, 16, [100, 80, 64], True), (64, 1, 150, 16, [200, 160, 150], True),
    (128, 1, 8, 64, [2565, 70, 1000], True), (64, 2, 8, 16, [2597, 1700, 9], True), (128, 4, 8, 64, [2690, 70, 2400], True), (64, 2, 80, 32, [2600, 1700, 100], True), (128, 1, 130, 64, [2600, 133, 1800], False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_with_large_values_that_first_rows_do_not_see(D, G, n, page, lengths, causal, dtype):
    """Values 2^20 to 2^40 times as large in a sequence's last pages, hidden from its first rows, whose results come from the small ones; and in the
    pages of another sequence.  Tolerances are each row's own."""
    pages, table = _cache(lengths, 2, page, D, n + D)
    for length, entries, by in zip(lengths[:2], table, (2.0 ** 40, 2.0 ** 20)):
        hidden = range(-(-(length - n + 1) // page), -(-length // page))        # begin behind the keys of the first row
        assert len(hidden) > 0
        pages.v_scale[entries[list(hidden)].long()] *= by
    pages.v_scale[table[2, :-(-lengths[2] // page)].long()] *= 2.0 ** -30
    _check_rows(pages, table, lengths, [n] * 3, 2, G, D, dtype, causal)
    if n == 8:
        _check_rows(pages, table, lengths, [n] * 3, 2, G, D, dtype, causal, max_queries=200)
        _check_rows(pages, table, lengths, [1] * 3, 2, G, D, dtype, causal)


@GPU
@pytest.mark.parametrize("D,G,n", [(64, 1, 1), (128, 8, 1), (64, 2, 7), (128, 4, 8), (64, 3, 50), (128, 1, 140)])
def test_attention_of_scores_far_below_zero(D, G, n):
    """Scores near -10^36, within fp32's range: no less a row's keys than others.  The keys are equal and their scores with them, so weights are exactly alike and
    results are means, rounded to bf16 (2^-8); a log-sum-exp is off by its fp32 sum of D products of one sign, D 2^-24 of it, and a few roundings."""
    lengths = [n, 150, 1, 2600]
    added = [n, n, 1, n]
    pages, table = _cache(lengths, 1, 16, D, D + n)
    pages.k.copy_(torch.full((D,), 96.0)), pages.k_scale.fill_(2.0 ** 60), pages.v_scale.fill_(2.0 ** -5)
    pages.v.view(torch.uint8).masked_fill_(pages.v.isnan(), 0)
    starts = torch.tensor([0, n, 2 * n, 2 * n + 1, 3 * n + 1], dtype=torch.int32)
    q = torch.full((3 * n + 1, G, D), -2.0 ** 50).bfloat16()
    got, lse = (t.cpu().double() for t in P.attention(q.cuda(), P.Pages(*(t.cuda() for t in pages)), table.cuda(), starts.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                                                      max_queries=n, return_lse=True))
    score = -2.0 ** 50 * 96 * 2.0 ** 60 * D ** 0.5
    for b, (length, m) in enumerate(zip(lengths, added)):
        of = table[b, torch.arange(length) // 16].long(), torch.arange(length) % 16
        v = pages.v[of[0], 0, of[1]].double() * 2.0 ** -5
        for i in range(m):
            seen, r = length - m + 1 + i, int(starts[b]) + i
            want, size = v[:seen].mean(0), v[:seen].abs().mean(0)
            assert ((got[r] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -23 * (length / 32 + 16)) * size + 2.0 ** -25 * v.abs().amax()).all()
            assert ((lse[r] - score).abs() <= -score * (D + 8) * 2.0 ** -24).all()


@GPU
@pytest.mark.parametrize("G,n,dtype,lengths", [(8, 1, torch.bfloat16, [131001, 70000]), (2, 2, torch.float16, [131001, 5, 40000]), (2, 20, torch.bfloat16, [100003]), (1, 130, torch.float16, [60000, 131])])
def test_attention_of_very_long_contexts(G, n, dtype, lengths):
    pages, table = _cache(lengths, 1, 128, 128, n)
    _check_rows(pages, table, lengths, [min(n, length) for length in lengths], 1, G, 128, dtype)


def test_attention_reference_against_softmax():
    pages, table = _cache([20, 33], 2, 16, 64, 1)
    q, starts, ln = torch.randn(6, 4, 64).bfloat16(), torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([20, 33], dtype=torch.int32)
    o, lse = P.attention(q, pages, table, starts, ln, max_queries=3, return_lse=True)
    k, v = P.read(pages, table, ln, 33, torch.float32)
    for b, rows in ((0, [0, 1]), (1, [2, 3, 4])):
        for i, r in enumerate(rows):
            seen = int(ln[b]) - len(rows) + 1 + i
            for h in range(4):
                s = (k[b, :seen, h // 2] @ q[r, h].float()) / 8.0
                assert torch.allclose(o[r, h].float(), torch.softmax(s, 0) @ v[b, :seen, h // 2], atol=1e-2, rtol=1e-2)
                assert torch.allclose(lse[r, h], torch.logsumexp(s, 0), atol=1e-4)
    assert (o[5] == 0).all() and lse[5].eq(float("-inf")).all()


def test_refusals():
    pages = P.Pages.allocate(3, 2, 16, 64, device="cpu")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)                                            # noqa: E731
    k, q, slots = torch.zeros(4, 2, 64), torch.zeros(4, 4, 64).bfloat16(), torch.arange(4)
    ok = dict(max_queries=1)
    for bad in (
            lambda: P.Pages.allocate(1, 1, 24, 64, device="cpu"), lambda: P.Pages.allocate(1, 1, 16, 80, device="cpu"), lambda: P.Pages.allocate(1, 0, 16, 64, device="cpu"),
            lambda: P.plan(i32(2), i32(2), i32(2, 3), i32(4), i32(1), page_size=8, rows=0), lambda: P.plan(i32(2).long(), i32(2), i32(2, 3), i32(4), i32(1), page_size=16, rows=0),
            lambda: P.plan(i32(2), i32(3), i32(2, 3), i32(4), i32(1), page_size=16, rows=0), lambda: P.plan(i32(2), i32(2), i32(3, 2).T, i32(4), i32(1), page_size=16, rows=0),
            lambda: P.plan(i32(2), i32(2), i32(2, 3), i32(4), i32(2), page_size=16, rows=0), lambda: P.plan(i32(2), i32(2), i32(2, 3), i32(4), i32(1), page_size=16, rows=-1),
            lambda: P.release(i32(2), i32(2), i32(2, 3), i32(4), i32(1), page_size=16), lambda: P.release(i32(2), i32(3).bool(), i32(2, 3), i32(4), i32(1), page_size=16),
            lambda: P.store(k[:, :1], k[:, :1], pages, slots), lambda: P.store(k, k.half(), pages, slots), lambda: P.store(k, k, pages, slots[:3]),
            lambda: P.store(k.double(), k.double(), pages, slots), lambda: P.store(k, k, pages, slots.int()), lambda: P.store(k, k, pages, slots + 60),
            lambda: P.store(k.transpose(1, 2).contiguous().transpose(1, 2), k, pages, slots), lambda: P.store(k, k, pages, torch.tensor([0, 5, 1, 2])),
            lambda: P.store(k, k, pages._replace(k=pages.k.half()), slots), lambda: P.store(k, k, pages._replace(k_scale=pages.k_scale[:2]), slots),
            lambda: P.read(pages, i32(2, 3), i32(3), 4), lambda: P.read(pages, i32(2, 3), i32(2), 4, torch.float16), lambda: P.read(pages, i32(1, 1) + 3, i32(1) + 1, 4),
            lambda: P.attention(q.double(), pages, i32(2, 3), i32(3), i32(2), **ok), lambda: P.attention(q[:, :3], pages, i32(2, 3), i32(3), i32(2), **ok),
            lambda: P.attention(q[..., :32], pages, i32(2, 3), i32(3), i32(2), **ok), lambda: P.attention(q, pages, i32(2, 3), i32(2), i32(2), **ok),
            lambda: P.attention(q, pages, i32(2, 3), i32(3), i32(2), max_queries=0), lambda: P.attention(q, pages, i32(2, 3), i32(3), i32(2), scale=float("nan"), **ok),
            lambda: P.attention(q, pages, i32(2, 3), i32(3), i32(2), out=q.half(), **ok), lambda: P.attention(q.requires_grad_(True), pages, i32(2, 3), i32(3), i32(2), **ok)):
        with pytest.raises(ValueError):
            bad()


@GPU
def test_host_tensors_are_refused_on_the_gpu():
    pages = P.Pages.allocate(3, 2, 16, 64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")                            # noqa: E731
    k, q, slots = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 4, 64, device="cuda").bfloat16(), torch.arange(4)
    for bad in (lambda: P.plan(i32(2), i32(2).cpu(), i32(2, 3), i32(4), i32(1), page_size=16, rows=2), lambda: P.store(k, k, pages, slots),
                lambda: P.read(pages, i32(2, 3).cpu(), i32(2), 4), lambda: P.attention(q, pages, i32(2, 3), i32(3).cpu(), i32(2), max_queries=1),
                lambda: P.attention(q, pages._replace(v_scale=pages.v_scale.cpu()), i32(2, 3), i32(3), i32(2), max_queries=1)):
        with pytest.raises(ValueError, match="host"):
            bad()
