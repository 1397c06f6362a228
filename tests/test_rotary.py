"""Rotary positions: the CPU statement against complex arithmetic in 64 bits, gradients against differences, refusals; the kernel against
the formula in 64 bits at odd sizes, strides and far positions.

Tolerance of the kernel: an output is a c - b s in fp32 from a sine and a cosine that are 2^-22 off at most (the fraction of a turn is rounded to
fp32, 2^-26 turns, and sincospif is within 2 units in the last place), rounded once: half a step of the type times |y| + 2^-21 (|a| + |b|).  Where |y| is below the type's smallest
normal number N, steps no longer shrink with it: they are eps N apart (fp16 2^-24), so half of that, eps / 2 N, is added."""
import math

import pytest
import torch

from spiraltorch_b200.ops import elementwise as E
from spiraltorch_b200.ops import rotary as R

GPU = pytest.mark.gpu


def _complex(x, pos, freq, inter, magnitude=1.0, sign=1):
    n, y = freq.numel(), x.double().clone()
    turn = torch.polar(torch.tensor(magnitude, dtype=torch.float64), sign * pos.double()[..., None] * freq)[..., None, :]
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if inter else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., ia].double(), x[..., ib].double()) * turn
    y[..., ia], y[..., ib] = z.real, z.imag
    return y


def _allowed(x, y, n, inter, dtype):
    half = torch.finfo(dtype).eps / 2
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if inter else (slice(0, n), slice(n, 2 * n))
    size = torch.zeros_like(y)
    both = x[..., ia].double().abs() + x[..., ib].double().abs()
    size[..., ia], size[..., ib] = both, both
    return half * (y.abs() + torch.finfo(dtype).smallest_normal) + 2.0 ** -21 * size


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot", [2, 20, 64])
def test_reference_is_a_rotation(inter, rot):
    g = torch.Generator().manual_seed(1)
    x, pos = torch.randn(5, 3, 64, generator=g, dtype=torch.float64), torch.tensor([0, 1, 77, 100003, -4])
    f = R.frequencies(rot)
    assert torch.allclose(R.rotary(x, None, pos, f, interleaved=inter)[0], _complex(x, pos, f, inter), atol=1e-12)
    y = R.rotary(x, None, pos, f, interleaved=inter, magnitude=0.5)[0]
    back = R.rotary_(y.clone(), None, pos, f, interleaved=inter, magnitude=2.0, backward=True)[0]
    assert torch.allclose(back[..., :rot], x[..., :rot], atol=1e-12)
    assert torch.equal(y[..., rot:], x[..., rot:])


def test_agrees_with_the_training_form():
    x = torch.randn(12, 4, 64)
    cos, sin = E.rope_tables(6, 64, 10000.0, x.device)
    want = E.rope_reference(x, cos, sin, 6, False)
    got = R.rotary(x, None, torch.arange(12) % 6, R.frequencies(64))[0]
    assert torch.allclose(got, want, atol=1e-6)


def test_scalings():
    f, r = R.frequencies(64), 64
    assert torch.allclose(R.frequencies(r, scaling=R.Scaling("linear", 4.0)), f / 4)
    b = R.frequencies(r, scaling=R.Scaling("base", 4.0))
    assert b[0] == f[0] and math.isclose(float(b[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    s = R.Scaling("bands", 4.0, original=2048, low=1.0, high=32.0)
    b, turns = R.frequencies(r, scaling=s), 2048 * f / (2 * math.pi)
    assert torch.equal(b[turns >= 32], f[turns >= 32]) and torch.allclose(b[turns <= 1], f[turns <= 1] / 4)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (b[between] < f[between]).all() and (b[between] > f[between] / 4).all()


def test_gradients_against_differences():
    q, k = (torch.randn(3, h, 10, dtype=torch.float64, requires_grad=True) for h in (4, 2))
    pos, f = torch.tensor([0, 3, 900]), R.frequencies(6)
    for inter in (False, True):
        fn = lambda a, b: R.rotary(a, b, pos, f, interleaved=inter, magnitude=1.3)               # noqa: E731
        assert torch.autograd.gradcheck(fn, (q, k))
        assert torch.autograd.gradgradcheck(fn, (q, k))
    # one output or input alone
    only = torch.autograd.grad(R.rotary(q, k, pos, f)[1].sum(), k)[0]
    assert torch.allclose(only, R.rotary(torch.ones_like(k), None, -pos, f)[0])
    assert torch.autograd.grad(R.rotary(q.detach(), k, pos, f)[1].sum(), k)[0].shape == k.shape


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("inter", [False, True])
def test_tangents(device, inter):
    """The map is linear: a tangent is rotated as its tensor is."""
    import torch.autograd.forward_ad as fw
    g = torch.Generator().manual_seed(3)
    q, k, tq, tk = (torch.randn(5, h, 64, generator=g).to(device) for h in (4, 2, 4, 2))
    pos, f = torch.tensor([0, 3, 900, 5, 7], device=device), R.frequencies(32).to(device)
    call = lambda a, b: R.rotary(a, b, pos, f, interleaved=inter, magnitude=1.25)                # noqa: E731
    value, want = call(q, k), call(tq, tk)
    with fw.dual_level():
        for grad in (False, True):
            a, b = (fw.make_dual(x.clone().requires_grad_(grad), t) for x, t in ((q, tq), (k, tk)))
            for got, v, w in zip(call(a, b), value, want):
                assert torch.equal(fw.unpack_dual(got).tangent, w) and torch.equal(fw.unpack_dual(got).primal, v)
            only = call(q, b)
            assert torch.equal(fw.unpack_dual(only[1]).tangent, want[1])
            assert (t := fw.unpack_dual(only[0]).tangent) is None or (t == 0).all()
            assert torch.equal(fw.unpack_dual(call(a, None)[0]).tangent, want[0])
            wide = tq[..., :1].expand_as(tq)
            assert torch.equal(fw.unpack_dual(call(fw.make_dual(q.clone(), wide), k)[0]).tangent, call(wide.contiguous(), None)[0])
            plain = call(q, k)
            assert torch.equal(plain[0], value[0]) and fw.unpack_dual(plain[0]).tangent is None
        with pytest.raises(ValueError, match="tangent"):
            R.rotary_(fw.make_dual(q.clone(), tq), None, pos, f)
        with pytest.raises(ValueError, match="tangent"):
            R.rotary_(q.clone(), fw.make_dual(k.clone(), tk), pos, f)
        R.rotary_(q.clone(), k.clone(), pos, f)
        # over a gradient: of sum(rotated * w) along a tangent of w
        a = q.clone().requires_grad_(True)
        got = torch.autograd.grad((R.rotary(a, None, pos, f, interleaved=inter)[0] * fw.make_dual(q, tq)).sum(), a)[0]
        assert torch.equal(fw.unpack_dual(got).tangent, R.rotary_(tq.clone(), None, pos, f, interleaved=inter, backward=True)[0])


def test_refusals():
    q, k, pos, f = torch.randn(4, 2, 16), torch.randn(4, 1, 16), torch.arange(4), R.frequencies(16)
    for bad in (lambda: R.rotary(q.to(torch.int32), k, pos, f), lambda: R.rotary(q, k, pos[:3], f), lambda: R.rotary(q, k, pos.float(), f),
                lambda: R.rotary(q, k.half(), pos, f), lambda: R.rotary(q, k[:3], pos, f), lambda: R.rotary(q, k[..., :8], pos, f),
                lambda: R.rotary(q, k, pos, f.float()), lambda: R.rotary(q, k, pos, R.frequencies(18)), lambda: R.rotary(q, k, pos, f[:0]),
                lambda: R.rotary_(q.requires_grad_(True), k, pos, f), lambda: R.frequencies(7), lambda: R.frequencies(8, base=-1.0),
                lambda: R.Scaling("other", 2.0), lambda: R.Scaling("linear", 0.0), lambda: R.Scaling("bands", 2.0, low=3.0, high=3.0)):
        with pytest.raises(ValueError):
            bad()


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,h,hk,dim,rot,inter", [
    (1, 1, 1, 64, 64, False), (1, 32, 8, 128, 128, True), (7, 3, 1, 128, 32, False), (64, 12, 12, 64, 32, True), (129, 5, 5, 128, 116, False),
    (33, 4, 2, 96, 52, True), (5, 2, 2, 10, 6, False), (3, 2, 1, 7, 2, True), (1000, 16, 16, 128, 128, False), (4097, 7, 1, 64, 64, True)])
def test_kernel(dtype, rows, h, hk, dim, rot, inter):
    g = torch.Generator().manual_seed(rows)
    q, k, dq, dk = (torch.randn(rows, n, dim, generator=g).to(dtype) for n in (h, hk, h, hk))
    pos = torch.randint(0, 1 << 20, (rows,), generator=g)
    pos[0] = (1 << 20) - 1
    f = R.frequencies(rot)
    for p in (pos, pos.int()):
        a, b = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
        out = R.rotary(a, b, p.cuda(), f.cuda(), interleaved=inter, magnitude=1.25)
        grads = torch.autograd.grad(out, (a, b), (dq.cuda(), dk.cuda()))
        for got, x, sign in ((out[0], q, 1), (out[1], k, 1), (grads[0], dq, -1), (grads[1], dk, -1)):
            want = _complex(x, pos, f, inter, 1.25, sign)
            off = (got.detach().cpu().double() - want).abs()
            assert (off <= _allowed(x * 1.25, want, f.numel(), inter, dtype)).all(), off.max()
            assert torch.equal(got[..., rot:].cpu(), x[..., rot:])


@GPU
def test_kernel_angles_in_fp32():
    """Heads of (1, 0) give cosine and sine themselves: sincospif is within a unit in the last place of its argument's, 2^-24 at most, what its argument
    lacks of the angle is added with one more rounding, 2^-25, and angles are exact to 2^-30."""
    f, pos = R.frequencies(128), torch.randint(0, 1 << 20, (20000,), generator=torch.Generator().manual_seed(2))
    x = torch.zeros(20000, 1, 128)
    x[..., :64] = 1.0
    got = R.rotary(x.cuda(), None, pos.cuda(), f.cuda())[0].cpu().double()[:, 0]
    angle = pos.double()[:, None] * f
    off = (got - torch.cat([angle.cos(), angle.sin()], -1)).abs().max()
    assert off <= 1.5 * 2.0 ** -24 + 2.0 ** -30, off * 2.0 ** 24


@GPU
@pytest.mark.parametrize("half", [776, 1016, 1544, 2040, 2048])
@pytest.mark.parametrize("inter", [False, True])
def test_kernel_of_one_wide_head(half, inter):
    """Several tokens' angles of a block pass 48 KB of shared memory; and the widest head."""
    g = torch.Generator().manual_seed(half)
    rows, f = 2500, R.frequencies(2 * half)
    x, pos = torch.randn(rows, 1, 2 * half + 16, generator=g).bfloat16(), torch.randint(0, 1 << 20, (rows,), generator=g)
    want = _complex(x, pos, f, inter)
    got = R.rotary(x.cuda(), None, pos.cuda(), f.cuda(), interleaved=inter)[0].cpu()
    assert ((got.double() - want).abs() <= _allowed(x, want, half, inter, x.dtype)).all()
    assert torch.equal(R.rotary_(x.cuda(), None, pos.cuda(), f.cuda(), interleaved=inter)[0].cpu(), got)


@GPU
def test_views_in_place_and_without_keys():
    rows, h, hk, D = 37, 6, 2, 128
    fused = torch.randn(rows, (h + 2 * hk) * D + 8, device="cuda").bfloat16()
    before = fused.clone()
    q, k = fused[:, :h * D].view(rows, h, D), fused[:, h * D:(h + hk) * D].view(rows, hk, D)
    pos, f = torch.arange(rows, device="cuda") * 1000, R.frequencies(D).cuda()
    want = R.rotary(q.clone(), k.clone(), pos, f)
    R.rotary_(q, k, pos, f)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, (h + hk) * D:], before[:, (h + hk) * D:])
    assert torch.equal(R.rotary(before[:, :h * D].view(rows, h, D), None, pos, f)[0], want[0])
    # leading dimensions, a transposed view, rows that start off a 16-byte boundary
    x = torch.randn(2, 5, h, D, device="cuda").bfloat16()
    p2 = torch.arange(10, device="cuda").view(2, 5)
    flat = R.rotary(x.view(10, h, D), None, p2.view(-1), f)[0]
    assert torch.equal(R.rotary(x, None, p2, f)[0], flat.view_as(x))
    assert torch.equal(R.rotary(x.transpose(0, 1), None, p2.T, f)[0], flat.view_as(x).transpose(0, 1))
    odd = torch.empty(10 * h * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(10, h, D).copy_(x.view(10, h, D))
    assert torch.equal(R.rotary(odd, None, p2.view(-1), f)[0], flat)
    assert R.rotary(x[:0], None, p2[:0], f)[0].shape == (0, 5, h, D)
    with pytest.raises(ValueError, match="host"):
        R.rotary(x, None, p2.cpu(), f)


@GPU
def test_captured_backward_beside_an_eager_one():
    q = torch.randn(9, 4, 64, device="cuda").bfloat16().requires_grad_(True)
    pos, f, dy = torch.arange(9, device="cuda"), R.frequencies(64).cuda(), torch.randn(9, 4, 64, device="cuda").bfloat16()
    want = torch.autograd.grad(R.rotary(q, None, pos, f)[0], q, dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = q.detach().clone().requires_grad_(True)
        torch.autograd.grad(R.rotary(leaf, None, pos, f)[0], leaf, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(R.rotary(leaf, None, pos, f)[0], leaf, dy)[0]
    graph.replay()
    assert torch.equal(got, want)
    pos.add_(5)
    graph.replay()
    assert torch.equal(got, torch.autograd.grad(R.rotary(q, None, pos, f)[0], q, dy)[0])
