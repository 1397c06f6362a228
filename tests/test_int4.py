"""Weights of four bits: quantising against the definition element by element in 64 bits, products against 64 bits at odd sizes, strides and types, gradients
against the formula and against differences, refusals.

Quantising is exact: codes, scales and what they stand for are compared for equality.  Tolerance of a product: the numbers that enter are exact, each of at
most in/16 + 40 additions that follow one another in fp32 (a matrix instruction's of 16 columns as one) is off by at most 2^-22 of the sum of magnitudes A = |x| |W|^T
(an instruction may cut off instead of rounding, and adds up 16 columns inside), and the result is rounded once, half a step.  An activation is 1-Lipschitz but for gelu's 1.13
and computes within 2^-20 of its argument."""
import math

import pytest
import torch

from spiraltorch_b200.ops import int4

GPU = pytest.mark.gpu
cuda = torch.device("cuda")


def _by_hand(w, group):
    """Codes and scales of a matrix by Python's own arithmetic."""
    from fractions import Fraction
    n, k = w.shape
    codes, scales = [], []
    for r in range(n):
        row, crow, srow = [Fraction(float(v)) for v in w[r]], [], []
        for i in range(0, k, group):
            part = row[i:i + group]
            far = max(part, key=lambda v: (abs(v), -v))      # the negative one of two
            size = abs(far) / 8
            if size:
                e = math.floor(math.log2(float(size)))
                unit = Fraction(2) ** (e - 3)
                while size / unit >= 16:
                    unit *= 2
                while size / unit < 8:
                    unit /= 2
                size = round(size / unit) * unit             # Python rounds ties to even
            size = min(max(size, Fraction(2) ** -20), Fraction(7680))
            s = -size if far > 0 else size
            srow.append(float(s))
            crow += [min(max(round(v / s), -8), 7) for v in part]
        codes.append(crow)
        scales.append(srow)
    return torch.tensor(codes, dtype=torch.int8), torch.tensor(scales, dtype=torch.float32)


def _matrix(n, k, dtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    return w.to(dtype).to(device)


def _hard(group):
    """Rows of borders: all zero, ties of codes and scales, equal extrema of both signs, tiny, huge and subnormal elements."""
    rows = []
    for s in (0.5, 9 * 2.0 ** -7, 15 * 2.0 ** -6, -11 * 2.0 ** -5):
        rows.append(torch.tensor([s * (i % 17 - 8) / 1.0 * 0.5 for i in range(group)] + [s * (i % 16 - 8 + 0.5) for i in range(group)]))
    rows += [torch.zeros(2 * group), torch.cat([torch.full((group,), 3.0), torch.full((group,), -3.0)]),
             torch.tensor([3.0, -3.0] * group), torch.full((2 * group,), 2.0 ** -24), torch.tensor([1e5, -1.0] * group), torch.tensor([-7e4, 5e4] * group)]
    for m in (8.5, 9.5, 15.5, 15.75, 8.0, 17.0):      # scales on and beside a tie of 4 bits
        rows.append(torch.tensor([m, -m / 2] * group) * 2.0 ** -3)
        rows.append(torch.tensor([-m * (1 + 2.0 ** -23), m / 3] * group))
    return torch.stack(rows)


@pytest.mark.parametrize("group", int4.GROUPS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (17, 65), (16, 128), (5, 200)])
def test_quantize_statement_is_the_definition(shape, group):
    w = _matrix(*shape, torch.float32)
    codes, scales = _by_hand(w, group)
    q, s = int4.quantize_reference(w, group)
    assert torch.equal(q, codes) and torch.equal(s, scales)
    held = int4.quantize(w, group)
    want = codes.double() * scales.double().repeat_interleave(group, 1)[:, :shape[1]]
    for t in (torch.float64, torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(int4.dequantize(held, t).double(), want)


@pytest.mark.parametrize("group", int4.GROUPS)
def test_quantize_statement_at_borders(group):
    w = _hard(group)
    codes, scales = _by_hand(w, group)
    q, s = int4.quantize_reference(w, group)
    assert torch.equal(q, codes) and torch.equal(s, scales)


def test_quantize_error_bound_and_non_finite():
    w = _matrix(64, 256, torch.float32, 3)
    held = int4.quantize(w, 64)
    s = int4._row_scales(held).abs().repeat_interleave(64, 1)
    assert ((int4.dequantize(held, torch.float32) - w).abs() <= 1.5 * s).all()      # half a step, and a step where the side of the extremum's opposite ends at 7
    for bad in (math.nan, math.inf, -math.inf):
        v = w.clone()
        v[5, 70] = bad
        d = int4.dequantize(int4.quantize(v, 64), torch.float32)
        assert d[5, 64:128].isnan().all() and d.isnan().sum() == 64


def test_tiles_are_in_the_order_of_the_matrix_instruction():
    q = torch.randint(-8, 8, (33, 130), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    tiles = int4._tiles(q)
    assert tiles.shape == (3, 3, 512) and torch.equal(int4._untile(tiles, 33, 130), q)
    word = tiles.view(torch.int32)[1, 1].view(32, 4)
    for lane in range(32):
        for s in range(4):
            for e in range(4):
                r, k = 16 + lane // 4 + 8 * (e & 1), 64 + 16 * s + 2 * (lane % 4) + 8 * (e >> 1)
                assert (int(word[lane, s]) >> (4 * e) & 15) - 8 == q[r, k] and (int(word[lane, s]) >> (4 * e + 16) & 15) - 8 == q[r, k + 1]


def test_linear_statement_and_gradients():
    g = torch.Generator().manual_seed(2)
    held = int4.quantize(_matrix(7, 45, torch.float32), 32)
    w = int4.dequantize(held, torch.float64)
    x, b, r = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((2, 3, 45), (7,), (2, 3, 7)))
    y = int4.linear(x, held, b, residual=r)
    assert torch.allclose(y, x @ w.T + b + r, atol=1e-12)
    dy = torch.randn(y.shape, generator=g, dtype=torch.float64)
    dx, db, dr = torch.autograd.grad(y, (x, b, r), dy)
    assert torch.allclose(dx, dy @ w, atol=1e-12) and torch.allclose(db, dy.sum((0, 1)), atol=1e-12) and torch.equal(dr, dy)
    assert torch.autograd.gradcheck(lambda x, b, r: int4.linear(x, held, b, residual=r), (x, b, r))
    assert torch.autograd.gradgradcheck(lambda x: int4.linear(x, held) ** 2, (x,))
    with torch.no_grad():
        assert torch.equal(int4.linear(x, held, act="relu"), torch.relu(x @ w.T))
        assert torch.allclose(int4.linear(x, held, b, act="gelu", residual=r), torch.nn.functional.gelu(x @ w.T + b, approximate="tanh") + r, atol=1e-12)
        assert int4.linear(x[0, 0], held).shape == (7,) and int4.linear(x[:0], held).shape == (0, 3, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_statement_under_autocast(dtype):
    """Sums stay in fp32, as the kernels' do."""
    held = int4.quantize(_matrix(7, 45, torch.float32), 32)
    x, b, dy = _matrix(3, 45, dtype, 1).requires_grad_(True), _matrix(1, 7, dtype, 2)[0], _matrix(3, 7, dtype, 3)
    want = int4.linear(x, held, b)
    dx = torch.autograd.grad(want, x, dy)[0]
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = int4.linear(x, held, b)
        assert torch.equal(y, want) and y.dtype == dtype
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx)
        with torch.no_grad():
            assert torch.equal(int4.linear(x, held, b), want)


def test_refusals():
    w = _matrix(20, 70, torch.float32)
    held = int4.quantize(w, 32)
    x = torch.randn(3, 70)
    for call in (lambda: int4.quantize(w, 48), lambda: int4.quantize(w[0]), lambda: int4.quantize(w.int()), lambda: int4.quantize(w, 64, out=held),
                 lambda: int4.quantize(w[:, :64], 32, out=held), lambda: int4.Weights.allocate(0, 4), lambda: int4.Weights.allocate(4, 4, 16),
                 lambda: int4.linear(x[:, :69], held), lambda: int4.linear(x, held, torch.zeros(21)), lambda: int4.linear(x, held, torch.zeros(20).half()),
                 lambda: int4.linear(x, held, residual=torch.zeros(2, 20)), lambda: int4.linear(x, held, act="tanh"), lambda: int4.linear(x.int(), held),
                 lambda: int4.Weights(held.codes, held.scales, 20, 140, 32), lambda: int4.Weights(held.codes, held.scales, 20, 70, 64),
                 lambda: int4.linear(x.clone().requires_grad_(), held, act="gelu"), lambda: int4.linear(torch.tensor(1.0), held),
                 lambda: int4.linear(x[:1].expand((1 << 30) + 1, 70), held)):
        with pytest.raises(ValueError):
            call()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError):
            int4.linear(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), held)


def test_weights_quantised_anew_are_no_gradient_of_the_old():
    held = int4.quantize(_matrix(7, 45, torch.float32), 32)
    x = torch.randn(3, 45, requires_grad=True)
    y = int4.linear(x, held)
    int4.quantize(_matrix(7, 45, torch.float32, 1), 32, out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_weights_quantised_anew_are_no_second_derivative_of_the_old():
    held = int4.quantize(_matrix(7, 45, torch.float32), 32)
    w = int4.dequantize(held, torch.float32)
    x, dy = torch.randn(3, 45, requires_grad=True), torch.randn(3, 7, requires_grad=True)
    dx = torch.autograd.grad(int4.linear(x, held), x, dy, create_graph=True)[0]
    again = torch.autograd.grad(dx.sum(), dy, retain_graph=True)[0]
    assert torch.allclose(again, torch.ones(3, 45) @ w.T, atol=1e-5)
    int4.quantize(_matrix(7, 45, torch.float32, 1), 32, out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(dx.sum(), dy)
    # other scales alone are other weights too
    y = int4.linear(x, held)
    held.scales.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def _check_weights_of_inference_mode(device, dtype):
    w, x = _matrix(7, 45, dtype, device=device), _matrix(3, 45, dtype, 1, device).requires_grad_(True)
    want = int4.linear(x, int4.quantize(w, 32))
    with torch.inference_mode():
        held = int4.quantize(w, 32)
        moved = held.to(device)
        assert torch.equal(int4.linear(x, held), want)
    for h in (held, moved):
        y = int4.linear(x, h)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(int4.linear(x, int4.quantize(w, 32)).sum(), x)[0])
    y = int4.linear(x, held)
    int4.quantize(w * 2, 32, out=held)
    assert torch.equal(int4.dequantize(held, dtype), 2 * int4.dequantize(int4.quantize(w, 32), dtype))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = int4.linear(x, held)
    with torch.inference_mode():
        int4.quantize(w, 32, out=held)
        parts = int4.Weights(held.codes.clone(), held.scales.clone(), 7, 45, 32)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert torch.equal(int4.linear(x.detach(), parts), want)
    with pytest.raises(ValueError, match="inference mode"):
        int4.linear(x, parts)


def test_weights_of_inference_mode():
    _check_weights_of_inference_mode("cpu", torch.float32)


@GPU
def test_weights_of_inference_mode_on_the_gpu():
    _check_weights_of_inference_mode("cuda", torch.bfloat16)


def test_weights_are_copied_saved_and_not_changed(tmp_path):
    import copy
    held = int4.quantize(_matrix(20, 70, torch.float32), 32)
    torch.save(held, tmp_path / "w")
    for other in (copy.deepcopy(held), torch.load(tmp_path / "w", weights_only=False), held.to("cpu")):
        assert torch.equal(int4.dequantize(other), int4.dequantize(held)) and other.nbytes == held.nbytes
    with pytest.raises(AttributeError):
        held.in_features = 69


# ---- kernels --------------------------------------------------------------------------------------------------------------------
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@GPU
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", int4.GROUPS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (16, 128), (17, 65), (37, 200), (130, 777), (64, 2048)])
def test_quantize_kernel(shape, group, dtype):
    w = _matrix(*shape, dtype)
    want = int4.quantize(w, group)
    got = int4.quantize(w.to(cuda), group)
    assert torch.equal(got.codes.cpu(), want.codes) and torch.equal(got.scales.cpu(), want.scales)
    for t in DTYPES:
        d = int4.dequantize(got, t)
        assert d.dtype == t and torch.equal(d.float().cpu(), int4.dequantize_reference(want))


@GPU
@pytest.mark.parametrize("group", int4.GROUPS)
def test_quantize_kernel_at_borders_and_strides(group):
    w = _hard(group)
    w[2, 3], w[4, 0], w[5, 1] = math.nan, math.inf, -math.inf
    codes, scales = int4.quantize_reference(w, group)
    got = int4.quantize(w.to(cuda), group)
    fine = torch.isfinite(scales)
    keep = fine.repeat_interleave(group, 1)
    assert torch.equal(int4._untile(got.codes.cpu(), *w.shape)[keep], codes[keep])
    s = int4._row_scales(got).cpu()
    assert torch.equal(s[fine], scales[fine]) and s[~fine].isnan().all()
    # a view at an odd place of a wider matrix, a transposed one, and memory that is written to again
    wide = torch.randn(50, 201, generator=torch.Generator().manual_seed(4)).to(cuda)
    for view in (wide[3:40, 5:190], wide[:, :200], wide.T, wide[:, ::2]):
        want = int4.quantize(view.cpu().contiguous(), group)
        got = int4.quantize(view, group)
        assert torch.equal(got.codes.cpu(), want.codes) and torch.equal(got.scales.cpu(), want.scales)
        again = int4.quantize(view * 2, group, out=got)
        assert again is got and torch.equal(int4.dequantize(got, torch.float32).cpu(), 2 * int4.dequantize(want, torch.float32))


def _allowed(x, w, y, dtype, act=None):
    a = x.abs() @ w.abs().T
    return torch.finfo(dtype).eps / 2 * (y.abs() + torch.finfo(dtype).smallest_normal) + 1.13 * (x.shape[1] / 16 + 40) * 2.0 ** -22 * (a + 1.0)


def _product_case(rows, n, k, group, dtype, bias, act, residual, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = int4.quantize(_matrix(n, k, torch.float32, seed).to(cuda) * 0.1, group)
    x = torch.randn(rows, k, generator=g).to(dtype).to(cuda)
    b = torch.randn(n, generator=g).to(dtype).to(cuda) if bias else None
    r = torch.randn(rows, n, generator=g).to(dtype).to(cuda) if residual else None
    w = int4.dequantize(held, torch.float32).double()
    y = x.double() @ w.T
    if bias:
        y = y + b.double()
    y = torch.relu(y) if act == "relu" else torch.nn.functional.gelu(y, approximate="tanh") if act == "gelu" else y
    if residual:
        y = y + r.double()
    return held, x, b, r, w, y


ROWS = [1, 2, 7, 8, 9, 16, 17, 33, 64, 100, 129, 300]


@GPU
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 64, 64), (37, 100, 32), (130, 129, 128), (300, 777, 64), (257, 2048, 128), (64, 4160, 32)])
def test_linear_kernel(rows, n, k, group):
    for dtype, bias, act, residual in ((torch.bfloat16, False, None, False), (torch.float16, True, "relu", True), (torch.bfloat16, True, "gelu", True)):
        held, x, b, r, w, y = _product_case(rows, n, k, group, dtype, bias, act, residual, rows + n)
        got = int4.linear(x, held, b, act=act, residual=r)
        assert got.dtype == dtype and got.shape == y.shape
        assert ((got.double() - y).abs() <= _allowed(x.double(), w, y, dtype)).all()


@GPU
@pytest.mark.parametrize("rows,n,k,group,act", [(1000, 4003, 300, 32, "gelu"), (190, 18900, 256, 64, None), (1, 9000, 2100, 64, "relu"), (7, 300, 17000, 128, "gelu"),
                                                (16, 20000, 1000, 128, None), (12, 48, 9000, 32, "relu"), (600, 16, 20000, 64, None)])
def test_linear_sizes_that_share_and_repeat_tiles(rows, n, k, group, act):
    """More tiles than SMs, tiles of 192 tokens, more rows of weights than blocks, clusters and stretches beyond their 8 blocks."""
    held, x, b, r, w, y = _product_case(rows, n, k, group, torch.bfloat16, True, act, True)
    got = int4.linear(x, held, b, act=act, residual=r)
    assert ((got.double() - y).abs() <= _allowed(x.double(), w, y, torch.bfloat16)).all()
    x.requires_grad_(True)
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(6)).to(x.dtype).to(cuda)
    want = dy.double() @ w
    got = torch.autograd.grad(int4.linear(x, held), x, dy)[0]
    assert ((got.double() - want).abs() <= _allowed(dy.double(), w.T, want, x.dtype)).all()


@GPU
@pytest.mark.parametrize("rows", [3, 20])
def test_linear_offsets_beyond_32_bits(rows):
    """Rows of x and of the residual 2^30 and 2^28 elements apart: their last ones lie behind 2^32 bytes."""
    held, x, b, r, w, y = _product_case(rows, 136, 200, 64, torch.bfloat16, True, None, True)
    step = 1 << (30 if rows == 3 else 28)
    memory = torch.empty((rows - 1) * step + 256, dtype=torch.bfloat16, device=cuda)
    far = memory.as_strided((rows, 200), (step, 1))
    far.copy_(x)
    assert torch.equal(int4.linear(far, held, b, residual=r), int4.linear(x, held, b, residual=r))
    far = memory.as_strided((rows, 136), (step, 1))
    far.copy_(r)
    assert torch.equal(int4.linear(x, held, b, residual=far), int4.linear(x, held, b, residual=r))


@GPU
@pytest.mark.parametrize("rows", [1, 5, 16, 40, 200])
def test_linear_views_and_places(rows):
    held, x, b, r, w, _ = _product_case(rows, 150, 328, 64, torch.bfloat16, True, None, True)
    for pad, at in ((0, 0), (8, 8), (3, 1), (2, 2), (7, 0)):
        wide = torch.full((rows, 328 + pad), math.nan, dtype=x.dtype, device=cuda)
        xv = wide[:, at:at + 328] if at + 328 <= wide.shape[1] else wide[:, :328]
        xv.copy_(x)
        rv = torch.zeros(rows, 150 + pad, dtype=x.dtype, device=cuda)[:, :150]
        rv.copy_(r)
        assert torch.equal(int4.linear(xv, held, b, residual=rv), int4.linear(x, held, b, residual=r))
    assert torch.equal(int4.linear(x.T.contiguous().T, held), int4.linear(x, held))
    assert torch.equal(int4.linear(x.view(rows, 1, 328), held), int4.linear(x, held).view(rows, 1, 150))
    one = x[:1].expand(rows, 328)
    assert torch.equal(int4.linear(one, held), int4.linear(one.contiguous(), held))
    assert torch.equal(int4.linear(x, held, b[:1].expand(150)), int4.linear(x, held, b[:1].expand(150).contiguous()))
    # memory around the result stays as it was, rows of zero tokens launch nothing
    assert int4.linear(x[:0], held).shape == (0, 150)


@GPU
@pytest.mark.parametrize("rows", [1, 12, 50, 200])
def test_linear_non_finite_values_stay_in_their_rows(rows):
    held, x, _, _, w, _ = _product_case(rows, 70, 200, 32, torch.bfloat16, False, None, False)
    base = int4.linear(x, held)
    x2 = x.clone()
    x2[0, 150] = math.nan
    got = int4.linear(x2, held)
    assert got[0].isnan().all() and torch.equal(got[1:], base[1:])
    v = w.float().clone()
    v[33, 40] = math.inf
    got = int4.linear(x, int4.quantize(v, 32))
    assert got[:, 33].isnan().all() and not got[:, :33].isnan().any() and not got[:, 34:].isnan().any()


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [20, 84, 200, 1000, 1230, 4050])      # half of the last 64 columns have no group of 32, where a warp's columns end with the row's or before
@pytest.mark.parametrize("rows", [1, 9, 16])
def test_linear_reads_the_scales_of_its_own_rows(rows, k, dtype):
    _, x, _, _, w, _ = _product_case(rows, 37, k, 32, dtype, False, None, False)
    held = int4.quantize(w.float(), 32)
    base = int4.linear(x, held)
    # an infinity at the beginning of a row is in no other row's scales
    v = w.float().clone()
    v[20, 0] = math.inf
    got = int4.linear(x, int4.quantize(v, 32))
    assert got[:, 20].isnan().all() and torch.equal(got[:, :20], base[:, :20]) and torch.equal(got[:, 21:], base[:, 21:])
    # what lies behind the last scales is not read
    memory = torch.full((held.scales.numel() + 512,), 0xFF, dtype=torch.uint8, device=cuda).repeat(2).view(torch.bfloat16)
    scales = memory[:held.scales.numel()].view(held.scales.shape)
    scales.copy_(held.scales)
    assert torch.equal(int4.linear(x, int4.Weights(held.codes, scales, 37, k, 32)), base)


@GPU
@pytest.mark.parametrize("group", int4.GROUPS)
@pytest.mark.parametrize("k", [64, 200, 4050])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17])
def test_linear_of_inputs_near_the_ends_of_the_type(rows, k, group):
    """Inputs up to the largest bf16 by weights that leave the product finite, however the codes are summed before they meet their scale; and products of
    few binary digits, which every order of sums gives exactly, down to 2^-126."""
    held, _, _, _, w, _ = _product_case(rows, 50, k, group, torch.bfloat16, False, None, False)
    held = int4.quantize((w * 1e-4).float(), group)
    w = int4.dequantize(held, torch.float32).double()
    x = torch.full((rows, k), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device=cuda)
    x[:, ::3] *= -1
    x[rows // 2:] = 3e37
    got = int4.linear(x, held)
    want = x.double() @ w.T
    a = x.double().abs() @ w.abs().T
    assert got.isfinite().all()
    assert ((got.double() - want).abs() <= torch.finfo(torch.bfloat16).eps / 2 * want.abs() + (k / 16 + 40) * 2.0 ** -22 * a).all()
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-8, 8, (50, k), generator=g).float()
    codes[:, ::32] = -8
    held = int4.quantize(codes.to(cuda), group)      # scales of 1
    x = torch.randint(-1, 2, (rows, k), generator=g).to(torch.bfloat16).to(cuda)
    x[:, 16:] = 0
    base = int4.linear(x, held)
    assert torch.equal(base.double(), x.double() @ codes.double().to(cuda).T)
    for e in (-100, -120, -126):
        assert torch.equal(int4.linear(x * 2.0 ** e, held), base * 2.0 ** e)


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,k,group", [(1, 16, 64, 64), (5, 37, 100, 32), (33, 300, 129, 128), (200, 130, 777, 64), (300, 520, 264, 32)])
def test_linear_gradients(rows, n, k, group, dtype):
    held, x, b, r, w, _ = _product_case(rows, n, k, group, dtype, True, None, True)
    for t in (x, b, r):
        t.requires_grad_(True)
    y = int4.linear(x, held, b, residual=r)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda)
    dx, db, dr = torch.autograd.grad(y, (x, b, r), dy)
    want = dy.double() @ w
    assert ((dx.double() - want).abs() <= _allowed(dy.double(), w.T, want, dtype)).all()
    assert torch.equal(dr, dy)
    want = dy.double().sum(0)
    assert ((db.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + rows * 2.0 ** -24 * dy.double().abs().sum(0)).all()
    # a gradient that is one number for all, and the input alone
    got = torch.autograd.grad(int4.linear(x, held).sum(), x)[0]
    want = torch.ones_like(dy).double() @ w
    assert ((got.double() - want).abs() <= _allowed(torch.ones_like(dy).double(), w.T, want, dtype)).all()


@GPU
def test_linear_streams_graphs_and_updates():
    held, x, b, r, w, _ = _product_case(9, 130, 512, 64, torch.bfloat16, True, None, True)
    want = int4.linear(x, held, b, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int4.linear(x, held, b, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int4.linear(x, held, b, act="gelu", residual=r)
    with torch.cuda.graph(other := torch.cuda.CUDAGraph()):      # two captured calls, in turns and at once
        z = int4.linear(torch.cat([x, x, x]), held, b)
    new = _matrix(130, 512, torch.bfloat16, 8, cuda)
    int4.quantize(new, 64, out=held)      # the replay multiplies by what the weights are now
    x.copy_(torch.randn_like(x))
    graph.replay()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other.replay()
    graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, int4.linear(x, held, b, act="gelu", residual=r))
    assert torch.equal(z, int4.linear(torch.cat([x, x, x]), held, b))


@GPU
@pytest.mark.parametrize("rows", [3, 27])
def test_the_first_call_of_a_process_may_be_captured(rows):
    """What the launchers set up at their first use does not end a capture."""
    import subprocess
    import sys
    from pathlib import Path
    code = f"""
import torch
from spiraltorch_b200.ops import int4
held = int4.quantize(torch.randn(256, 512, device="cuda", dtype=torch.bfloat16))
x = torch.randn({rows}, 512, device="cuda", dtype=torch.bfloat16)
with torch.cuda.graph(g := torch.cuda.CUDAGraph()):
    y = int4.linear(x, held)
g.replay()
assert torch.equal(y, int4.linear(x, held))
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(__file__).resolve().parents[1], timeout=300)


@GPU
def test_kernel_refusals():
    held = int4.quantize(torch.randn(20, 70, device=cuda), 32)
    x = torch.randn(3, 70, device=cuda)
    for call in (lambda: int4.linear(x, held), lambda: int4.linear(x.bfloat16().cpu(), held), lambda: int4.linear(x.bfloat16(), held, torch.zeros(20).bfloat16()),
                 lambda: int4.dequantize(held, torch.float64), lambda: int4.quantize(torch.randn(20, 70), 32, out=held), lambda: int4.linear(x.bfloat16(), held.to("cpu"))):
        with pytest.raises(ValueError):
            call()


# ---- where the framework uses them ------------------------------------------------------------------------------------------------
def _small_model(device="cpu", dtype=torch.float32):
    from spiraltorch_b200.models.gpt import GPTConfig, GPTModel
    return GPTModel(GPTConfig(vocab_size=96, d_model=128, n_layers=2, n_heads=2, ffn=256, seq_len=256, init_std=0.08), device=device, dtype=dtype)


def _with_quantised(model, head):
    """The same model, its matrices replaced by what four bits stand for."""
    for name, p in model.p.items():
        if p.dim() == 2 and (head or name != "embed.weight"):
            p.data.copy_(int4.dequantize(int4.quantize(p, 64), p.dtype))
    return model


@pytest.mark.parametrize("head", [False, True])
def test_decoder_with_four_bit_weights(head):
    """Equal, but for the order of sums, to a decoder of the model whose weights are what the four bits stand for (with a head of 16 bits the embedding stays)."""
    prompts = [[1, 2, 3], [7], list(range(30))]
    d = _small_model().decoder(3, 64, weight_bits=4, head_bits=4 if head else 16)
    assert len(d.weights) == 8 + head
    plain = _with_quantised(_small_model(), False)
    e = plain.decoder(3, 64)
    got, want = d.extend(prompts), e.extend(prompts)
    if head:      # the embedding of the tokens stays in 16 bits, the product with it does not
        assert not torch.allclose(got, want, atol=1e-4) and torch.nn.functional.cosine_similarity(got, want).min() > 0.97
    else:
        assert torch.allclose(got, want, atol=1e-4)
    for p, q in zip(d.model.p.values(), plain.p.values()):      # an update of the model, and the four bits made anew
        p.data.mul_(0.5)
        q.data.mul_(0.5)
    d.refresh()
    one = torch.tensor([4, 5, 6])
    if not head:
        assert torch.allclose(d.step(one), e.step(one), atol=1e-4)
    with pytest.raises(ValueError, match="4 or 16"):
        _small_model().decoder(1, 8, weight_bits=8)


def test_generate_with_four_bit_weights():
    model = _small_model()
    assert model.generate([[1, 2, 3], [9]], 5, weight_bits=4) == _with_quantised(_small_model(), False).generate([[1, 2, 3], [9]], 5)


def test_generate_with_groups_of_another_size():
    model, prompts = _small_model(), [[1, 2, 3], [9]]
    for group in (32, 128):
        d = model.decoder(2, 16, weight_bits=4, head_bits=4, group=group)
        assert all(w.group == group for w in d.weights.values())
        tokens, scores = model.generate(prompts, 5, weight_bits=4, head_bits=4, group=group, scores=0)
        want, judged = d.generate(prompts, 5, scores=0)
        assert tokens == want and [s.logprob for s in scores] == [s.logprob for s in judged]
    with pytest.raises(ValueError, match="groups"):
        model.generate(prompts, 2, weight_bits=4, group=48)


def test_frozen_layers_in_four_bits_train_their_adapters():
    from spiraltorch_b200 import hf_study as H
    torch.manual_seed(0)
    model = H.ByteCausalLM(d_model=32, n_layer=1, n_head=2, max_len=16)
    dense = model.blocks[0].attn.qkv.weight.detach().clone()
    H.inject_lora(model, ["attn.qkv", "mlp.out"], rank=2, base_bits=4, group=32)
    layer = model.blocks[0].attn.qkv
    with torch.no_grad():
        layer.lora_b.normal_()
    w = int4.dequantize(int4.quantize(dense, 32), torch.float32)
    x = torch.randn(3, 32, requires_grad=True)
    y = layer(x)
    want = x @ (w.t() + layer.merged_delta()) + layer.base.bias
    assert torch.allclose(y, want, atol=1e-5)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, (x, layer.lora_a, layer.lora_b), dy, retain_graph=True)
    ref = torch.autograd.grad(want, (x, layer.lora_a, layer.lora_b), dy)
    assert all(torch.allclose(a, b, atol=1e-5) for a, b in zip(got, ref))
    assert [n for n, p in model.named_parameters() if p.requires_grad] == [f"blocks.0.{m}.lora_{s}" for m in ("attn.qkv", "mlp.out") for s in "ab"]
    state = model.state_dict()
    other = H.ByteCausalLM(d_model=32, n_layer=1, n_head=2, max_len=16)
    H.inject_lora(other, ["attn.qkv", "mlp.out"], rank=2, base_bits=4, group=32)
    other.load_state_dict(state)
    ids = torch.randint(0, 256, (2, 16))
    assert torch.equal(other(ids), model(ids))
    assert torch.equal(layer.base.double().held().scales, layer.base.held().scales)      # a cast leaves the scales' bits
    with pytest.raises(H.StudyError, match="4 or 16"):
        H.inject_lora(H.ByteCausalLM(d_model=32, n_layer=1, n_head=2), ["attn.qkv"], rank=2, base_bits=8)


def test_a_study_run_with_frozen_layers_in_four_bits(tmp_path):
    from spiraltorch_b200 import hf_study as H
    out = H.lora_finetune_run({"steps": 2, "batch_size": 2, "seq_len": 16, "model": {"d_model": 32, "n_layer": 1, "n_head": 2}, "eval_batches": 1, "base_bits": 4}, tmp_path)
    assert out["steps"] == 2 and math.isfinite(out["eval_loss_after"])


@GPU
def test_decoder_with_four_bit_weights_on_the_gpu():
    """A whole run: prompts, steps, a captured step, an update and its replay, against the model whose weights are what the four bits stand for.  Both round the same
    products to bf16 and sum them in other orders, so a layer's input may differ by a bf16 step here and there; the logits' directions agree."""
    model = _small_model("cuda", torch.bfloat16)
    plain = _with_quantised(_small_model("cuda", torch.bfloat16), False)
    d, e = model.decoder(3, 128, weight_bits=4), plain.decoder(3, 128)
    prompts = [[1, 2, 3], [7], list(range(60))]

    def close(a, b):
        assert torch.nn.functional.cosine_similarity(a.float(), b.float()).min() > 0.999

    close(d.extend(prompts), e.extend(prompts))
    tokens = torch.tensor([4, 5, 6], device="cuda")
    close(d.step(tokens), e.step(tokens))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = d.step(tokens)
    for p, q in zip(model.p.values(), plain.p.values()):
        p.data.mul_(0.5)
        q.data.mul_(0.5)
    d.refresh()
    graph.replay()
    close(logits, e.step(tokens))
    big = _small_model("cuda", torch.bfloat16)
    tokens, scores = big.generate(prompts, 4, weight_bits=4, head_bits=4, scores=3)
    assert [len(t) for t in tokens] == [4, 4, 4]
    for t, s in zip(tokens, scores):
        assert [row[0] for row in s.top_ids] == t and s.logprob == [row[0] for row in s.top_logprobs] and all(x >= 0 for x in s.entropy)


@GPU
def test_frozen_layers_in_four_bits_on_the_gpu():
    from spiraltorch_b200 import hf_study as H
    torch.manual_seed(0)
    layer = torch.nn.Linear(200, 136).to(cuda, torch.bfloat16)
    w = int4.dequantize(int4.quantize(layer.weight.detach(), 64), torch.float32).double()
    wrapped = H.LoraWrapped(layer, 4, 8.0, base_bits=4)
    x = torch.randn(2, 30, 200, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    y = wrapped.base(x)
    dy = torch.randn_like(y)
    dx = torch.autograd.grad(y, x, dy)[0]
    want = dy.double() @ w
    assert ((dx.double() - want).abs().view(60, 200) <= _allowed(dy.double().view(60, 136), w.T, want.view(60, 200), torch.bfloat16)).all()
    wrapped(x).sum().backward()
    assert wrapped.lora_b.grad.isfinite().all() and x.grad.isfinite().all()


def _check_frozen_layer_under_autocast(device, dtype):
    from spiraltorch_b200 import hf_study as H
    torch.manual_seed(0)
    layer = torch.nn.Linear(45, 24).to(device)
    frozen = H.FrozenLinear4(layer, 32)
    for x in (torch.randn(3, 45, device=device), torch.randn(3, 45, device=device, dtype=dtype)):
        with torch.autocast(device, dtype=dtype):
            y = frozen(x.requires_grad_())
            assert y.dtype == layer(x).dtype == dtype
        assert torch.equal(y, int4.linear(x.to(dtype), frozen.held(), layer.bias.to(dtype)))
        assert torch.autograd.grad(y.sum(), x)[0].dtype == x.dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_frozen_layers_in_four_bits_under_autocast(dtype):
    _check_frozen_layer_under_autocast("cpu", dtype)


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_frozen_layers_in_four_bits_under_autocast_on_the_gpu(dtype):
    _check_frozen_layer_under_autocast("cuda", dtype)


@GPU
@pytest.mark.parametrize("rows", [5, 40])
def test_frozen_layers_in_four_bits_of_fp32_models_on_the_gpu(rows):
    """The product of the rounded activations, within its tolerance; their gradient, that of the rounded output's."""
    from spiraltorch_b200 import hf_study as H
    torch.manual_seed(0)
    layer = torch.nn.Linear(200, 136).to(cuda)
    frozen = H.FrozenLinear4(layer)
    w = int4.dequantize(frozen.held(), torch.float32).double()
    x = torch.randn(rows, 200, device=cuda, requires_grad=True)
    y = frozen(x)
    xb = x.detach().bfloat16().double()
    want = xb @ w.T + layer.bias.detach().bfloat16().double()
    assert y.dtype == torch.float32 and ((y.double() - want).abs() <= _allowed(xb, w, want, torch.bfloat16)).all()
    dy = torch.randn_like(y)
    dx = torch.autograd.grad(y, x, dy)[0]
    db = dy.bfloat16().double()
    assert dx.dtype == torch.float32 and ((dx.double() - db @ w).abs() <= _allowed(db, w.T, db @ w, torch.bfloat16)).all()


@GPU
def test_a_study_run_with_frozen_layers_in_four_bits_on_the_gpu(tmp_path):
    from spiraltorch_b200 import hf_study as H
    out = H.lora_finetune_run({"steps": 2, "batch_size": 2, "seq_len": 16, "model": {"d_model": 32, "n_layer": 1, "n_head": 2}, "eval_batches": 1, "pretrain_steps": 1,
                               "base_bits": 4, "device": "cuda"}, tmp_path)
    assert out["steps"] == 2 and math.isfinite(out["eval_loss_after"])
