"""GPU: layer norm and gated unit at sizes where a launch of a thread or more an element does not take them, and other limits."""
import math

import pytest
import torch

from test_gpu_features import check_gated, half

pytestmark = pytest.mark.gpu


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device='cuda').normal_(generator=g) * scale


def test_layer_norm_gradients_of_more_columns_than_a_launch_takes():
    """Two rows of 2^28 columns and a few: weight and bias gradients on both sides of the borders between launches."""
    from bayesian_optimization_amd import features
    cols = (1 << 28) + 67
    x, dy = rand((2, cols), torch.bfloat16, 1), rand((2, cols), torch.bfloat16, 2)
    y, mean, rstd = features.layer_norm(x)
    dx, dw, db = features.layer_norm_backward(dy, x, None, mean, rstd)
    for lo in range(0, cols, 1 << 26):
        at = slice(lo, min(cols, lo + (1 << 26)))
        d, xh = dy[:, at].double(), (x[:, at].double() - mean.double()[:, None]) * rstd.double()[:, None]
        for got, terms in ((dw, d * xh), (db, d)):
            want = terms.sum(0)      # three roundings a term and one of the sum in 32 bits, half a step of bfloat16 at the end
            assert bool(((got[at].double() - want).abs() <= 5 * 2.0 ** -24 * terms.abs().sum(0) + 2.0 ** -8 * 1.01 * want.abs()).all()), lo
    assert bool(torch.isfinite(dx).all())


@pytest.mark.parametrize('dtype,rows,cols,hidden', [
    (torch.bfloat16, (1 << 30) + 70, 1, 1),            # 2^24 tiles of 64 rows and more, in both directions
    (torch.float32, (1 << 29) + 37, 1, 1),             # the kernels for few hidden units
    (torch.float16, (1 << 27) + 100, 3, 2),            # rows packed into the workspace in pieces: a short contraction,
    (torch.bfloat16, (1 << 23) + 5000000, 257, 2),     # and a longer one
    (torch.bfloat16, 3, 1, (1 << 26) + 5)])            # hidden units, a wave each
def test_gated_unit_of_more_than_a_launch_takes(dtype, rows, cols, hidden):
    from bayesian_optimization_amd import features
    U, H = 2.0 ** -24, torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    x, dh = rand((rows, cols), dtype, 3), rand((rows, hidden), dtype, 4)
    wg, wu = rand((hidden, cols), dtype, 5, cols ** -0.5), rand((hidden, cols), dtype, 6, cols ** -0.5)
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    dx, dwg, dwu = features.gated_unit_backward(dh, x, wg, wu, kept)
    wgd, wud = wg.double(), wu.double()
    sums = [torch.zeros(hidden, cols, dtype=torch.float64, device='cuda') for _ in range(4)]
    step = max(1, (1 << 27) // (cols + hidden))
    for lo in range(0, rows, step):
        at = slice(lo, min(rows, lo + step))
        xd, d = x[at].double(), dh[at].double()
        g, u = xd @ wgd.t(), xd @ wud.t()
        eg, eu = ((cols + 1) * U * (xd.abs() @ w.abs().t()) for w in (wgd, wud))
        s = torch.sigmoid(g)
        a, da = g * s, s * (1 + g * torch.sigmoid(-g))
        assert bool(((kept[0, at].double() - g).abs() <= eg + 1e-37).all()) and bool(((kept[1, at].double() - u).abs() <= eu + 1e-37).all()), lo
        # as in the tests of smaller sizes: |act'| <= 1.13, |act''| <= 0.8, some 16 roundings in the activation
        ea = 1.13 * eg + 16 * U * (1 + g.abs()) * torch.minimum(g.abs(), torch.ones_like(g))
        eda = 0.8 * eg + 16 * U * (1 + g.abs())
        want = a * u
        assert bool(((h[at].double() - want).abs() <= ea * u.abs() + a.abs() * eu + ea * eu + 2 * U * want.abs() + H * want.abs() * 1.01 + tiny).all()), lo
        dg, du = d * u * da, d * a
        edg = d.abs() * (eu * da.abs() + u.abs() * eda + eu * eda) + (H * 1.01 + 4 * U) * dg.abs() + tiny
        edu = d.abs() * ea + (H * 1.01 + 4 * U) * du.abs() + tiny
        if hidden < 1 << 20:       # (a sum over more: beyond what this tolerance says anything about)
            want = dg @ wgd + du @ wud
            terms = (dg.abs() + edg) @ wgd.abs() + (du.abs() + edu) @ wud.abs()
            off = edg @ wgd.abs() + edu @ wud.abs() + (2 * hidden + 1) * U * terms + H * want.abs() * 1.01 + tiny
            assert bool(((dx[at].double() - want).abs() <= off).all()), lo
        for i, (v, e) in enumerate(((dg, edg), (du, edu)) if rows > 1000 else ()):
            for k in range(cols):      # (a library's product over so many rows takes seconds)
                xk = xd[:, k:k + 1]
                sums[i][:, k] += (v * xk).sum(0)
                sums[2 + i][:, k] += ((e + (rows / 2048 / 32 + 300) * U * v.abs()) * xk.abs()).sum(0)      # (256 pieces of 8 waves, 32 rows an instruction)
    if rows > 1000:
        for got, want, e in ((dwg, sums[0], sums[2]), (dwu, sums[1], sums[3])):
            assert bool(((got.double() - want).abs() <= e + H * want.abs() * 1.01).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_operands_read_in_place_are_not_copied(dtype):
    """Memory that a call takes beside its result: none where rows are aligned and whole steps long, a copy of x and the weights else."""
    from bayesian_optimization_amd import features
    rows, cols, hidden = 1 << 17, 256, 512
    x, w = rand((rows, cols + 8), dtype, 7), rand((hidden, cols + 8), dtype, 8, 0.1)
    result = rows * hidden * x.element_size()
    for a, b, copy in ((x[:, :cols], w[:, :cols], 0), (x[:, :cols].contiguous(), w[:, :cols].contiguous(), 0), (x[:, 1:cols + 1], w[:, 1:cols + 1], rows * cols * x.element_size())):
        want = features.gated_unit(a, b, b)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        h = features.gated_unit(a, b, b)
        assert copy <= torch.cuda.max_memory_allocated() - before - result <= copy * 1.02 + (1 << 20)
        assert torch.equal(h, want)
        del h, want


# Gradients of few elements among many rows or hidden units, which the kernels for large operands take: split contractions, both products
@pytest.mark.parametrize('rows,cols,hidden', [(8192, 1, 256), (4096, 512, 1), (300000, 60, 64), (100003, 31, 128), (70000, 128, 16), (40001, 1000, 4), (131072, 25, 150), (128, 30, 100000)])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_gradients_of_few_elements_among_many_rows(dtype, act, rows, cols, hidden):
    """dg and du as two numbers there too: off by the square of half a step, not by half a step."""
    check_gated(dtype, act, rows, cols, hidden, slope=half(dtype) ** 2)


# Every backward kernel: one launch, fragments into registers with one part and two, 64 x 64 tiles, both tiles for large operands, few columns
RANGES = [(95, 621, 128), (60, 1, 21), (600, 10, 1), (1000, 520, 200), (3000, 400, 100), (2050, 621, 777), (8200, 1024, 1100), (50007, 15, 300), (1, 40, 7)]


@pytest.mark.parametrize('rows,cols,hidden', RANGES)
# scales of x, of the weights and of dh; which gradients are then numbers of float16's range
@pytest.mark.parametrize('sx,sw,sd,what', [(1.0, 0.1, 1e-4, 'xw'), (300.0, 3e-4, 1e-6, 'w'), (3e-4, 300.0, 1e-6, 'x'), (3000.0, 0.002, 1e4, 'x'), (5e-4, 1.2e4, 1e4, 'w')])
def test_float16_gradients_whose_slopes_leave_its_range(rows, cols, hidden, sx, sw, sd, what):
    """dg and du around 1e-7, or beyond 65504, with gradients in between: off by their rounding relative to themselves, and by 2^-39 of the
    largest of them, wherever that lies."""
    from bayesian_optimization_amd import features
    from test_gpu_features import gated_ref, rand as normal, within
    U, H, f16 = 2.0 ** -24, 2.0 ** -11, torch.float16
    x, dh = normal((rows, cols), f16, 1, sx), normal((rows, hidden), f16, 2, sd)
    wg, wu = normal((hidden, cols), f16, 3, sw * cols ** -0.5), normal((hidden, cols), f16, 4, sw * cols ** -0.5)
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    dx, dwg, dwu = features.gated_unit_backward(dh, x, wg, wu, kept)
    g, u, a, da = gated_ref(x, wg, wu, 'silu')
    eg, eu = ((cols + 1) * U * (x.double().abs() @ w.double().abs().t()) for w in (wg, wu))
    ea = 1.13 * eg + 16 * U * (1 + g.abs()) * torch.minimum(g.abs(), torch.ones_like(g))
    eda = 0.8 * eg + 16 * U * (1 + g.abs())
    d = dh.double()
    dg, du = d * u * da, d * a
    low = 2.0 ** -39 * max(float(dg.abs().max()), float(du.abs().max()))
    edg = d.abs() * (eu * da.abs() + u.abs() * eda + eu * eda) + (H * 1.01 + 4 * U) * dg.abs() + low
    edu = d.abs() * ea + (H * 1.01 + 4 * U) * du.abs() + low
    wga, wua, xa, tiny = wg.double().abs(), wu.double().abs(), x.double().abs(), 2.0 ** -25

    def check(got, want, off, name):
        inside = want.abs() + off < 65504
        assert int(inside.sum()) > 0.9 * want.numel()
        within(torch.where(inside, got.double(), want), want, off + H * want.abs() * 1.01 + tiny, name)
    if 'x' in what:
        want = dg @ wg.double() + du @ wu.double()
        check(dx, want, edg @ wga + edu @ wua + (2 * hidden + 1) * U * ((dg.abs() + edg) @ wga + (du.abs() + edu) @ wua), 'dx')
    if 'w' in what:
        for got, v, e in ((dwg, dg, edg), (dwu, du, edu)):
            check(got, v.t() @ x.double(), e.t() @ xa + (rows + 1) * U * ((v.abs() + e).t() @ xa), 'dw')


@pytest.mark.parametrize('rows,cols,hidden', RANGES[:7])
def test_float16_gradients_around_an_infinity(rows, cols, hidden):
    """An infinite or NaN gradient that comes in enters what depends on it, and does not count as the largest of the others."""
    from bayesian_optimization_amd import features
    x, dh = rand((rows, cols), torch.float16, 1), rand((rows, hidden), torch.float16, 2, 1e-4)
    wg, wu = rand((hidden, cols), torch.float16, 3, 0.1 * cols ** -0.5), rand((hidden, cols), torch.float16, 4, 0.1 * cols ** -0.5)
    _, kept = features.gated_unit(x, wg, wu, keep=True)
    want = features.gated_unit_backward(dh, x, wg, wu, kept)
    for bad in (float('inf'), float('nan')):
        d = dh.clone()
        d[rows // 2, 0] = bad
        dx, dwg, dwu = features.gated_unit_backward(d, x, wg, wu, kept)
        assert not bool(torch.isfinite(dx[rows // 2]).any()) and not bool(torch.isfinite(dwu[0]).any())
        others = torch.arange(rows, device='cuda') != rows // 2
        assert bool(((dx[others].double() - want[0][others].double()).abs() <= 2.0 ** -10 * want[0][others].double().abs() + 2.0 ** -24).all())
        assert torch.isfinite(dwg[1:]).all() and torch.isfinite(dwu[1:]).all()
    zero = features.gated_unit_backward(torch.zeros_like(dh), x, wg, wu, kept)
    assert all(float(v.abs().max()) == 0 for v in zero)


# a few rows, fragments into registers, 64 x 64 tiles, rows streamed through LDS, tiles for large operands
@pytest.mark.parametrize('rows,cols,hidden', [(5, 2, 7), (100, 2, 9), (3000, 2, 600), (70001, 2, 40), (2100, 300, 1000)])
@pytest.mark.parametrize('dtype,big,least', [(torch.float32, 1e18, -12.0), (torch.bfloat16, 1e18, -12.0), (torch.float16, 6e4, -7.0)])
def test_gelu_keeps_its_lower_tail(dtype, big, least, rows, cols, hidden):
    """Far below zero gelu is next to nothing, and times a large factor a number again: off relative to itself by half a step, by the fit
    (6e-5 for 16 bits, 4e-7 for 32) and by the rounding of the exponent g^2 / 2, three roundings of 2^-24 of it, with a dozen others."""
    from bayesian_optimization_amd import features
    U = 2.0 ** -24
    x = torch.zeros((rows, cols), dtype=dtype, device='cuda')
    x[:, 0] = torch.linspace(least, -0.5, rows, device='cuda').to(dtype)      # g and u are products of two numbers, without a sum
    x[:, 1] = big
    w = torch.zeros((2, hidden, cols), dtype=dtype, device='cuda')
    w[0, :, 0], w[1, :, 1] = 1.0, big
    h, kept = features.gated_unit(x, w[0], w[1], 'gelu', keep=True)
    g, u = x[:, :1].double(), x[:, 1:2].double() * w[1, 0, 1].double()
    assert torch.equal(kept[0, :, 0], x[:, 0].float()) and bool(((kept[1, :, :1].double() - u).abs() <= U * u).all())
    want = 0.5 * g * torch.erfc(-g / math.sqrt(2)) * u
    rel = half(dtype) * 1.01 + (4e-7 if dtype == torch.float32 else 6e-5) + (2 * g * g + 16) * U
    assert bool((want.abs() > 1e-3).all())
    inside = want.abs() * 1.01 < torch.finfo(dtype).max
    off = (h.double() - want).abs() / want.abs()
    assert bool(((off <= rel) | ~inside).all()), (off - rel).max()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows,cols,hidden', [(30, 11, 9), (600, 10, 1), (4096, 512, 1), (70000, 7, 20), (1000, 3, 600), (130, 31, 3000), (1000, 520, 200), (2050, 621, 777)])
def test_an_infinite_weight_enters_its_column_alone(dtype, rows, cols, hidden):
    """Whatever dg and du enter the products as: the gradient of that column is infinite with the sign of its term, the others are as without."""
    from bayesian_optimization_amd import features
    x = rand((rows, cols), dtype, 1)
    wg, wu = rand((hidden, cols), dtype, 3, 0.1 * cols ** -0.5), rand((hidden, cols), dtype, 4, 0.1 * cols ** -0.5)
    _, kept = features.gated_unit(x, wg, wu, keep=True)
    dh = torch.ones((rows, hidden), dtype=dtype, device='cuda')
    want, _, _ = features.gated_unit_backward(dh, x, wg, wu, kept)
    wu[hidden - 1, cols - 1] = float('inf')
    dx, _, _ = features.gated_unit_backward(dh, x, wg, wu, kept)
    assert torch.equal(dx[:, :-1], want[:, :-1])
    du = torch.nn.functional.silu(kept[0, :, -1].double())
    sure = du.abs() > 1e-4             # (a factor that float16 holds)
    assert bool((dx[:, -1].double() == torch.where(du > 0, float('inf'), -float('inf')))[sure].all()) and int(sure.sum()) > 0.9 * rows
