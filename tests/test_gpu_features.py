"""GPU: layer norm and gated unit, forward and backward, against their formulas in 64 bits.

Tolerances count roundings.  U = 2^-24 is half a step of float32, H half a step of the output's type relative to the value.  A
sum of n float32 terms in any order is off by at most n U times the sum of their magnitudes; the kernels' sums are shorter
chains joined by a tree, and the chains (not n) are counted where n would drown the check."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rand(shape, dtype, seed, scale=1.0, offset=0.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * scale + offset).to(dtype)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), '%s: %d of %d off, worst %g over' % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() - tol).max()))


def norm_ref(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    xh = (x - mean) * rstd
    return xh * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double()), mean, rstd, xh


def norm_tol(x, xh, rstd, w, b, dtype, y):
    # a thread sums at most 16 elements, a tree of at most 10 levels joins them (long rows: chains of cols / 1024 packs): 32 roundings
    # and, for rows read in a loop, one more per pack; the mean is off by that times max|x|, rstd by half as many relative
    chain = 32 + x.shape[1] / 4096
    big = x.double().abs().amax(1, keepdim=True)
    exh = chain * U * big * rstd + (chain + 8) * U * xh.abs() + (chain * U * big * rstd) ** 2 * xh.abs()
    ww = 1.0 if w is None else w.double().abs()
    return exh, exh * ww + 3 * U * (xh.abs() * ww + (0.0 if b is None else b.double().abs())) + half(dtype) * y.abs() * 1.01 + 1e-38 + (
        2.0 ** -24 if dtype == torch.float16 else 0.0)      # float16 below its smallest normal number: half a step there


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 1), (5, 2), (2, 7), (7, 8), (1, 9), (33, 31), (95, 621), (6, 63), (6, 64), (6, 65), (4, 511), (4, 513),
                                       (9, 1024), (5, 1025), (3, 2047), (2, 4100), (3, 8193), (2, 16384), (2, 16389), (3, 40001)])
def test_layer_norm_forward_and_backward(dtype, rows, cols):
    from bayesian_optimization_amd import features
    eps = 1e-5
    x, dy = rand((rows, cols), dtype, 1, offset=0.7), rand((rows, cols), dtype, 2)
    w, b = rand((cols,), dtype, 3, 0.3, 1.0), rand((cols,), dtype, 4, 0.3)
    y, mean, rstd = features.layer_norm(x, w, b, eps)
    dx, dw, db = features.layer_norm_backward(dy, x, w, mean, rstd)
    assert y.dtype == dx.dtype == dw.dtype == db.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
    yr, mr, rr, xh = norm_ref(x, w, b, eps)
    exh, tol = norm_tol(x, xh, rr, w, b, dtype, yr)
    within(y, yr, tol, 'y')
    within(mean[:, None], mr, (32 + cols / 4096) * U * x.double().abs().amax(1, keepdim=True), 'mean')
    g = dy.double() * w.double()
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    ref = rr * (g - m1 - xh * m2)
    chain = 40 + cols / 4096
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    erel = 2 * chain * U * (1 + x.double().abs().amax(1, keepdim=True) * rr)
    tol = rr * (chain * U * (g.abs() + a1 + xh.abs() * a2) + exh * a2 + xh.abs() * (g.abs() * exh).mean(1, keepdim=True)) + erel * ref.abs() \
        + half(dtype) * ref.abs() * 1.01 + (2.0 ** -24 if dtype == torch.float16 else 1e-38)
    within(dx, ref, tol, 'dx')
    for got, want, terms, err in ((dw, (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0), (dy.double().abs() * exh).sum(0)),
                                  (db, dy.double().sum(0), dy.double().abs().sum(0), 0.0)):
        within(got, want, (rows + 4) * U * terms + err + half(dtype) * want.abs() * 1.01 + (2.0 ** -24 if dtype == torch.float16 else 1e-38), 'column sums')


def test_layer_norm_without_weight_and_bias_and_the_constant_row():
    from bayesian_optimization_amd import features
    x = rand((4, 100), torch.float32, 5)
    x[2] = 3.25                       # variance 0: y is 0, rstd = eps^-1/2
    y, mean, rstd = features.layer_norm(x, None, None, 1e-4)
    assert torch.equal(y[2], torch.zeros(100, device='cuda')) and abs(float(rstd[2]) - 100.0) < 1e-3
    yr, _, rr, xh = norm_ref(x, None, None, 1e-4)
    within(y, yr, norm_tol(x, xh, rr, None, None, torch.float32, yr)[1], 'y')
    dx, dw, db = features.layer_norm_backward(torch.ones_like(x), x, None, mean, rstd)
    assert float(dx.abs().max()) < 1e-3 and torch.equal(db, torch.full((100,), 4.0, device='cuda'))


def test_layer_norm_keeps_the_variance_of_rows_far_from_zero():
    """mean 1000, deviation 1: the centred second moment has no cancellation; E[x^2] - E[x]^2 in 32 bits would be off by 6 %."""
    from bayesian_optimization_amd import features
    x = rand((8, 621), torch.float32, 6, 1.0, 1000.0)
    _, _, rstd = features.layer_norm(x)
    _, _, rr, _ = norm_ref(x, None, None, 1e-5)
    assert float((rstd.double() / rr[:, 0] - 1).abs().max()) < 1e-5


def test_layer_norm_gradient_against_differences():
    from bayesian_optimization_amd import features
    x, dy = rand((3, 17), torch.float32, 7), rand((3, 17), torch.float32, 8)
    w, b = rand((17,), torch.float32, 9), rand((17,), torch.float32, 10)
    _, mean, rstd = features.layer_norm(x, w, b)
    dx, dw, db = features.layer_norm_backward(dy, x, w, mean, rstd)

    def loss(x_, w_, b_):
        return float((norm_ref(x_, w_, b_, 1e-5)[0] * dy.double()).sum())
    for t, grad in ((x, dx), (w, dw), (b, db)):
        for at in (0, 5, t.numel() - 1):
            e = torch.zeros(t.numel(), dtype=torch.float64, device='cuda')
            e[at] = 1e-5
            hi, lo = ((t.double() + s * e.view_as(t)) for s in (1, -1))
            args = [v.double() for v in (x, w, b)]
            k = next(i for i, v in enumerate((x, w, b)) if v is t)
            up, down = list(args), list(args)
            up[k], down[k] = hi, lo
            assert abs((loss(*up) - loss(*down)) / 2e-5 - float(grad.flatten()[at])) < 1e-4


@pytest.mark.parametrize('dtype', TYPES)
def test_layer_norm_takes_strided_and_unaligned_rows(dtype):
    from bayesian_optimization_amd import features
    base = rand((12, 1003), dtype, 11)
    x = base[1::2, 3:624]             # row stride 2006, starts at element 3 of a row
    w = rand((621,), dtype, 12)
    y, mean, rstd = features.layer_norm(x, w)
    y2, mean2, rstd2 = features.layer_norm(x.contiguous(), w)
    assert torch.equal(y, y2) and torch.equal(mean, mean2) and torch.equal(rstd, rstd2)
    dy = rand((6, 700), dtype, 13)[:, 5:626]
    for a, c in zip(features.layer_norm_backward(dy, x, w, mean, rstd), features.layer_norm_backward(dy.contiguous(), x.contiguous(), w, mean, rstd)):
        assert torch.equal(a, c)


def test_layer_norm_nan_and_infinity_stay_in_their_row():
    from bayesian_optimization_amd import features
    x = rand((5, 300), torch.float32, 14)
    x[1, 7], x[3, 299] = float('nan'), float('inf')
    y, _, _ = features.layer_norm(x)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3]).all()) and bool(torch.isfinite(y[[0, 2, 4]]).all())


def test_layer_norm_offsets_past_32_bits():
    from bayesian_optimization_amd import features
    rows, cols = (1 << 20) + 3, 4096
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device='cuda')
    x[:] = rand((1, cols), torch.bfloat16, 15)
    x[-1] = rand((cols,), torch.bfloat16, 16)
    y, mean, rstd = features.layer_norm(x)
    one, _, _ = features.layer_norm(x[-2:].contiguous())
    assert torch.equal(y[-2:], one) and torch.equal(y[0], one[0])
    dx, _, db = features.layer_norm_backward(x, x, None, mean, rstd)
    dx1, _, _ = features.layer_norm_backward(x[-2:].contiguous(), x[-2:].contiguous(), None, mean[-2:], rstd[-2:])
    assert torch.equal(dx[-2:], dx1)


def gated_ref(x, wg, wu, act):
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    if act == 'silu':
        s = torch.sigmoid(g)
        return g, u, g * s, s * (1 + g * torch.sigmoid(-g))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g, u, g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


GATED_SHAPES = [(1, 1, 1), (1, 621, 16), (2, 5, 3), (3, 64, 64), (17, 33, 65), (95, 621, 128), (64, 128, 192), (65, 130, 63), (1, 2048, 300),
                (5, 512, 1000), (200, 64, 1), (130, 1, 70), (300, 257, 513), (512, 512, 512), (257, 1024, 640)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('rows,cols,hidden', GATED_SHAPES)
def test_gated_unit_forward_and_backward(dtype, act, rows, cols, hidden):
    check_gated(dtype, act, rows, cols, hidden)


# large enough for the kernels that load straight into LDS, both tile sizes, whole and broken steps, split contractions, edges
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols,hidden', [(1100, 1024, 1000), (2050, 621, 777), (300, 4096, 1030), (128, 2048, 2111), (4100, 520, 2049), (2305, 1024, 4224), (20000, 64, 128),
                                              (129, 8192, 640), (8200, 640, 1024),
                                              (70001, 40, 90), (66000, 128, 33), (40000, 190, 300), (33000, 256, 515)])
def test_gated_unit_large(dtype, rows, cols, hidden):
    check_gated(dtype, 'gelu' if rows % 2 else 'silu', rows, cols, hidden)


# many rows and few hidden units: every number of fragments, whole and padded, less than 64 columns, pieces of the contraction of
# which the last is empty (20017 rows over 39 pieces of 33 slabs)
@pytest.mark.parametrize('rows,cols,hidden', [(16384, 64, 1), (16385, 65, 8), (17003, 483, 4), (20017, 61, 16), (20017, 621, 21), (16391, 100, 24), (30011, 40, 31),
                                              (16411, 129, 32), (16500, 67, 33), (20021, 621, 48), (33000, 32, 57), (24001, 130, 64), (66000, 17, 3), (16384, 2050, 12)])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
def test_gated_unit_many_rows_few_hidden_units(act, rows, cols, hidden):
    check_gated(torch.float32, act, rows, cols, hidden)


# many rows, few columns, many hidden units: every number of column fragments, whole and broken slabs on both sides
@pytest.mark.parametrize('rows,cols,hidden', [(4096, 1, 1025), (4099, 3, 1040), (5001, 16, 1000), (50007, 15, 129), (20011, 17, 300), (9999, 32, 640), (33001, 33, 200),
                                              (33009, 48, 144), (16501, 49, 333), (40001, 64, 131), (65536, 4, 65), (131073, 7, 65), (8197, 16, 1100)])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('dtype', TYPES)
def test_gated_unit_few_columns(dtype, act, rows, cols, hidden):
    check_gated(dtype, act, rows, cols, hidden)


def test_gated_unit_few_columns_strides_infinities_and_parts():
    from bayesian_optimization_amd import features
    rows, cols, hidden = 20005, 19, 213
    x = rand((rows, cols + 9), torch.float32, 85)[:, 3:3 + cols]
    wg, wu = (rand((hidden, cols + 5), torch.float32, s, 0.2)[:, 1:1 + cols] for s in (86, 87))
    dh = rand((rows, hidden + 2), torch.float32, 88)[:, 1:1 + hidden]
    near = [v.contiguous() for v in (x, wg, wu)]
    _, kept = features.gated_unit(*near, keep=True)
    full = features.gated_unit_backward(dh.contiguous(), *near, kept)
    assert all(torch.equal(a, b) for a, b in zip(features.gated_unit_backward(dh, x, wg, wu, kept), full))
    part = features.gated_unit_backward(dh, *near, kept, need_dw=False)
    assert torch.equal(part[0], full[0]) and part[1] is None and part[2] is None
    part = features.gated_unit_backward(dh, *near, kept, need_dx=False)
    assert part[0] is None and torch.equal(part[1], full[1]) and torch.equal(part[2], full[2])
    x, wg, wu = near
    a = gated_ref(x, wg, wu, 'silu')[2]
    wu[hidden - 1, 18] = float('inf')      # the last weight of all: nothing but its own column
    dx, _, _ = features.gated_unit_backward(torch.ones_like(kept[0]), x, wg, wu, kept)
    assert bool((dx[:, 18] == torch.where(a[:, -1] > 0, float('inf'), -float('inf'))).all()) and bool(torch.isfinite(dx[:, :18]).all())
    bad = dh.contiguous()
    bad[77, 5] = float('nan')
    dx, dwg, dwu = features.gated_unit_backward(bad, *[v.contiguous() for v in (x, wg, near[2].nan_to_num(posinf=0.5))], kept)
    assert bool(torch.isnan(dx[77]).all()) and bool(torch.isfinite(dx[:77]).all()) and bool(torch.isfinite(dx[78:]).all())
    assert bool(torch.isnan(dwg[5]).all()) and int(torch.isnan(dwg).sum()) == cols and int(torch.isnan(dwu).sum()) == cols


def test_gated_unit_many_rows_strides_infinities_and_parts():
    from bayesian_optimization_amd import features
    rows, cols, hidden = 16390, 70, 5
    x = rand((rows, cols + 9), torch.float32, 81)[:, 3:3 + cols]
    far = torch.zeros((hidden, 1 << 22), device='cuda')      # rows of weights far apart
    wg, wu = far[:, 1:1 + cols], far[:, 200:200 + cols]
    wg.copy_(rand((hidden, cols), torch.float32, 82, 0.1))
    wu.copy_(rand((hidden, cols), torch.float32, 83, 0.1))
    dh = rand((rows, hidden + 2), torch.float32, 84)[:, 1:1 + hidden]
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    near = [v.contiguous() for v in (x, wg, wu)]
    h2, kept2 = features.gated_unit(*near, keep=True)
    full = features.gated_unit_backward(dh.contiguous(), *near, kept2)
    for a, b in [(h, h2), (kept, kept2)] + list(zip(features.gated_unit_backward(dh, x, wg, wu, kept), full)):
        assert float((a.double() - b.double()).abs().max()) <= 2e-6 * float(b.double().abs().max()) + 1e-6
    part = features.gated_unit_backward(dh, *near, kept2, need_dw=False)
    assert torch.equal(part[0], full[0]) and part[1] is None and part[2] is None
    part = features.gated_unit_backward(dh, *near, kept2, need_dx=False)
    assert part[0] is None and torch.equal(part[1], full[1]) and torch.equal(part[2], full[2])
    # an infinite weight of the last hidden unit, a NaN row of x: what they enter and nothing else
    x, wg, wu = near
    wu[4, 69] = float('inf')
    dx, _, _ = features.gated_unit_backward(torch.ones_like(h), x, wg, wu, kept2)
    g, _, a, _ = gated_ref(x, near[1], near[2].nan_to_num(posinf=0.0), 'silu')
    assert bool((dx[:, 69] == torch.where(a[:, 4] > 0, float('inf'), -float('inf'))).all()) and bool(torch.isfinite(dx[:, :69]).all())
    wu[4, 69] = 0.5
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    x[77] = float('nan')
    h2, kept2 = features.gated_unit(x, wg, wu, keep=True)
    assert bool(torch.isnan(h2[77]).all()) and torch.equal(torch.cat([h[:77], h[78:]]), torch.cat([h2[:77], h2[78:]]))


# Gradients of few elements, where the terms of a sum may cancel in all of them: in 16 bits dg and du enter as two numbers, the rounded one
# and what the rounding left, itself rounded by at most half of a step, so that they are off by the square of half a step
@pytest.mark.parametrize('rows,cols,hidden', [(1, 1, 1), (2, 170, 14), (60, 1, 21), (500, 1, 1), (512, 5, 200), (600, 10, 1), (3109, 2, 4), (1000, 3, 600), (311, 56, 1),
                                              (213819, 10, 1), (20001, 5, 77), (3, 1300, 2000), (1, 4095, 2001), (65, 62, 3001)])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_gated_unit_gradients_of_few_elements(dtype, act, rows, cols, hidden):
    check_gated(dtype, act, rows, cols, hidden, slope=half(dtype) ** 2)


def check_gated(dtype, act, rows, cols, hidden, slope=None):
    from bayesian_optimization_amd import features
    x, dh = rand((rows, cols), dtype, 1), rand((rows, hidden), dtype, 2)
    wg, wu = rand((hidden, cols), dtype, 3, cols ** -0.5), rand((hidden, cols), dtype, 4, cols ** -0.5)
    h, kept = features.gated_unit(x, wg, wu, act, keep=True)
    assert torch.equal(h, features.gated_unit(x, wg, wu, act))
    dx, dwg, dwu = features.gated_unit_backward(dh, x, wg, wu, kept, act)
    H, tiny = half(dtype), (2.0 ** -24 if dtype == torch.float16 else 1e-37)
    g, u, a, da = gated_ref(x, wg, wu, act)
    # products: cols terms; exact in 32 bits for the short types, one rounding more for float32
    eg, eu = ((cols + 1) * U * (x.double().abs() @ w.double().abs().t()) for w in (wg, wu))
    within(kept[0], g, eg + 1e-37, 'g')
    within(kept[1], u, eu + 1e-37, 'u')
    # |act'| <= 1.13, |act''| <= 0.8; the activation itself: some 16 roundings of numbers of the size of g and 1
    ea = 1.13 * eg + 16 * U * (1 + g.abs()) * torch.minimum(g.abs(), torch.ones_like(g))
    eda = 0.8 * eg + 16 * U * (1 + g.abs())
    want = a * u
    within(h, want, ea * u.abs() + a.abs() * eu + ea * eu + 2 * U * want.abs() + H * want.abs() * 1.01 + tiny, 'h')
    d = dh.double()
    dg, du = d * u * da, d * a
    S = H if slope is None else slope
    edg = d.abs() * (eu * da.abs() + u.abs() * eda + eu * eda) + (S * 1.01 + 4 * U) * dg.abs() + tiny      # rounded once to the type of x
    edu = d.abs() * ea + (S * 1.01 + 4 * U) * du.abs() + tiny
    wga, wua, xa = wg.double().abs(), wu.double().abs(), x.double().abs()
    want = dg @ wg.double() + du @ wu.double()
    terms = (dg.abs() + edg) @ wga + (du.abs() + edu) @ wua
    within(dx, want, edg @ wga + edu @ wua + (2 * hidden + 1) * U * terms + H * want.abs() * 1.01 + tiny, 'dx')
    for got, v, e in ((dwg, dg, edg), (dwu, du, edu)):
        want = v.t() @ x.double()
        within(got, want, e.t() @ xa + (rows + 1) * U * ((v.abs() + e).t() @ xa) + H * want.abs() * 1.01 + tiny, 'dw')


@pytest.mark.parametrize('dtype', TYPES)
def test_gated_unit_takes_strided_and_unaligned_arrays(dtype):
    from bayesian_optimization_amd import features
    for rows, cols, hidden in ((70, 129, 77), (300, 256, 384), (1030, 1000, 1100), (1030, 1024, 1100)):
        x = rand((2 * rows, cols + 9), dtype, 21)[::2, 3:3 + cols]
        wg, wu = (rand((hidden, cols + 5), dtype, s, 0.1)[:, 1:1 + cols] for s in (22, 23))
        dh = rand((rows, hidden + 3), dtype, 24)[:, 2:2 + hidden]
        h, kept = features.gated_unit(x, wg, wu, keep=True)
        h2, kept2 = features.gated_unit(x.contiguous(), wg.contiguous(), wu.contiguous(), keep=True)
        H = 2.05 * half(dtype) if dtype != torch.float32 else 2e-6
        for a, c in [(h, h2), (kept, kept2)] + list(zip(features.gated_unit_backward(dh, x, wg, wu, kept),
                                                       features.gated_unit_backward(dh.contiguous(), x.contiguous(), wg.contiguous(), wu.contiguous(), kept2))):
            # another alignment may take another kernel, whose sums run in another order: last-bit differences only
            assert float((a.double() - c.double()).abs().max()) <= H * float(c.double().abs().max()) + 1e-6
        odd = features.gated_unit(x, wg, wu.contiguous())      # weights with different row strides
        assert float((odd.double() - h.double()).abs().max()) <= H * float(h.double().abs().max()) + 1e-6


def test_gated_unit_gradient_against_differences():
    from bayesian_optimization_amd import features
    x, dh = rand((4, 9), torch.float32, 31), rand((4, 6), torch.float32, 32)
    wg, wu = rand((6, 9), torch.float32, 33), rand((6, 9), torch.float32, 34)
    for act in ('silu', 'gelu'):
        _, kept = features.gated_unit(x, wg, wu, act, keep=True)
        grads = features.gated_unit_backward(dh, x, wg, wu, kept, act)

        def loss(*v):
            _, u, a, _ = gated_ref(*v, act)
            return float((a * u * dh.double()).sum())
        for k, grad in enumerate(grads):
            for at in (0, 7, grad.numel() - 1):
                args = [v.double() for v in (x, wg, wu)]
                e = torch.zeros(grad.numel(), dtype=torch.float64, device='cuda')
                e[at] = 1e-5
                up, down = list(args), list(args)
                up[k], down[k] = args[k] + e.view_as(args[k]), args[k] - e.view_as(args[k])
                assert abs((loss(*up) - loss(*down)) / 2e-5 - float(grad.flatten()[at])) < 1e-4


def test_gated_unit_extremes_saturate():
    """Products far out on both sides: silu(-90) and gelu(-20) are 0 to 32 bits, silu(90) and gelu(20) the identity; no NaN."""
    from bayesian_optimization_amd import features
    x = torch.tensor([[-90.0], [-20.0], [0.0], [20.0], [90.0], [-1e30], [1e30]], device='cuda')
    one = torch.ones((1, 1), device='cuda')
    for act in ('silu', 'gelu'):
        h, kept = features.gated_unit(x, one, one * 0 + 1, act, keep=True)
        a = h[:5, 0] / torch.where(x[:5, 0] == 0, 1.0, x[:5, 0])
        assert bool(torch.isfinite(h[:5]).all()) and abs(float(a[0])) < 1e-30 and float(a[4]) == 90.0 and float(h[5, 0]) == 0.0
        dx, dwg, _ = features.gated_unit_backward(torch.ones_like(h), x, one, one, kept, act)
        assert bool(torch.isfinite(dx[:5]).all()) and float(dx[2, 0]) == 0.0


def test_gated_unit_zero_rows_and_partial_gradients():
    from bayesian_optimization_amd import features
    wg, wu = rand((6, 9), torch.bfloat16, 41), rand((6, 9), torch.bfloat16, 42)
    x = torch.empty((0, 9), dtype=torch.bfloat16, device='cuda')
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    assert h.shape == (0, 6)
    dx, dwg, dwu = features.gated_unit_backward(h, x, wg, wu, kept)
    assert dx.shape == (0, 9) and float(dwg.abs().max()) == 0 and float(dwu.abs().max()) == 0
    y, mean, rstd = features.layer_norm(x)
    dx, dw, db = features.layer_norm_backward(x, x, None, mean, rstd)
    assert dx.shape == (0, 9) and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0
    x = rand((4, 9), torch.bfloat16, 43)
    h, kept = features.gated_unit(x, wg, wu, keep=True)
    full = features.gated_unit_backward(h, x, wg, wu, kept)
    part = features.gated_unit_backward(h, x, wg, wu, kept, need_dw=False)
    assert torch.equal(part[0], full[0]) and part[1] is None and part[2] is None
    part = features.gated_unit_backward(h, x, wg, wu, kept, need_dx=False)
    assert part[0] is None and torch.equal(part[1], full[1]) and torch.equal(part[2], full[2])


def test_gated_unit_offsets_past_32_bits():
    from bayesian_optimization_amd import features
    rows, cols, hidden = (1 << 20) + 70, 64, 4096
    x = rand((rows, cols), torch.bfloat16, 51)
    wg, wu = rand((hidden, cols), torch.bfloat16, 52, 0.1), rand((hidden, cols), torch.bfloat16, 53, 0.1)
    h = features.gated_unit(x, wg, wu)
    tail = features.gated_unit(x[-300:].contiguous(), wg, wu)
    assert float((h[-300:].double() - tail.double()).abs().max()) <= 2.05 * half(torch.bfloat16) * float(tail.abs().max())


@pytest.mark.parametrize('dtype', TYPES)
def test_operators_repeat_bit_for_bit_and_replay_from_a_graph(dtype):
    """Captured once, replayed on new inputs in the same buffers with eager work in between; every replay equals the eager call."""
    from bayesian_optimization_amd import features
    for rows, cols, hidden in ((95, 621, 128), (512, 512, 256), (1100, 1000, 1024), (17000, 70, 12), (66000, 128, 33)):
        x, dh = rand((rows, cols), dtype, 61), rand((rows, hidden), dtype, 62)
        w, wg, wu = rand((cols,), dtype, 63), rand((hidden, cols), dtype, 64, 0.05), rand((hidden, cols), dtype, 65, 0.05)

        def step():
            y, mean, rstd = features.layer_norm(x, w)
            h, kept = features.gated_unit(y, wg, wu, keep=True)
            dy, dwg, dwu = features.gated_unit_backward(dh, y, wg, wu, kept)
            return (y, h, dwg, dwu) + features.layer_norm_backward(dy, x, w, mean, rstd)
        first = step()
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        with torch.cuda.graph(graph2):
            out2 = step()
        for i in range(4):
            x.copy_(rand((rows, cols), dtype, 70 + i))
            dh.copy_(rand((rows, hidden), dtype, 80 + i))
            graph.replay()
            graph2.replay()
            torch.cuda.synchronize()
            eager = step()
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(eager, out, out2)), (rows, i)


def test_calls_at_the_same_time():
    """Two threads, a stream each, in step: every call has its workspace to itself."""
    import threading
    from bayesian_optimization_amd import draws, features
    jobs = [(torch.float32, 20017, 70, 12), (torch.bfloat16, 1100, 1000, 1024)]
    data = []
    for i, (dtype, rows, cols, hidden) in enumerate(jobs):
        data.append((rand((rows, cols), dtype, 101 + i), rand((hidden, cols), dtype, 111 + i, 0.05), rand((hidden, cols), dtype, 121 + i, 0.05),
                     rand((rows, hidden), dtype, 131 + i), rand((2, 200000), dtype, 141 + i), torch.rand(2, 30, device='cuda', dtype=torch.float64)))

    def step(x, wg, wu, dh, s, u):
        y, mean, rstd = features.layer_norm(x)
        h, kept = features.gated_unit(y, wg, wu, keep=True)
        dy, dwg, dwu = features.gated_unit_backward(dh, y, wg, wu, kept)
        return (h, dwg, dwu) + features.layer_norm_backward(dy, x, None, mean, rstd) + draws.sample(s, u, top_p=0.9, min_p=0.01)
    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                gate.wait(60)
                got = step(*data[i])
                stream.synchronize()
                wrong.extend(k for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_refusals_on_the_gpu():
    from bayesian_optimization_amd import features
    x = rand((4, 8), torch.float32, 91)
    w = rand((6, 8), torch.float32, 92)
    for bad in (lambda: features.layer_norm(x.t()), lambda: features.layer_norm(x, w[0].double()), lambda: features.layer_norm(x, w[0, :5]),
                lambda: features.layer_norm(x, eps=-1.0), lambda: features.layer_norm(x.double()), lambda: features.layer_norm(x[None]),
                lambda: features.layer_norm(x, w[0].cpu()), lambda: features.layer_norm(x[:1].expand(4, 8)),
                lambda: features.gated_unit(x, w, w[:5]), lambda: features.gated_unit(x, w, w, act='relu'),
                lambda: features.gated_unit(x, w.half(), w.half()), lambda: features.gated_unit(x, w[:0], w[:0]),
                lambda: features.gated_unit_backward(x, x, w, w, torch.zeros(2, 4, 6, device='cuda')),
                lambda: features.gated_unit_backward(w[:4, :6], x, w, w, torch.zeros(2, 4, 6, device='cuda', dtype=torch.float64))):
        with pytest.raises(ValueError):
            bad()


def test_feature_map_likelihood_gradient_against_differences():
    """The chain as it is used: spectra-like rows -> layer norm -> gated unit -> features -> -logL, and back.  float32 map under a
    float64 likelihood: central differences with a step of 2^-6 are off by the step squared and by 1e-6 / 2^-6."""
    import bayesian_optimization_amd as bo
    from bayesian_optimization_amd import features, hyperopt
    rng = np.random.default_rng(0)
    n, cols = 40, 61
    raw = rng.standard_normal((n, cols)).cumsum(axis=1) / 5.0
    yv = np.sin(raw[:, 3]) + 0.1 * rng.standard_normal(n)
    fmap = features.FeatureMap(cols, 24, 3, act='gelu', seed=1)
    x = torch.from_numpy(raw).float().cuda()
    theta = np.array([0.9, 1.1, 1.3])
    nll, g_theta, grads = hyperopt.lml_features(fmap, x, yv, theta, 0.3)
    assert np.isfinite(nll) and g_theta.shape == (3,)

    def value():
        z = fmap.forward(x)
        return hyperopt.lml_inputs(z.double().cpu().numpy(), yv, theta, 0.3)[0]
    assert abs(value() - nll) < 1e-9 * abs(nll)
    for name in ('norm_weight', 'norm_bias', 'w_gate', 'w_up', 'w_out'):
        p = fmap.params[name]
        direction = grads[name].double() / grads[name].double().norm()
        kept, step = p.clone(), 2.0 ** -6
        p.copy_((kept.double() + step * direction).float())
        up = value()
        p.copy_((kept.double() - step * direction).float())
        down = value()
        p.copy_(kept)
        want = float(grads[name].double().norm())
        assert abs((up - down) / (2 * step) - want) < 2e-2 * want + 1e-3, name
    # and on: a model on the features, candidates through the same map, a drawn batch of picks
    gp = bo.GP(0)
    gp.fit(fmap.numpy(raw), yv, theta, 0.3)
    gp.set_candidates(fmap.numpy(rng.standard_normal((500, cols)).cumsum(axis=1) / 5.0))
    gp.posterior()
    best, _ = gp.acquire()
    picks, logp = gp.draw(rng.random(8), temperature=0.05, top_p=0.9)
    assert picks.shape == (8,) and (picks >= 0).all() and (picks < 500).all() and (logp <= 0).all()
    assert gp.draw([0.3], temperature=0.0)[0][0] == best
    gp.close()
