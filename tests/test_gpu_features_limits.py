"""GPU: layer norm and gated unit at sizes where a launch of a thread or more an element does not take them, and other limits."""
import numpy as np
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
