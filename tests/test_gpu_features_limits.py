"""GPU: layer norm and gated unit at sizes where a launch of a thread or more an element does not take them, and other limits."""
import numpy as np
import pytest
import torch

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
