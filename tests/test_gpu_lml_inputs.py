"""GPU: the gradient of -logL w.r.t. the training inputs, against its formula in 64 bits and against differences."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def ref(X, y, theta, sigma, kernel):
    """Formula with explicit inverse; also returns the sums of magnitudes that the error scales with."""
    n, d = X.shape
    diff = X[:, None, :] - X[None, :, :]
    D = ((diff / theta) ** 2).sum(-1)
    r = np.sqrt(5 * D)
    K, F = (np.exp(-D / 2),) * 2 if kernel == 0 else ((1 + r + r * r / 3) * np.exp(-r), 5 / 3 * (1 + r) * np.exp(-r))
    eps = sigma ** 2 if sigma else 1e-15 * n
    A = K + eps * np.eye(n)
    L = np.linalg.cholesky(A)
    Ki = np.linalg.inv(A)
    a = Ki @ y
    ya = y @ a
    P = (n * np.outer(a, a) / ya - Ki) * F
    np.fill_diagonal(P, 0)
    nll = n / 2 * (math.log(2 * math.pi) + 1 + math.log(ya / n)) + np.log(np.diag(L)).sum()
    gx = (P[:, :, None] * diff).sum(1) / theta ** 2
    gt = -0.5 * (P[:, :, None] * diff ** 2).sum((0, 1)) / theta ** 3
    return nll, gt, gx, np.linalg.cond(A), (np.abs(P)[:, :, None] * np.abs(diff)).sum(1) / theta ** 2


@pytest.mark.parametrize('kernel', [0, 1])
@pytest.mark.parametrize('n,d', [(1, 1), (2, 3), (5, 16), (31, 2), (32, 4), (33, 4), (64, 3), (65, 1), (94, 4), (128, 16), (129, 2), (300, 5), (513, 8), (700, 16), (2100, 3)])
def test_matches_the_formula(gp0, n, d, kernel):
    rng = np.random.default_rng(n + d)
    X, theta = rng.random((n, d)), 0.3 + 0.5 * rng.random(d)
    y = np.sin(3 * X.sum(1)) + 0.1 * rng.standard_normal(n) + 0.5
    nll, gt, gx = gp0.lml_inputs(X, y, theta, 0.2, kernel)
    want, gtw, gxw, cond, mag = ref(X, y, theta, 0.2, kernel)
    tol = 2.0 ** -53 * cond * 64      # Kinv and alpha in 64 bits: a small multiple of cond * 2^-53, relative to the terms
    assert abs(nll - want) <= tol * max(1.0, abs(want)) + 1e-10
    assert np.all(np.abs(gx - gxw) <= tol * mag.max(0) + 1e-12)
    assert np.all(np.abs(gt - gtw) <= tol * np.abs(gtw).max() * 10 + 1e-9 * np.abs(gtw).max() + 1e-12)
    nll2, g2, st = gp0.lml_batch(X, y, theta[None], [0.2], kernel, grad=True)
    assert nll2[0] == nll and np.array_equal(g2[0], gt) and st[0] == 0      # the same numbers as the call without inputs
    again = gp0.lml_inputs(X, y, theta, 0.2, kernel)
    assert again[0] == nll and np.array_equal(again[2], gx)


@pytest.mark.parametrize('n', [40, 150])
def test_against_differences(gp0, n):
    rng = np.random.default_rng(7)
    X, theta = rng.random((n, 3)), np.array([0.4, 0.6, 0.5])
    y = np.cos(4 * X[:, 0]) + X[:, 1]
    for kernel in (0, 1):
        _, _, gx = gp0.lml_inputs(X, y, theta, 0.1, kernel)
        for i, t in ((0, 0), (n // 2, 1), (n - 1, 2)):
            up, down = X.copy(), X.copy()
            up[i, t] += 1e-5
            down[i, t] -= 1e-5
            v = gp0.lml_batch(up, y, theta[None], [0.1], kernel)[0][0] - gp0.lml_batch(down, y, theta[None], [0.1], kernel)[0][0]
            assert abs(v / 2e-5 - gx[i, t]) < 1e-4 * max(1.0, np.abs(gx).max())


def test_moves_of_all_inputs_together_change_nothing(gp0):
    """The covariance depends on differences only: every column of the gradient adds up to zero."""
    rng = np.random.default_rng(8)
    for n in (100, 1000):
        X = rng.random((n, 4))
        _, _, gx = gp0.lml_inputs(X, np.sin(X.sum(1)), [0.5] * 4, 0.1, 0)
        assert np.all(np.abs(gx.sum(0)) < 1e-9 * np.abs(gx).sum(0))


def test_refusals_and_failure(gp0):
    X, y = np.random.default_rng(9).random((20, 2)), np.zeros(20) + 1.0
    for bad in (lambda: gp0.lml_inputs(X, y[:5], [1, 1], 0.1), lambda: gp0.lml_inputs(X, y, [1, 1, 1], 0.1), lambda: gp0.lml_inputs(X, y, [0, 1], 0.1),
                lambda: gp0.lml_inputs(X, y, [1, 1], -0.1), lambda: gp0.lml_inputs(X, y, [1, 1], 0.1, kernel=7),
                lambda: gp0.lml_inputs(np.ones((5, 17)), np.ones(5), np.ones(17), 0.1), lambda: gp0.lml_inputs(X, y, [1, np.nan], 0.1)):
        with pytest.raises(ValueError):
            bad()
    for n in (20, 200):               # a NaN pivot is reported as not positive definite (the rule of the other calls)
        bad = np.random.default_rng(n).random((n, 2))
        bad[7, 1] = np.nan
        with pytest.raises(np.linalg.LinAlgError):
            gp0.lml_inputs(bad, np.sin(np.arange(float(n))), [0.5, 0.5], 0.1)
    nll, g, gx = gp0.lml_inputs(X, np.sin(X.sum(1)), [1, 1], 0.1)      # and the next call works
    assert np.isfinite(nll) and np.isfinite(gx).all()


def test_replayed_launch_sequence_gives_the_same_numbers(gp0):
    """Up to 16 panels the launch sequence is captured once and replayed: every replay on other data equals a fresh context's."""
    import bayesian_optimization_amd as bo
    rng = np.random.default_rng(10)
    for _ in range(4):
        X = rng.random((400, 3))
        y = rng.standard_normal(400)
        got = gp0.lml_inputs(X, y, [0.3, 0.4, 0.5], 0.2)
        batch = gp0.lml_batch(X, y, [[0.3, 0.4, 0.5]], [0.2], grad=True)
        fresh = bo.GP(0)
        want = fresh.lml_inputs(X, y, [0.3, 0.4, 0.5], 0.2)
        fresh.close()
        assert got[0] == want[0] == batch[0][0] and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]) and np.array_equal(batch[1][0], want[1])


def test_multi_and_hyperopt_entry_points(gp0):
    import bayesian_optimization_amd as bo
    from bayesian_optimization_amd import hyperopt
    X = np.random.default_rng(11).random((60, 2))
    y = np.sin(X.sum(1))
    want = gp0.lml_inputs(X, y, [0.5, 0.5], 0.1)
    mg = bo.MultiGP([0, 0])
    for got in (mg.lml_inputs(X, y, [0.5, 0.5], 0.1), hyperopt.lml_inputs(X, y, [0.5, 0.5], 0.1)):
        assert got[0] == want[0] and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    mg.close()
