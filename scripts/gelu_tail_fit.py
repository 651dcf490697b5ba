#!/usr/bin/env python3
"""Coefficients of gelu's lower tail (activation() in bayesian_optimization_amd/csrc/k_gated.hpp):
    q = Phi(-|g|) = 1/2 erfc(z) = 1/2 exp(-z^2) t R(t),   z = |g| / sqrt 2,   t = 1 / (1 + c z),
R a polynomial fitted to erfcx(z) / t over z in [0, 10.5] (exp(-z^2) is nothing in 32 bits beyond): least squares on the relative error,
reweighted by it (Lawson's method) until the largest errors are alike; c by a search.  For results of 32 bits 10 terms, the relative error
alone; for results of 16 bits 6 terms, where the relative error counts as against 6e-5 (a tenth of half a step of float16) and the
absolute one as against 2e-7 (what a result near g = 0 may be off by besides).  Prints c, the coefficients rounded to 32 bits, and the
largest errors with them: relative in 64 bits and with every step rounded to 32 bits, absolute.
    python3 scripts/gelu_tail_fit.py"""
import numpy as np
from scipy.special import erfc, erfcx

Z = np.concatenate((np.linspace(0.0, 10.5, 6001), np.geomspace(1e-4, 10.5, 3000)))


def fit(terms, c, allowed, rounds):
    """Largest error relative to `allowed`, and R's coefficients."""
    t = 1.0 / (1.0 + c * Z)
    want = erfcx(Z) / t
    # Chebyshev polynomials of the interval, so that the equations stay well conditioned
    lo, hi = t.min(), t.max()
    A = np.polynomial.chebyshev.chebvander((2 * t - lo - hi) / (hi - lo), terms - 1) / (want * allowed)[:, None]
    w, best = np.ones_like(t), (np.inf, None)
    for _ in range(rounds):
        s = np.sqrt(w)
        x = np.linalg.lstsq(A * s[:, None], s / allowed, rcond=None)[0]
        e = np.abs(A @ x - 1.0 / allowed)
        if e.max() < best[0]:
            best = (e.max(), x)
        w = w * (e / e.max() + 1e-9)
        w /= w.sum()
    p = np.polynomial.chebyshev.Chebyshev(best[1], domain=[lo, hi]).convert(kind=np.polynomial.Polynomial).coef
    return best[0], p


def relative_in_32_bits(c, p, g):
    """Largest relative error of t R(t) for g in 32 bits, with every step rounded to them; a fused product and sum is rounded once."""
    f = np.float32
    t = f(1) / (f(1) + f(c * np.sqrt(0.5)) * g)
    r = np.full_like(t, f(p[-1]))
    for k in p[-2::-1]:
        r = (r.astype(np.float64) * t + f(k)).astype(f)
    return np.abs((t * r).astype(np.float64) / erfcx(g.astype(np.float64) * np.sqrt(0.5)) - 1).max()


if __name__ == '__main__':
    for terms, allowed in ((6, np.minimum(6e-5, 2e-7 / (0.5 * erfc(Z)))), (10, np.ones_like(Z))):
        lo, hi = 0.2, 0.9
        for _ in range(3):
            grid = np.linspace(lo, hi, 22)
            errors = [fit(terms, c, allowed, 60)[0] for c in grid]
            i = int(np.argmin(errors))
            lo, hi = grid[max(i - 1, 0)], grid[min(i + 1, 21)]
        c = round(float(grid[i]), 4)
        _, p = fit(terms, c, allowed, 400)
        p = p.astype(np.float32)
        t = 1.0 / (1.0 + c * Z)
        e = np.abs(np.polynomial.polynomial.polyval(t, p.astype(np.float64)) * t / erfcx(Z) - 1)
        print('%d terms, c = %.4f: relative error %.2e (%.2e in 32 bits), absolute error of q %.2e' % (
            terms, c, e.max(), relative_in_32_bits(c, p, np.linspace(0, 14.5, 200001, dtype=np.float32)), (e * 0.5 * erfc(Z)).max()))
        print('    ' + ', '.join('%.9gf' % v for v in p))
