"""GPU: draws at the ends of a row's mass and at the borders between its scores, where rounding decides.

A pick has to have a weight whatever u is, and lie at u to within the rounding of the running sums: sums of n weights in 64 bits in any
order are off by at most n 2^-53 of their total.  u beyond its range counts as the nearest end of it, 0 or 1 - 2^-53."""
import math

import numpy as np
import pytest
import torch

from test_gpu_draws import kept_weights

pytestmark = pytest.mark.gpu
ENDS = [1.0, 2.0, math.inf, 1 - 2.0 ** -53, 1 - 2.0 ** -52, 1 - 2.0 ** -50, 0.0, -1.0, math.nan]


def check_ends(scores, u, index, logp, temperature=1.0, **st):
    S, U, index, logp = (v.double().cpu().numpy() if v.dtype != torch.int64 else v.cpu().numpy() for v in (scores, u, index, logp))
    U = np.clip(np.where(np.isnan(U), 0.0, U), 0.0, 1 - 2.0 ** -53)
    n = S.shape[1]
    for r in range(S.shape[0]):
        w, t = kept_weights(S[r], temperature, st.get('top_k', 0), st.get('top_p', 1.0), st.get('min_p', 0.0))
        run = np.cumsum(w)
        Z = run[-1]
        slack = n * 2.0 ** -53 * Z * 4
        at = index[r]
        assert (at >= 0).all() and (at < n).all(), (r, at)
        assert (w[at] > 0).all(), (r, 'not in the kept set', at[w[at] <= 0], U[r][w[at] <= 0])
        assert (run[at] - w[at] - slack <= U[r] * Z).all() and (U[r] * Z <= run[at] + slack).all(), r
        assert np.allclose(logp[r], t[at] - math.log(Z), rtol=1e-13, atol=n * 2.0 ** -52 + 1e-14), r


def ends_and_borders(scores, seed, **st):
    """The ends, and running sums of the kept weights at random places, where a sum equals u times the whole but for its rounding."""
    rng = np.random.default_rng(seed)
    U = []
    for row in scores.double().cpu().numpy():
        w, _ = kept_weights(row, st.get('temperature', 1.0), st.get('top_k', 0), st.get('top_p', 1.0), st.get('min_p', 0.0))
        run = np.cumsum(w)
        U.append(np.concatenate((ENDS, np.minimum(run[rng.integers(0, run.size, 12)] / run[-1], 1 - 2.0 ** -53))))
    return torch.from_numpy(np.array(U)).cuda()


def masked(rows, cols, dtype, seed, how):
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = (torch.randn(rows, cols, generator=g, device='cuda', dtype=torch.float64) * 2.0).to(dtype)
    if how == 'tail':                  # nothing behind a place of each row's own
        first = torch.randint(1, cols, (rows, 1), generator=g, device='cuda')
        s = torch.where(torch.arange(cols, device='cuda') >= first, torch.tensor(-math.inf, dtype=dtype, device='cuda'), s)
    elif how == 'runs':                # runs of masked scores inside
        keep = torch.rand(rows, (cols + 36) // 37, generator=g, device='cuda') < 0.4
        keep[:, 0] = True
        s = torch.where(keep.repeat_interleave(37, dim=1)[:, :cols], s, torch.tensor(math.nan, dtype=dtype, device='cuda'))
    elif how == 'lowest':              # the type's lowest number: valid, without weight
        s[:, cols // 3:] = torch.finfo(dtype).min
    return s


SETTINGS = [dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=3000, top_p=0.97, temperature=3.0), dict(temperature=0.02),
            dict(top_k=600, min_p=1e-3, temperature=2.0)]


@pytest.mark.parametrize('how', ['tail', 'runs', 'lowest', 'none'])
@pytest.mark.parametrize('dtype', [torch.float64, torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,cols', [(80, 2), (80, 63), (80, 100), (80, 400), (80, 1000), (80, 1025), (60, 5000), (30, 20000), (4, 40000), (8, 70001), (2, 300001)])
def test_ends_and_borders(dtype, rows, cols, how):
    """One workgroup of every size a row, and many."""
    from bayesian_optimization_amd import draws
    s = masked(rows, cols, dtype, cols + rows, how)
    for i, st in enumerate(SETTINGS):
        u = ends_and_borders(s, i, **st)
        check_ends(s, u, *draws.sample(s, u, **st), **st)


def test_members_of_a_list_without_weight():
    """Scores so far below the best that their weight is 0 stand in a list with it: they are kept, and never drawn."""
    from bayesian_optimization_amd import draws
    for cols in (30, 3000, 200001):
        s = masked(20, cols, torch.float64, cols, 'none')
        s[:, cols // 2:] -= 2000.0
        s[3, :] -= 2000.0
        s[3, 7] = 0.0
        for st in (dict(top_k=cols - 3), dict(top_k=min(500, cols - 1)), dict()):
            u = ends_and_borders(s, 1, **st)
            check_ends(s, u, *draws.sample(s, u, **st), **st)


@pytest.mark.parametrize('rows,cols,dtype', [((1 << 26) + 3, 2, torch.float16), ((1 << 22) + 5, 513, torch.bfloat16), ((1 << 22) + 5, 1025, torch.bfloat16)])
def test_more_rows_than_a_launch_takes(rows, cols, dtype):
    """2^32 threads and more, at 64 or 1024 a row: the rows around the border of two launches, and all of them against smaller calls."""
    from bayesian_optimization_amd import draws
    g = torch.Generator(device='cuda').manual_seed(cols)
    s = torch.empty(rows, cols, dtype=dtype, device='cuda').normal_(generator=g)
    u = torch.rand(rows, 1, generator=g, device='cuda', dtype=torch.float64)
    top_k = torch.randint(0, 4, (rows,), generator=g, device='cuda')
    for st in (dict(top_p=0.9), dict(top_k=top_k, temperature=0.5)):
        index, logp = draws.sample(s, u, **st)
        step = (rows + 6) // 7
        for r in range(0, rows, step):
            part = dict(st, top_k=top_k[r:r + step]) if 'top_k' in st else st
            i, lp = draws.sample(s[r:r + step], u[r:r + step], **part)
            assert torch.equal(i, index[r:r + step]) and torch.equal(lp, logp[r:r + step]), r
