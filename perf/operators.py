"""Cases of the learned-input and drawn-pick operators: layer norm, gated unit, likelihood gradient with respect to the
training inputs, and draws from scores.  ``own`` false: their plain form in elementary torch operations; true: the calls a
user makes of this package."""
import math

import numpy as np
import torch

own = False

_TYPES = {'f64': torch.float64, 'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_BYTES = {'f64': 8, 'f32': 4, 'bf16': 2, 'f16': 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one pick from the 400-point grid of a notebook loop: nothing but latency
        dict(name='draw_grid_400_f64', op='draw', rows=1, cols=400, draws=1, dtype='f64', temperature=0.1, top_k=0, top_p=0.9, min_p=0.0),
        # a batch of score rows of odd length, one pick each: many models or states answered side by side, in a short type
        dict(name='draw_rows_256x65537_bf16', op='draw', rows=256, cols=65537, draws=1, dtype='bf16', temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
        # the 64^4 candidate lattice, a plate of 95 experiments drawn from its acquisition at once
        dict(name='draw_lattice_16m_f64', op='draw', rows=1, cols=64 ** 4, draws=95, dtype='f64', temperature=0.25, top_k=0, top_p=0.9, min_p=0.001),
        # the measured mixtures: 95 spectra of 621 channels, one training step of the normalisation
        dict(name='norm_train_95x621_f32', op='norm', rows=95, cols=621, dtype='f32', backward=True),
        # a large training set with wide rows
        dict(name='norm_train_16384x4096_bf16', op='norm', rows=16384, cols=4096, dtype='bf16', backward=True),
        # a candidate sweep of 1 M spectra: forward only, rows of odd length
        dict(name='norm_sweep_1m_x621_bf16', op='norm', rows=1 << 20, cols=621, dtype='bf16', backward=False),
        # one candidate at a time, as a simplex search asks for them
        dict(name='gated_one_1x2048_8192_bf16', op='gated', rows=1, cols=2048, hidden=8192, dtype='bf16', act='silu', backward=False),
        # the measured mixtures: one training step of the gated unit
        dict(name='gated_train_95x621_128_f32', op='gated', rows=95, cols=621, hidden=128, dtype='f32', act='gelu', backward=True),
        # a large training set
        dict(name='gated_train_16384x2048_8192_bf16', op='gated', rows=16384, cols=2048, hidden=8192, dtype='bf16', act='silu', backward=True),
        # a candidate sweep of 1 M rows, forward only
        dict(name='gated_sweep_1m_x256_512_f16', op='gated', rows=1 << 20, cols=256, hidden=512, dtype='f16', act='silu', backward=False),
        # likelihood gradient at the features of the measured mixtures (one left out)
        dict(name='inputs_94x4_rbf', op='inputs', n=94, d=4, kernel='rbf', sigma=0.1),
        # and of a large training set
        dict(name='inputs_8192x8_matern', op='inputs', n=8192, d=8, kernel='matern52', sigma=0.1),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['draw', 'draw', 'norm', 'norm', 'gated', 'gated', 'inputs'])
    if op == 'draw':
        cols = _log(rng, 1, 1 << 24)
        rows = _log(rng, 1, max(1, min(1024, (1 << 24) // cols)))
        return dict(op=op, rows=rows, cols=cols, draws=_log(rng, 1, 128), dtype=rng.choice(['f64', 'f32', 'bf16', 'f16']),
                    temperature=round(rng.uniform(0.05, 2.0), 4), top_k=rng.choice([0, 1, _log(rng, 1, 2 * cols)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.999), 4)]), min_p=rng.choice([0.0, round(rng.uniform(0.0005, 0.3), 4)]))
    if op == 'norm':
        cols = _log(rng, 1, 16384)
        rows = _log(rng, 1, max(1, min(1 << 20, (1 << 27) // cols)))
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(['f32', 'bf16', 'f16']), backward=rng.random() < 0.6)
    if op == 'gated':
        cols, hidden = _log(rng, 1, 4096), _log(rng, 1, 8192)
        rows = _log(rng, 1, max(1, min(1 << 18, (1 << 35) // (cols * hidden))))
        return dict(op=op, rows=rows, cols=cols, hidden=hidden, dtype=rng.choice(['f32', 'bf16', 'f16']), act=rng.choice(['silu', 'gelu']),
                    backward=rng.random() < 0.6)
    return dict(op=op, n=_log(rng, 2, 4096), d=rng.randint(1, 16), kernel=rng.choice(['rbf', 'matern52']), sigma=round(rng.uniform(0.05, 0.3), 4))


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device='cuda', dtype=torch.float32) * scale).to(dtype)

    op, state = case['op'], dict(case=case)
    if op == 'draw':
        rows, cols, dtype = case['rows'], case['cols'], _TYPES[case['dtype']]
        if case['dtype'] == 'f64':      # an acquisition: expected improvement of posteriors mostly below the incumbent
            z = torch.randn(rows, cols, generator=gen, device='cuda', dtype=torch.float64) * 1.2 - 1.0
            state['scores'] = z * 0.5 * torch.erfc(-z / math.sqrt(2.0)) + torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        else:                           # log scores
            state['scores'] = normal(rows, cols, dtype=dtype, scale=2.5)
        state['u'] = torch.rand(rows, case['draws'], generator=gen, device='cuda', dtype=torch.float64)
    elif op == 'norm':
        rows, cols, dtype = case['rows'], case['cols'], _TYPES[case['dtype']]
        # spectra have a base line: every row with an offset and a scale of its own
        x = normal(rows, cols) * (0.5 + torch.rand(rows, 1, generator=gen, device='cuda')) + normal(rows, 1)
        state.update(x=x.to(dtype), weight=(1.0 + 0.1 * normal(cols)).to(dtype), bias=normal(cols, dtype=dtype, scale=0.1))
        if case['backward']:
            state['dy'] = normal(rows, cols, dtype=dtype)
    elif op == 'gated':
        rows, cols, hidden, dtype = case['rows'], case['cols'], case['hidden'], _TYPES[case['dtype']]
        state.update(x=normal(rows, cols, dtype=dtype), w_gate=normal(hidden, cols, dtype=dtype, scale=cols ** -0.5),
                     w_up=normal(hidden, cols, dtype=dtype, scale=cols ** -0.5))
        if case['backward']:
            state['dh'] = normal(rows, hidden, dtype=dtype)
    else:                               # host arrays: what the likelihood calls of this package take
        r = np.random.default_rng(seed)
        X = r.random((case['n'], case['d']))
        state.update(X=X, y=np.sin(3.0 * X.sum(axis=1)) + 0.1 * r.standard_normal(case['n']), theta=0.3 + 0.5 * r.random(case['d']))
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_draw(scores, u, case):
    s = scores.double()
    s = torch.where(torch.isnan(s), -torch.inf, s)
    top = s.max(dim=1, keepdim=True).values
    t = torch.where(s == top, 0.0, (s - top) / case['temperature'])
    w = torch.exp(t)
    order = torch.sort(s, dim=1, descending=True, stable=True).indices
    ws = torch.gather(w, 1, order)
    place = torch.arange(s.shape[1], device=s.device)
    keep = ws > 0
    if case['top_k'] > 0:
        keep &= place < case['top_k']
    keep &= ws >= case['min_p']
    ws = torch.where(keep, ws, 0.0)
    run = torch.cumsum(ws, dim=1)
    if case['top_p'] < 1.0:
        keep &= ((run - ws) < case['top_p'] * run[:, -1:]) | (place == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    run = torch.cumsum(kept, dim=1)
    total = run[:, -1:]
    pick = torch.searchsorted(run, u * total, right=True)
    last = torch.where(kept > 0, place, 0).max(dim=1, keepdim=True).values
    pick = torch.minimum(pick, last)
    return dict(index=pick, logp=torch.gather(t, 1, pick) - torch.log(total))


def _plain_norm(s, case, eps=1e-5):
    x, w, b = s['x'].float(), s['weight'].float(), s['bias'].float()
    dtype = s['x'].dtype
    c = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + eps)
    xh = c * rstd
    out = dict(y=(xh * w + b).to(dtype))
    if case['backward']:
        dy = s['dy'].float()
        g = dy * w
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        out.update(dx=dx.to(dtype), dweight=(dy * xh).sum(dim=0).to(dtype), dbias=dy.sum(dim=0).to(dtype))
    return out


def _plain_gated(s, case):
    x, wg, wu = s['x'].float(), s['w_gate'].float(), s['w_up'].float()
    dtype = s['x'].dtype
    g, u = x @ wg.t(), x @ wu.t()
    if case['act'] == 'silu':
        f = 1.0 / (1.0 + torch.exp(-g))
        a, da = g * f, f * (1.0 + g * (1.0 - f))
    else:
        f = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        a, da = g * f, f + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    out = dict(h=(a * u).to(dtype))
    if case['backward']:
        dh = s['dh'].float()
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).to(dtype), dw_gate=(dg.t() @ x).to(dtype), dw_up=(du.t() @ x).to(dtype))
    return out


def _plain_inputs(s, case):
    X, y, theta = (torch.from_numpy(s[k]).cuda() for k in ('X', 'y', 'theta'))
    n = case['n']
    xs = X / theta
    D = torch.zeros(n, n, dtype=torch.float64, device='cuda')
    for t in range(case['d']):
        D += (xs[:, t, None] - xs[None, :, t]) ** 2
    if case['kernel'] == 'rbf':
        K = torch.exp(-0.5 * D)
        F = K
    else:
        r = torch.sqrt(5.0 * D)
        e = torch.exp(-r)
        K, F = (1.0 + r + r * r / 3.0) * e, (5.0 / 3.0) * (1.0 + r) * e
    L = torch.linalg.cholesky(K + case['sigma'] ** 2 * torch.eye(n, dtype=torch.float64, device='cuda'))
    Kinv = torch.cholesky_inverse(L)
    alpha = Kinv @ y
    ya = y @ alpha
    nll = 0.5 * n * (math.log(2.0 * math.pi) + 1.0) + 0.5 * n * torch.log(ya / n) + torch.log(torch.diagonal(L)).sum()
    P = (n / ya * alpha[:, None] * alpha[None, :] - Kinv) * F
    P.fill_diagonal_(0.0)
    row = P.sum(dim=1, keepdim=True)
    gx = (xs * row - P @ xs) / theta
    gt = -0.5 * (2.0 * (xs * xs * row).sum(dim=0) - 2.0 * (xs * (P @ xs)).sum(dim=0)) / theta
    return dict(nll=float(nll), grad_theta=gt.cpu().numpy(), grad_X=gx.cpu().numpy())


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state['case']
    op = case['op']
    if own:
        from bayesian_optimization_amd import draws, features, hyperopt
        if op == 'draw':
            index, logp = draws.sample(state['scores'], state['u'], temperature=case['temperature'], top_k=case['top_k'],
                                       top_p=case['top_p'], min_p=case['min_p'])
            return dict(index=index, logp=logp)
        if op == 'norm':
            y, mean, rstd = features.layer_norm(state['x'], state['weight'], state['bias'])
            if not case['backward']:
                return dict(y=y)
            dx, dw, db = features.layer_norm_backward(state['dy'], state['x'], state['weight'], mean, rstd)
            return dict(y=y, dx=dx, dweight=dw, dbias=db)
        if op == 'gated':
            if not case['backward']:
                return dict(h=features.gated_unit(state['x'], state['w_gate'], state['w_up'], act=case['act']))
            h, kept = features.gated_unit(state['x'], state['w_gate'], state['w_up'], act=case['act'], keep=True)
            dx, dwg, dwu = features.gated_unit_backward(state['dh'], state['x'], state['w_gate'], state['w_up'], kept, act=case['act'])
            return dict(h=h, dx=dx, dw_gate=dwg, dw_up=dwu)
        nll, gt, gx = hyperopt.lml_inputs(state['X'], state['y'], state['theta'], case['sigma'], kernel={'rbf': 0, 'matern52': 1}[case['kernel']])
        return dict(nll=nll, grad_theta=gt, grad_X=gx)
    if op == 'draw':
        return _plain_draw(state['scores'], state['u'], case)
    if op == 'norm':
        return _plain_norm(state, case)
    if op == 'gated':
        return _plain_gated(state, case)
    return _plain_inputs(state, case)


def work(case):
    op = case['op']
    if op == 'draw':
        e = case['rows'] * case['cols']
        return dict(bytes=e * _BYTES[case['dtype']] + case['rows'] * case['draws'] * 24, flops=4 * e)
    if op == 'norm':
        e, b = case['rows'] * case['cols'], _BYTES[case['dtype']]
        if case['backward']:
            return dict(bytes=4 * e * b + 4 * case['cols'] * b, flops=18 * e)
        return dict(bytes=2 * e * b + 2 * case['cols'] * b, flops=7 * e)
    if op == 'gated':
        m, k, h, b = case['rows'], case['cols'], case['hidden'], _BYTES[case['dtype']]
        if case['backward']:
            return dict(bytes=(2 * m * k + 2 * m * h + 4 * h * k) * b, flops=12 * m * k * h)
        return dict(bytes=(m * k + m * h + 2 * h * k) * b, flops=4 * m * k * h)
    n, d = case['n'], case['d']
    return dict(bytes=8 * (2 * n * d + n + 2 * d + 1), flops=n ** 3 + n * n * (6 * d + 12))


# ------------------------------------------------------------------------------------- the definitions again, in 64 bits
def _exact_draw(state, case):
    """Row by row on the host: rank, cut, renormalise, walk."""
    S, U = state['scores'].double().cpu().numpy(), state['u'].cpu().numpy()
    index, logp = np.empty(U.shape, np.int64), np.empty(U.shape)
    for r in range(S.shape[0]):
        s = np.where(np.isnan(S[r]), -np.inf, S[r])
        t = (s - s.max()) / case['temperature']
        w = np.exp(t)
        ranked = np.argsort(-s, kind='stable')
        if case['top_k'] > 0:
            ranked = ranked[:case['top_k']]
        ranked = ranked[(w[ranked] >= case['min_p']) & (w[ranked] > 0.0)]
        mass = np.cumsum(w[ranked])
        if case['top_p'] < 1.0:
            before = np.concatenate(([0.0], mass[:-1]))
            ranked = ranked[:max(1, int(np.count_nonzero(before < case['top_p'] * mass[-1])))]
        members = np.sort(ranked)
        mass = np.cumsum(w[members])
        at = np.minimum(np.searchsorted(mass, U[r] * mass[-1], side='right'), members.size - 1)
        index[r] = members[at]
        logp[r] = t[index[r]] - math.log(math.fsum(w[members]) if members.size < 1 << 20 else mass[-1])
    return dict(index=torch.from_numpy(index), logp=torch.from_numpy(logp))


def _exact_norm(s, case, eps=1e-5):
    x, w, b = s['x'].double(), s['weight'].double(), s['bias'].double()
    n = x.shape[1]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    r = (var + eps) ** -0.5
    out = dict(y=torch.addcmul(b, (x - mean) * r, w))
    if case['backward']:
        dy = s['dy'].double()
        z = (x - mean) * r
        q = dy * w
        out['dx'] = (r / n) * (n * q - q.sum(1, keepdim=True) - z * (q * z).sum(1, keepdim=True))
        out['dweight'], out['dbias'] = torch.einsum('ij,ij->j', dy, z), dy.sum(0)
    return out


def _exact_gated(s, case):
    x, wg, wu = s['x'].double(), s['w_gate'].double(), s['w_up'].double()
    gate, up = torch.nn.functional.linear(x, wg), torch.nn.functional.linear(x, wu)
    if case['act'] == 'silu':
        sig = torch.sigmoid(gate)
        slope = sig + gate * sig * torch.sigmoid(-gate)
        on = gate * sig
    else:
        cdf = 0.5 * torch.erfc(-gate / math.sqrt(2.0))
        slope = cdf + gate * torch.exp(-gate * gate / 2.0) / math.sqrt(2.0 * math.pi)
        on = gate * cdf
    out = dict(h=on * up)
    if case['backward']:
        dh = s['dh'].double()
        both = torch.cat((dh * up * slope, dh * on), dim=1)
        out['dx'] = torch.mm(both, torch.cat((wg, wu), dim=0))
        dw = torch.mm(both.t(), x)
        out['dw_gate'], out['dw_up'] = dw[:case['hidden']], dw[case['hidden']:]
    return out


def _exact_inputs(s, case):
    """Pair by pair along one input column at a time, on the host."""
    from scipy.linalg import cho_factor, cho_solve
    X, y, theta, n = s['X'], s['y'], s['theta'], case['n']
    sq = [(X[:, t][:, None] - X[:, t][None, :]) / theta[t] for t in range(case['d'])]
    D = sum(q * q for q in sq)
    if case['kernel'] == 'rbf':
        K = np.exp(-D / 2.0)
        F = K.copy()
    else:
        r = np.sqrt(D)
        K = (1.0 + math.sqrt(5.0) * r + 5.0 * D / 3.0) * np.exp(-math.sqrt(5.0) * r)
        F = 5.0 / 3.0 * (1.0 + math.sqrt(5.0) * r) * np.exp(-math.sqrt(5.0) * r)
    K[np.diag_indices(n)] += case['sigma'] ** 2
    c = cho_factor(K, lower=True)
    a = cho_solve(c, y)
    G = cho_solve(c, np.eye(n))
    G = (np.outer(a, a) * (n / y.dot(a)) - G) * F
    nll = 0.5 * n * (math.log(2.0 * math.pi) + 1.0 + math.log(y.dot(a) / n)) + np.log(np.diag(c[0])).sum()
    gx = np.stack([(G * q).sum(axis=1) / theta[t] for t, q in enumerate(sq)], axis=1)
    gt = np.array([-0.5 * (G * q * q).sum() / theta[t] for t, q in enumerate(sq)])
    return dict(nll=float(nll), grad_theta=gt, grad_X=gx)


def exact(case, seed):
    state = prepare(case, seed)
    return {'draw': _exact_draw, 'norm': _exact_norm, 'gated': _exact_gated, 'inputs': _exact_inputs}[case['op']](state, case)
