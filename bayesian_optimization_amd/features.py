"""Learned inputs: a map in front of the covariance for data with more columns than length scales can be fitted for (the
measured spectra have 621 channels, BayesOpt/BayesOpt_v4.ipynb:681-697; gradients are supported up to 16 input columns).

``layer_norm`` and ``gated_unit`` and their backward passes run on torch tensors on a GPU, on the current stream, without
waiting for it.  ``FeatureMap`` puts them together: normalise a row, one gated unit, a few features.
``hyperopt.lml_features`` differentiates the likelihood through it."""
from __future__ import annotations

import numpy as np
import torch

from . import _lib as L
from ._device import TYPES, check_status, on_device, pointer, rows_of, stream_of, vector_of, workspace

ACTIVATIONS = {'silu': L.ACT_SILU, 'gelu': L.ACT_GELU}


def _act(act):
    if act not in ACTIVATIONS:
        raise ValueError('act must be one of %s; got %r' % (sorted(ACTIVATIONS), act))
    return ACTIVATIONS[act]


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the rows of x (rows, cols) float32 / bfloat16 / float16; weight and bias
    (cols,) of x's type or None.  Returns y, mean (rows,) and rstd (rows,), the last two float32, for layer_norm_backward."""
    rows, cols, stride = rows_of('x', x)
    weight, bias = vector_of('weight', weight, cols, x.dtype, x.device), vector_of('bias', bias, cols, x.dtype, x.device)
    if not 0.0 <= float(eps) < float('inf'):
        raise ValueError('eps must be finite and >= 0; got %r' % (eps,))
    y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    check_status('gpbo_layernorm', L.load().gpbo_layernorm(
        x.device.index, stream_of(x), TYPES[x.dtype], x.data_ptr(), stride, rows, cols, pointer(weight), pointer(bias), float(eps),
        y.data_ptr(), cols, stats[0].data_ptr(), stats[1].data_ptr()))
    return y, stats[0], stats[1]


def layer_norm_backward(dy, x, weight, mean, rstd):
    """Gradients (dx, dweight, dbias) of layer_norm from dy, with the mean and rstd it returned.  dweight and dbias have x's
    type; they are the column sums whether or not the forward pass had a weight and a bias."""
    rows, cols, stride = rows_of('x', x)
    _, _, dstride = rows_of('dy', dy, dtype=x.dtype, shape=(rows, cols), device=x.device)
    weight = vector_of('weight', weight, cols, x.dtype, x.device)
    mean, rstd = vector_of('mean', mean, rows, torch.float32, x.device), vector_of('rstd', rstd, rows, torch.float32, x.device)
    if mean is None or rstd is None:
        raise ValueError('mean and rstd of the forward pass are needed')
    lib = L.load()
    dx = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    dwb = torch.empty((2, cols), dtype=x.dtype, device=x.device)
    work, nbytes = workspace(lib.gpbo_layernorm_backward_workspace(TYPES[x.dtype], rows, cols), x.device)
    check_status('gpbo_layernorm_backward', lib.gpbo_layernorm_backward(
        x.device.index, stream_of(x), TYPES[x.dtype], dy.data_ptr(), dstride, x.data_ptr(), stride, rows, cols, pointer(weight),
        mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, dwb[0].data_ptr(), dwb[1].data_ptr(), pointer(work), nbytes))
    return dx, dwb[0], dwb[1]


def _weights(x, w_gate, w_up):
    rows, cols, stride = rows_of('x', x)
    on_device('w_gate', w_gate, x.device)
    if w_gate.dim() != 2 or w_gate.shape[0] < 1 or w_gate.shape[1] != cols:
        raise ValueError('w_gate must be (hidden, %d) with hidden >= 1; got %s' % (cols, tuple(w_gate.shape)))
    hidden, _, wg_stride = rows_of('w_gate', w_gate, dtype=x.dtype, device=x.device)
    _, _, wu_stride = rows_of('w_up', w_up, dtype=x.dtype, shape=(hidden, cols), device=x.device)
    if wg_stride != wu_stride:      # one row stride for both: weights laid out apart are brought together
        w_gate, w_up, wg_stride = w_gate.contiguous(), w_up.contiguous(), cols
    return rows, cols, stride, hidden, w_gate, w_up, wg_stride


def gated_unit(x, w_gate, w_up, act='silu', keep=False):
    """act(x w_gate^T) * (x w_up^T): x (rows, cols) float32 / bfloat16 / float16, w_gate and w_up (hidden, cols) of the same type;
    act 'silu' or 'gelu'.  keep: also return x w_gate^T and x w_up^T as one (2, rows, hidden) float32 tensor, which
    gated_unit_backward needs."""
    a = _act(act)
    rows, cols, stride, hidden, w_gate, w_up, ws = _weights(x, w_gate, w_up)
    lib = L.load()
    h = torch.empty((rows, hidden), dtype=x.dtype, device=x.device)
    kept = torch.empty((2, rows, hidden), dtype=torch.float32, device=x.device) if keep else None
    work, nbytes = workspace(lib.gpbo_gated_workspace(TYPES[x.dtype], rows, cols, hidden), x.device)
    check_status('gpbo_gated', lib.gpbo_gated(
        x.device.index, stream_of(x), TYPES[x.dtype], a, x.data_ptr(), stride, rows, cols, w_gate.data_ptr(), w_up.data_ptr(), ws, hidden,
        h.data_ptr(), hidden, kept[0].data_ptr() if keep else None, kept[1].data_ptr() if keep else None, pointer(work), nbytes))
    return (h, kept) if keep else h


def gated_unit_backward(dh, x, w_gate, w_up, kept, act='silu', need_dx=True, need_dw=True):
    """Gradients (dx, dw_gate, dw_up) of gated_unit from dh (rows, hidden), with what it kept; None for those not needed."""
    a = _act(act)
    rows, cols, stride, hidden, w_gate, w_up, ws = _weights(x, w_gate, w_up)
    _, _, dstride = rows_of('dh', dh, dtype=x.dtype, shape=(rows, hidden), device=x.device)
    on_device('kept', kept, x.device)
    if kept.shape != (2, rows, hidden) or kept.dtype != torch.float32:
        raise ValueError('kept must be (2, %d, %d) float32; got %s %s' % (rows, hidden, tuple(kept.shape), kept.dtype))
    kept = kept.contiguous()
    lib = L.load()
    dx = torch.empty((rows, cols), dtype=x.dtype, device=x.device) if need_dx else None
    dw = torch.empty((2, hidden, cols), dtype=x.dtype, device=x.device) if need_dw else None
    work, nbytes = workspace(lib.gpbo_gated_backward_workspace(TYPES[x.dtype], rows, cols, hidden), x.device)
    check_status('gpbo_gated_backward', lib.gpbo_gated_backward(
        x.device.index, stream_of(x), TYPES[x.dtype], a, dh.data_ptr(), dstride, x.data_ptr(), stride, rows, cols, w_gate.data_ptr(),
        w_up.data_ptr(), ws, hidden, kept[0].data_ptr(), kept[1].data_ptr(), pointer(dx), cols, dw[0].data_ptr() if need_dw else None,
        dw[1].data_ptr() if need_dw else None, cols, pointer(work), nbytes))
    return dx, (dw[0] if need_dw else None), (dw[1] if need_dw else None)


class FeatureMap:
    """z = gated_unit(layer_norm(x)) @ w_out^T: the inputs of a GP as a learned function of raw ones.  ``params`` holds the five
    tensors (norm_weight, norm_bias, w_gate, w_up, w_out); an optimiser of the caller's choice updates them in place."""

    def __init__(self, cols, hidden, features, dtype=torch.float32, device='cuda', act='silu', eps=1e-5, seed=0):
        if min(cols, hidden, features) < 1:
            raise ValueError('cols, hidden and features must be >= 1')
        self.act, self.eps = act, float(eps)
        _act(act)
        g = torch.Generator().manual_seed(seed)

        def normal(r, c):
            return (torch.randn(r, c, generator=g) * c ** -0.5).to(device=device, dtype=dtype)
        self.params = {'norm_weight': torch.ones(cols, dtype=dtype, device=device), 'norm_bias': torch.zeros(cols, dtype=dtype, device=device),
                       'w_gate': normal(hidden, cols), 'w_up': normal(hidden, cols), 'w_out': normal(features, hidden)}

    def forward(self, x, keep=False):
        """z (rows, features) float32; keep: also what backward() needs."""
        p = self.params
        y, mean, rstd = layer_norm(x, p['norm_weight'], p['norm_bias'], self.eps)
        h = gated_unit(y, p['w_gate'], p['w_up'], self.act, keep=keep)
        h, kept = h if keep else (h, None)
        z = h.float() @ p['w_out'].float().t()
        return (z, (x, mean, rstd, y, kept, h)) if keep else z

    def backward(self, dz, saved):
        """Gradients of the parameters, by name, and of x, under 'x'; dz (rows, features) float32."""
        p = self.params
        x, mean, rstd, y, kept, h = saved
        dz = dz.float()
        dh = (dz @ p['w_out'].float()).to(h.dtype)
        dy, dwg, dwu = gated_unit_backward(dh, y, p['w_gate'], p['w_up'], kept, self.act)
        dx, dw, db = layer_norm_backward(dy, x, p['norm_weight'], mean, rstd)
        return {'norm_weight': dw, 'norm_bias': db, 'w_gate': dwg, 'w_up': dwu, 'w_out': (dz.t() @ h.float()).to(h.dtype), 'x': dx}

    def numpy(self, x):
        """Features of host rows as the float64 array GP.fit and GP.set_candidates take."""
        w = self.params['w_gate']
        z = self.forward(torch.as_tensor(np.ascontiguousarray(x), device=w.device).to(w.dtype).contiguous())
        return z.double().cpu().numpy()
