"""Learned inputs: a map in front of the covariance for data with more columns than length scales can be fitted for (the
measured spectra have 621 channels, BayesOpt/BayesOpt_v4.ipynb:681-697; gradients are supported up to 16 input columns).

``layer_norm`` and ``gated_unit`` and their backward passes run on torch tensors on a GPU, on the current stream, without
waiting for it.  They are not recorded by torch's autograd: a tensor that requires a gradient is taken with a warning, unless gradients
are off, and the backward passes are called by hand.  ``FeatureMap`` puts them together: normalise a row, one gated unit, a few features.
``hyperopt.lml_features`` differentiates the likelihood through it."""
from __future__ import annotations

import numpy as np
import torch

from . import _lib as L
from ._device import TYPES, check_status, off_tape, pointer, rows_of, scratch, stream_of, tensor, vector_of, workspace

ACTIVATIONS = {'silu': L.ACT_SILU, 'gelu': L.ACT_GELU}
_like, _f32 = torch.empty_like, torch.float32


def _act(act):
    a = ACTIVATIONS.get(act)
    if a is None:
        raise ValueError('act must be one of %s; got %r' % (sorted(ACTIVATIONS), act))
    return a


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the rows of x (rows, cols) float32 / bfloat16 / float16; weight and bias
    (cols,) of x's type or None.  Returns y, mean (rows,) and rstd (rows,), the last two float32, for layer_norm_backward."""
    rows, cols, stride, at = rows_of('x', x)
    dtype = x.dtype
    if weight is not None:
        weight = vector_of('weight', weight, cols, dtype, at)
    if bias is not None:
        bias = vector_of('bias', bias, cols, dtype, at)
    if not 0.0 <= eps < float('inf'):
        raise ValueError('eps must be finite and >= 0; got %r' % (eps,))
    y = _like(x) if stride == cols else x.new_empty((rows, cols))
    mean, rstd = x.new_empty(rows, dtype=_f32), x.new_empty(rows, dtype=_f32)
    st = L.load().gpbo_layernorm(at, stream_of(at), TYPES[dtype], x.data_ptr(), stride, rows, cols, pointer(weight), pointer(bias), eps,
                                 y.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr())
    if st:
        check_status('gpbo_layernorm', st)
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd):
    """Gradients (dx, dweight, dbias) of layer_norm from dy, with the mean and rstd it returned.  dweight and dbias have x's
    type; they are the column sums whether or not the forward pass had a weight and a bias."""
    rows, cols, stride, at = rows_of('x', x)
    dtype = x.dtype
    dstride = rows_of('dy', dy, dtype=dtype, shape=(rows, cols), device=at)[2]
    if weight is not None:
        weight = vector_of('weight', weight, cols, dtype, at)
    mean, rstd = vector_of('mean', mean, rows, _f32, at), vector_of('rstd', rstd, rows, _f32, at)
    code = TYPES[dtype]
    dx = _like(x) if stride == cols else x.new_empty((rows, cols))
    dw, db = x.new_empty(cols), x.new_empty(cols)
    nbytes = workspace('gpbo_layernorm_backward_workspace', code, rows, cols)
    work = scratch(nbytes, x.device)
    st = L.load().gpbo_layernorm_backward(at, stream_of(at), code, dy.data_ptr(), dstride, x.data_ptr(), stride, rows, cols, pointer(weight),
                                          mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, dw.data_ptr(), db.data_ptr(), pointer(work), nbytes)
    if st:
        check_status('gpbo_layernorm_backward', st)
    return dx, dw, db


def _weights(x, w_gate, w_up):
    rows, cols, stride, at = rows_of('x', x)
    hidden, wcols, wg_stride, _ = rows_of('w_gate', w_gate, dtype=x.dtype, device=at)
    if wcols != cols or hidden < 1:
        raise ValueError('w_gate must be (hidden, %d) with hidden >= 1; got %s' % (cols, tuple(w_gate.shape)))
    wu_stride = rows_of('w_up', w_up, dtype=x.dtype, shape=(hidden, cols), device=at)[2]
    if wg_stride != wu_stride:      # one row stride for both: weights laid out apart are brought together
        w_gate, w_up, wg_stride = w_gate.contiguous(), w_up.contiguous(), cols
    return rows, cols, stride, at, hidden, w_gate, w_up, wg_stride


def gated_unit(x, w_gate, w_up, act='silu', keep=False):
    """act(x w_gate^T) * (x w_up^T): x (rows, cols) float32 / bfloat16 / float16, w_gate and w_up (hidden, cols) of the same type;
    act 'silu' or 'gelu'.  keep: also return x w_gate^T and x w_up^T as one (2, rows, hidden) float32 tensor, which
    gated_unit_backward needs."""
    a = _act(act)
    rows, cols, stride, at, hidden, w_gate, w_up, ws = _weights(x, w_gate, w_up)
    dtype = x.dtype
    code = TYPES[dtype]
    h = x.new_empty((rows, hidden))
    kept = kg = ku = None
    if keep:
        kept = x.new_empty((2, rows, hidden), dtype=_f32)
        kg = kept.data_ptr()
        ku = kg + 4 * rows * hidden
    nbytes = workspace('gpbo_gated_workspace', code, rows, cols, hidden)
    if nbytes:      # that is for operands that have to be copied first
        nbytes = L.load().gpbo_gated_workspace_for(code, x.data_ptr(), stride, rows, cols, w_gate.data_ptr(), w_up.data_ptr(), ws, hidden)
    work = scratch(nbytes, x.device)
    st = L.load().gpbo_gated(at, stream_of(at), code, a, x.data_ptr(), stride, rows, cols, w_gate.data_ptr(), w_up.data_ptr(), ws, hidden,
                             h.data_ptr(), hidden, kg, ku, pointer(work), nbytes)
    if st:
        check_status('gpbo_gated', st)
    return (h, kept) if keep else h


def gated_unit_backward(dh, x, w_gate, w_up, kept, act='silu', need_dx=True, need_dw=True):
    """Gradients (dx, dw_gate, dw_up) of gated_unit from dh (rows, hidden), with what it kept; None for those not needed.  In 16 bits the
    gradients of the two projections are rounded to x's type on the way, in large problems: errors 1.4 times a single rounding's."""
    a = _act(act)
    rows, cols, stride, at, hidden, w_gate, w_up, ws = _weights(x, w_gate, w_up)
    dtype = x.dtype
    code = TYPES[dtype]
    dstride = rows_of('dh', dh, dtype=dtype, shape=(rows, hidden), device=at)[2]
    tensor('kept', kept, at)
    if tuple(kept.shape) != (2, rows, hidden) or kept.dtype != _f32:
        raise ValueError('kept must be (2, %d, %d) float32; got %s %s' % (rows, hidden, tuple(kept.shape), kept.dtype))
    if not kept.is_contiguous():
        kept = kept.contiguous()
    kg = kept.data_ptr()
    dx = (_like(x) if stride == cols else x.new_empty((rows, cols))) if need_dx else None
    dwg = x.new_empty((hidden, cols)) if need_dw else None
    dwu = x.new_empty((hidden, cols)) if need_dw else None
    nbytes = workspace('gpbo_gated_backward_workspace', code, rows, cols, hidden)
    work = scratch(nbytes, x.device)
    st = L.load().gpbo_gated_backward(at, stream_of(at), code, a, dh.data_ptr(), dstride, x.data_ptr(), stride, rows, cols, w_gate.data_ptr(),
                                      w_up.data_ptr(), ws, hidden, kg, kg + 4 * rows * hidden, pointer(dx), cols, pointer(dwg), pointer(dwu),
                                      cols, pointer(work), nbytes)
    if st:
        check_status('gpbo_gated_backward', st)
    return dx, dwg, dwu


def _exponent(dh):
    """The power of two, as a tensor, that brings the largest finite element between 2^-11 and 2^14, where float16 holds it and most of what is
    smaller; 0 if it lies there."""
    most = torch.where(torch.isfinite(dh), dh, 0.0).abs().amax() if dh.numel() else dh.new_zeros(())
    at = torch.frexp(most).exponent
    return torch.where(most > 0, at.clamp(-10, 14) - at, 0)


class FeatureMap:
    """z = gated_unit(layer_norm(x)) @ w_out^T: the inputs of a GP as a learned function of raw ones.  ``params`` holds the five
    tensors (norm_weight, norm_bias, w_gate, w_up, w_out), which may be parameters; an optimiser of the caller's choice updates them in
    place, with the gradients that backward() returns."""

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
        if getattr(x, 'requires_grad', False):
            off_tape('x', x)
        with torch.no_grad():
            y, mean, rstd = layer_norm(x, p['norm_weight'], p['norm_bias'], self.eps)
            h = gated_unit(y, p['w_gate'], p['w_up'], self.act, keep=keep)
            h, kept = h if keep else (h, None)
            z = h.float() @ p['w_out'].float().t()
        return (z, (x, mean, rstd, y, kept, h)) if keep else z

    @torch.no_grad()
    def backward(self, dz, saved):
        """Gradients of the parameters, by name, and of x, under 'x'; dz (rows, features) float32."""
        p = self.params
        x, mean, rstd, y, kept, h = saved
        dz = dz.float()
        dh = dz @ p['w_out'].float()
        ranged = h.dtype == torch.float16      # a likelihood's gradient knows no bounds: the passes through float16 are taken on a multiple of it
        if ranged:
            e = _exponent(dh)
            dh = torch.ldexp(dh, e)
        dy, dwg, dwu = gated_unit_backward(dh.to(h.dtype), y, p['w_gate'], p['w_up'], kept, self.act)
        dx, dw, db = layer_norm_backward(dy, x, p['norm_weight'], mean, rstd)
        grads = {'norm_weight': dw, 'norm_bias': db, 'w_gate': dwg, 'w_up': dwu, 'x': dx}
        if ranged:
            grads = {k: torch.ldexp(v.float(), -e).to(v.dtype) for k, v in grads.items()}
        grads['w_out'] = (dz.t() @ h.float()).to(h.dtype)
        return grads

    def numpy(self, x):
        """Features of host rows as the float64 array GP.fit and GP.set_candidates take."""
        w = self.params['w_gate']
        z = self.forward(torch.as_tensor(np.ascontiguousarray(x), device=w.device).to(w.dtype).contiguous())
        return z.double().cpu().numpy()
