"""Draws from scores: the stochastic counterpart of the argmax pick (BayesOpt/BayesOpt_v4.ipynb:647), for rows of scores that
are on the GPU as torch tensors.  ``GP.draw`` / ``MultiGP.draw`` do the same on the acquisition values of a context."""
from __future__ import annotations

import math

import torch

from . import _lib as L
from ._device import TYPES, Tensor, check_status, pointer, rows_of, scratch, stream_of, tensor, workspace

_TYPES = dict(TYPES)
_TYPES[torch.float64] = L.TYPE_F64
_f64 = torch.float64


_NAMES, _NEUTRAL = ('temperature', 'top_k', 'top_p', 'min_p'), (1.0, 0, 1.0, 0.0)


def _check(temperature, top_k, top_p, min_p):
    if not (temperature >= 0.0 and math.isfinite(temperature)):
        raise ValueError('temperature must be finite and >= 0; got %r' % (temperature,))
    if not (0 <= top_k < math.inf and top_k == int(top_k)):
        raise ValueError('top_k must be a whole number >= 0; got %r' % (top_k,))
    if not (0.0 <= top_p <= 1.0 and 0.0 <= min_p <= 1.0):
        raise ValueError('top_p and min_p must lie in [0, 1]; got %r and %r' % (top_p, min_p))


def _numbers(settings):
    """The four settings as plain numbers, checked; the neutral one for a tensor that is not on the host, which cannot be looked at
    without waiting for it."""
    numbers = tuple(v if not isinstance(v, Tensor) else v.item() if v.dim() == 0 and not v.is_cuda else neutral for v, neutral in zip(settings, _NEUTRAL))
    _check(*numbers)
    return numbers


def _per_row(settings, rows, device, at):
    """(rows, 4) float64 on the GPU from four settings, each a number or a tensor there of one number, or one per row."""
    columns = []
    for name, v, number in zip(_NAMES, settings, _numbers(settings)):
        if isinstance(v, Tensor) and (v.is_cuda or v.dim() > 0):
            tensor(name, v, at)
            if v.dim() > 0 and tuple(v.shape) != (rows,):
                raise ValueError('%s must be a number or a (%d,) tensor; got %s' % (name, rows, tuple(v.shape)))
            columns.append(v.detach().to(_f64).expand(rows))
        else:
            columns.append(torch.full((rows,), float(number), dtype=_f64, device=device))
    return torch.stack(columns, dim=1)


def sample(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One index per uniform number from softmax(scores / temperature), row by row.

    scores (rows, cols) float64 / float32 / bfloat16 / float16 on a GPU, elements of a row contiguous; u (rows, draws) float64
    in [0, 1) on the same GPU.  NaN and -inf are never drawn.  Kept are the top_k best (0: all), of those the ones whose
    weight is at least min_p times the best one's, of those the shortest run from the best down that holds top_p of their
    mass; equal scores rank by index.  A draw is the lowest kept index whose running mass, in index order, exceeds u times the
    whole; u beyond [0, 1) counts as the nearest end.  temperature = 0 takes the best score.  Each setting is a number, or a tensor on
    the same GPU of one number or one per row; what is out of range is refused in a number, and counts as the nearest end in a tensor there.
    Returns (index (rows, draws) int64, logp (rows, draws) float64); index -1 and logp -inf in a row with nothing to draw.
    Runs on the current stream and does not wait for it."""
    rows, cols, stride, at = rows_of('scores', scores, _TYPES)
    tensor('u', u, at)
    if u.dim() != 2 or u.shape[0] != rows or u.dtype != _f64:
        raise ValueError('u must be (%d, draws) float64; got %s %s' % (rows, tuple(u.shape), u.dtype))
    device, params = scores.device, None
    if isinstance(temperature, Tensor) or isinstance(top_k, Tensor) or isinstance(top_p, Tensor) or isinstance(min_p, Tensor):
        params = _per_row((temperature, top_k, top_p, min_p), rows, device, at)
        temperature, top_k, top_p, min_p = _NEUTRAL
    else:
        _check(temperature, top_k, top_p, min_p)
    if not u.is_contiguous():
        u = u.contiguous()
    draws, code = u.shape[1], _TYPES[scores.dtype]
    index = u.new_empty((rows, draws), dtype=torch.int64)
    logp = u.new_empty((rows, draws))
    nbytes = workspace('gpbo_draw_static_workspace', code, rows, cols, draws)
    work = scratch(nbytes, device)
    st = L.load().gpbo_draw_static(at, stream_of(at), code, scores.data_ptr(), stride, rows, cols, u.data_ptr(), draws, temperature,
                                   min(int(top_k), 1 << 62), top_p, min_p, pointer(params), index.data_ptr(), logp.data_ptr(), pointer(work), nbytes)
    if st:
        check_status('gpbo_draw_static', st)
    return index, logp
