"""Draws from scores: the stochastic counterpart of the argmax pick (BayesOpt/BayesOpt_v4.ipynb:647), for rows of scores that
are on the GPU as torch tensors.  ``GP.draw`` / ``MultiGP.draw`` do the same on the acquisition values of a context."""
from __future__ import annotations

import math

import torch

from . import _lib as L
from ._device import TYPES, check_status, on_device, pointer, rows_of, stream_of, workspace

_TYPES = dict(TYPES)
_TYPES[torch.float64] = L.TYPE_F64


def _setting(name, v, rows, device):
    """A Python number, or a tensor of one number per row."""
    if isinstance(v, torch.Tensor) and v.dim() > 0:
        if v.shape != (rows,) or v.device != device:
            raise ValueError('%s must be a number or a (%d,) tensor on %s; got %s on %s' % (name, rows, device, tuple(v.shape), v.device))
        return v.detach().to(torch.float64)
    return float(v)


def sample(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One index per uniform number from softmax(scores / temperature), row by row.

    scores (rows, cols) float64 / float32 / bfloat16 / float16 on a GPU, elements of a row contiguous; u (rows, draws) float64
    in [0, 1) on the same GPU.  NaN and -inf are never drawn.  Kept are the top_k best (0: all), of those the ones whose
    weight is at least min_p times the best one's, of those the shortest run from the best down that holds top_p of their
    mass; equal scores rank by index.  A draw is the lowest kept index whose running mass, in index order, exceeds u times the
    whole.  temperature = 0 takes the best score.  Each setting is a number, or a (rows,) tensor on the same GPU.
    Returns (index (rows, draws) int64, logp (rows, draws) float64); index -1 and logp -inf in a row with nothing to draw.
    Runs on the current stream and does not wait for it."""
    rows, cols, stride = rows_of('scores', scores, _TYPES)
    on_device('u', u, scores.device)
    if u.dim() != 2 or u.shape[0] != rows or u.dtype != torch.float64:
        raise ValueError('u must be (%d, draws) float64; got %s %s' % (rows, tuple(u.shape), u.dtype))
    settings = [_setting(n, v, rows, scores.device) for n, v in
                (('temperature', temperature), ('top_k', top_k), ('top_p', top_p), ('min_p', min_p))]
    params = None
    if any(isinstance(v, torch.Tensor) for v in settings):
        params = torch.stack([v if isinstance(v, torch.Tensor) else torch.full((rows,), v, dtype=torch.float64, device=scores.device)
                              for v in settings], dim=1).contiguous()
        settings = [1.0, 0, 1.0, 0.0]
    t, k, tp, mp = settings
    if not (t >= 0.0 and math.isfinite(t)):
        raise ValueError('temperature must be finite and >= 0; got %r' % (t,))
    if not (k >= 0 and k == int(k)):
        raise ValueError('top_k must be a whole number >= 0; got %r' % (k,))
    if not (0.0 <= tp <= 1.0 and 0.0 <= mp <= 1.0):
        raise ValueError('top_p and min_p must lie in [0, 1]; got %r and %r' % (tp, mp))
    u = u.contiguous()
    draws = u.shape[1]
    lib = L.load()
    index = torch.empty((rows, draws), dtype=torch.int64, device=scores.device)
    logp = torch.empty((rows, draws), dtype=torch.float64, device=scores.device)
    work, nbytes = workspace(lib.gpbo_draw_static_workspace(_TYPES[scores.dtype], rows, cols, draws), scores.device)
    check_status('gpbo_draw_static', lib.gpbo_draw_static(
        scores.device.index, stream_of(scores), _TYPES[scores.dtype], scores.data_ptr(), stride, rows, cols, u.data_ptr(), draws, t,
        min(int(k), 1 << 62), tp, mp, pointer(params), index.data_ptr(), logp.data_ptr(), pointer(work), nbytes))
    return index, logp
