"""What the operators on caller-owned GPU tensors share: checks of tensors, workspaces, streams and status codes."""
from __future__ import annotations

import torch

from . import _lib as L
from .gp import GpboError

TYPES = {torch.float32: L.TYPE_F32, torch.bfloat16: L.TYPE_BF16, torch.float16: L.TYPE_F16}


def on_device(name, t, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(t).__name__))
    if t.device != device:
        raise ValueError('%s is on %s, expected %s' % (name, t.device, device))


def rows_of(name, t, types=TYPES, dtype=None, shape=None, device=None):
    """(rows, cols, row stride) of a 2-D GPU tensor whose rows are contiguous; anything else is refused."""
    if not isinstance(t, torch.Tensor):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(t).__name__))
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError('%s must be %s; got shape %s' % (name, '2-D' if shape is None else tuple(shape), tuple(t.shape)))
    if t.dtype not in types or (dtype is not None and t.dtype != dtype):
        raise ValueError('%s must be %s; got %s' % (name, ' / '.join(str(v) for v in types) if dtype is None else dtype, t.dtype))
    if t.device.type != 'cuda' or (device is not None and t.device != device):
        raise ValueError('%s is on %s, expected %s (there is no CPU path)' % (name, t.device, 'a GPU' if device is None else device))
    rows, cols = t.shape
    if cols < 1:
        raise ValueError('%s has no columns' % name)
    if cols > 1 and t.stride(1) != 1:
        raise ValueError('%s: the elements of a row must be contiguous; got strides %s' % (name, tuple(t.stride())))
    stride = t.stride(0) if rows > 1 else cols
    if stride < cols:
        raise ValueError('%s: rows overlap; got strides %s' % (name, tuple(t.stride())))
    return rows, cols, stride


def vector_of(name, t, cols, dtype, device):
    """A contiguous (cols,) tensor or None."""
    if t is None:
        return None
    on_device(name, t, device)
    if t.shape != (cols,) or t.dtype != dtype:
        raise ValueError('%s must be (%d,) %s; got %s %s' % (name, cols, dtype, tuple(t.shape), t.dtype))
    return t.contiguous()


def workspace(nbytes, device):
    """A scratch tensor of a call's own (torch's allocator keeps it for the stream, and for a graph that is being captured)."""
    if nbytes < 0:
        raise ValueError('these sizes are out of range')
    return (torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes) if nbytes else (None, 0)


def pointer(t):
    return None if t is None else t.data_ptr()


def stream_of(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def check_status(name, st):
    if st == L.OK:
        return
    if st == L.ERR_BAD_ARG:
        raise ValueError('%s: bad arguments' % name)
    raise GpboError('%s: HIP error (status %d)' % (name, st))
