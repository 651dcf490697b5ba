"""What the operators on caller-owned GPU tensors share: checks of tensors, workspaces, streams and status codes.

A call on a few rows takes less time on the GPU than its checks take here, so the checks look at each attribute once and compare
device numbers, and results are allocated one by one rather than sliced out of each other."""
from __future__ import annotations

import warnings

import torch

from . import _lib as L
from .gp import GpboError

TYPES = {torch.float32: L.TYPE_F32, torch.bfloat16: L.TYPE_BF16, torch.float16: L.TYPE_F16}
Tensor = torch.Tensor

_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def stream_of(device: int):
    """The current stream of that GPU, as a hipStream_t."""
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def off_tape(name, t):
    """These calls are not part of torch's graph of gradients: says so where one would be expected."""
    if t.requires_grad and torch.is_grad_enabled():
        warnings.warn('%s requires a gradient, but this call is not recorded: backward() will not reach %s through it (call the operator\'s own '
                      'backward pass, under torch.no_grad())' % (name, name), stacklevel=4)


def tensor(name, t, device=None):
    """The number of the GPU that t is on; it must be `device` if one is given."""
    if not isinstance(t, Tensor):
        raise TypeError('%s must be a torch tensor, got %s' % (name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError('%s is on %s, expected a GPU (there is no CPU path)' % (name, t.device))
    if t.requires_grad:
        off_tape(name, t)
    at = t.get_device()
    if device is not None and at != device:
        raise ValueError('%s is on %s, expected cuda:%d' % (name, t.device, device))
    return at


def rows_of(name, t, types=TYPES, dtype=None, shape=None, device=None):
    """(rows, cols, row stride, GPU) of a 2-D GPU tensor whose rows are contiguous; anything else is refused."""
    at = tensor(name, t, device)
    size = t.shape
    if len(size) != 2 or (shape is not None and tuple(size) != shape):
        raise ValueError('%s must be %s; got shape %s' % (name, '2-D' if shape is None else shape, tuple(size)))
    if (t.dtype not in types) if dtype is None else (t.dtype != dtype):
        raise ValueError('%s must be %s; got %s' % (name, ' / '.join(str(v) for v in types) if dtype is None else dtype, t.dtype))
    rows, cols = size
    if cols < 1:
        raise ValueError('%s has no columns' % name)
    stride, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError('%s: the elements of a row must be contiguous; got strides %s' % (name, tuple(t.stride())))
    if rows <= 1:
        stride = cols
    elif stride < cols:
        raise ValueError('%s: rows overlap; got strides %s' % (name, tuple(t.stride())))
    return rows, cols, stride, at


def vector_of(name, t, n, dtype, device):
    """A contiguous (n,) tensor."""
    tensor(name, t, device)
    if t.dtype != dtype or tuple(t.shape) != (n,):
        raise ValueError('%s must be (%d,) %s; got %s %s' % (name, n, dtype, tuple(t.shape), t.dtype))
    return t if t.is_contiguous() else t.contiguous()


_sizes = {}


def workspace(size_of, *sizes):
    """Bytes that `size_of` (a *_workspace function of the library) names for these sizes; asked once for the same ones."""
    key = (size_of, sizes)
    n = _sizes.get(key)
    if n is None:
        n = getattr(L.load(), size_of)(*sizes)
        if n < 0:
            raise ValueError('%s: these sizes are out of range: %s' % (size_of, sizes[1:]))
        if len(_sizes) > 4096:
            _sizes.clear()
        _sizes[key] = n
    return n


def scratch(nbytes, device):
    """A scratch tensor of a call's own (torch's allocator keeps it for the stream, and for a graph that is being captured)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def pointer(t):
    return None if t is None else t.data_ptr()


def check_status(name, st):
    if st == L.ERR_BAD_ARG:
        raise ValueError('%s: bad arguments' % name)
    raise GpboError('%s: HIP error (status %d)' % (name, st))
