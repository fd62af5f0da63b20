"""The global norm of a list of gradients, and clipping by it.

The tables' own gradient never exists as a tensor -- the backward applies the optimizer as it goes -- but
the rest of a model (dense layers, experts, a router) is trained from ordinary gradients, and
``TableBatchedEmbeddingBags(max_grad_norm=...)`` limits the pooled gradient in front of the tables with the
same kernels.

Nothing synchronises: the norm stays on the device.  Everything is enqueued on the current CUDA stream of
the tensors' device.  There is no CPU path.
"""
from array import array

import torch

from . import _lib
from .expert_routing import _DTYPES, _call
from .table_batched_embeddings import _require


def _dense(t):
    """Whether the elements of ``t`` fill one stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _same_order(a, b):
    return a.stride() == b.stride() or all(n == 1 or i == j for n, i, j in zip(a.shape, a.stride(), b.stride()))


def _check_list(name, tensors):
    """The tensors of the list that are not None, and their common device (None: an empty list)."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else [t for t in tensors if t is not None]
    for t in tensors:
        _require(isinstance(t, torch.Tensor) and t.is_cuda, "%s must be CUDA tensors (this library has no CPU path)" % name)
        _require(t.layout == torch.strided and t.dtype in _DTYPES,
                 "%s must be dense float16, bfloat16, float32 or float64 tensors" % name)
        _require(_dense(t), "%s must fill their memory without gaps or repeats (got strides %s for %s)"
                 % (name, tuple(t.stride()), tuple(t.shape)))
    devices = {t.device for t in tensors}
    _require(len(devices) <= 1, "%s are on several devices" % name)
    return tensors, devices.pop() if devices else None


def _table(tensors):
    return (array("Q", [t.data_ptr() for t in tensors]), array("q", [t.numel() for t in tensors]),
            array("i", [_DTYPES[t.dtype] for t in tensors]))


def _address(a):
    return a.buffer_info()[0]


def _workspace(count, device):
    # a buffer of this call: calls on other streams and captured graphs have their own
    return torch.empty(_lib.lib().tbe_grad_norm_workspace_bytes(count), dtype=torch.uint8, device=device)


def grad_norm(tensors):
    """The 2-norm over all elements of ``tensors`` (a tensor or an iterable; None entries are left out), a
    float32 scalar on their device.  Sums are kept in float64.  An empty list has norm 0."""
    tensors, device = _check_list("tensors", tensors)
    if device is None:
        return torch.zeros((), device=torch.device("cuda", torch.cuda.current_device()))
    ptrs, sizes, dtypes = _table(tensors)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        ws = _workspace(len(tensors), device)
    _call(device, "tbe_grad_norm", _address(ptrs), _address(sizes), _address(dtypes), len(tensors), norm.data_ptr(),
          ws.data_ptr(), ws.numel())
    return norm


def clip_grad_norm(tensors, max_norm, eps=1e-6, out=None):
    """Scales ``tensors`` by ``min(1, max_norm / (norm + eps))`` and returns ``norm``, the 2-norm over all of
    them as they came in (see :func:`grad_norm`).

    In place, or, with ``out`` (as many tensors, of the same shapes, strides and types), into ``out``.  Every
    element is rounded once.  A norm of NaN makes every element NaN and an infinite one every finite element
    0, as the formula says: nothing is checked on the host.  A list in which two tensors share memory is
    refused, since an element must not be scaled twice."""
    max_norm, eps = float(max_norm), float(eps)
    _require(max_norm >= 0 and eps >= 0, "max_norm and eps must not be negative")
    if out is not None:
        _require(isinstance(tensors, torch.Tensor) == isinstance(out, torch.Tensor),
                 "out must be a tensor or a list like tensors")
        tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        _require(len(tensors) == len(out), "out must have as many entries as tensors")
        out = [o for t, o in zip(tensors, out) if t is not None]
    tensors, device = _check_list("tensors", tensors)
    if device is None:
        return torch.zeros((), device=torch.device("cuda", torch.cuda.current_device()))
    ptrs, sizes, dtypes = _table(tensors)
    to = ptrs
    if out is not None:
        for t, o in zip(tensors, out):
            _require(isinstance(o, torch.Tensor) and o.device == device and o.dtype == t.dtype and o.shape == t.shape
                     and _same_order(o, t), "out must match tensors in device, type, shape and strides")
        to = array("Q", [o.data_ptr() for o in out])
    norm = torch.empty((), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        ws = _workspace(len(tensors), device)
    _call(device, "tbe_grad_clip", _address(ptrs), _address(to), _address(sizes), _address(dtypes), len(tensors), max_norm,
          eps, norm.data_ptr(), ws.data_ptr(), ws.numel())
    return norm
