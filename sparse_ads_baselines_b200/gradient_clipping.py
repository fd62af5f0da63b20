"""The global norm of a list of gradients, and clipping by it.

The tables' own gradient never exists as a tensor -- the backward applies the optimizer as it goes -- but
the rest of a model (dense layers, experts, a router) is trained from ordinary gradients, and
``TableBatchedEmbeddingBags(max_grad_norm=...)`` limits the pooled gradient in front of the tables with the
same kernels.

Nothing synchronises: the norm stays on the device.  Everything is enqueued on the current CUDA stream of
the tensors' device.  There is no CPU path, and nothing is recorded: not by autograd (the norm is a constant to
it), not in forward mode (a tangent is refused), not by torch.jit.trace or make_fx (refused; torch.compile leaves
the graph around the call).  All tensors of a list lie on one device, and each fills its memory without gaps: a
column slice, which PyTorch's own clipping takes, is refused.
"""
import torch

from . import _lib


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


def _as_list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else tensors if isinstance(tensors, list) else list(tensors)


def grad_norm(tensors):
    """The 2-norm over all elements of ``tensors`` (a tensor or an iterable; None entries are left out), a
    float32 scalar on their device (inf where it passes float32's range).  Squares are summed in float64, those
    of 16-bit values eight at a time in float32; squares of float64 values beyond 1.8e308 or below 5e-324 leave its
    range.  An empty list has norm 0."""
    return _lib.glue().grad_norm(_as_list(tensors))


def clip_grad_norm(tensors, max_norm, eps=1e-6, out=None):
    """Scales ``tensors`` by ``min(1, max_norm / (norm + eps))`` and returns ``norm``, the 2-norm over all of
    them as they came in (see :func:`grad_norm`).

    In place, or, with ``out`` (as many tensors, of the same shapes, strides and types), into ``out``.  Norm and
    factor are taken in float64; the factor is rounded to float32 (not for float64 tensors), so is its product
    with an element, and the result to the element's type.  A norm of NaN makes every element NaN and one that is
    infinite in float64 every finite element 0, as the formula says: nothing is checked on the host.  A list in
    which two tensors share memory is refused, since an element must not be scaled twice."""
    if out is not None:
        if isinstance(tensors, torch.Tensor) != isinstance(out, torch.Tensor):
            raise RuntimeError("out must be a tensor or a list like tensors")
        out = _as_list(out)
    return _lib.glue().clip_grad_norm(_as_list(tensors), max_norm, eps, out)
