"""Samples routed to experts: the router's gate, samples sorted by expert, and the way back.

    weights, experts = gate(logits, k)            # [N, k] softmax weights (float32) and expert ids (int32)
    p = plan(experts, num_experts)                # stable sort of the N*k choices by expert
    y = dispatch(x, p)                            # [N*k, D]: rows p.offsets[e]:p.offsets[e+1] are expert e's
    ...                                           # the experts' own layers, row block by row block
    out = combine(y, p, weights)                  # [N, D]: weighted sum over every sample's rows

``combine`` is the weighted pooled lookup of ``table_batched_embeddings.forward`` with the rows chosen by
the router, and ``plan`` the sort that its backward makes.  All four are differentiable where it makes
sense (``gate`` in its logits, ``dispatch`` in ``x``, ``combine`` in ``y`` and ``weights``), once; nothing
synchronises, no size depends on the data, and no result depends on the order in which a GPU serves
atomics.  float16, bfloat16, float32 and float64; weights are float32 (float64 for float64).  Everything is
enqueued on the current CUDA stream of the tensors' device.  There is no CPU path.

A choice of ``-1`` (or any id outside ``0 .. num_experts-1``, for instance an expert of another rank) is
nobody's: its row lies behind ``p.offsets[-1]``, ``dispatch`` fills it with zeros and ``combine`` leaves it
out.  ``gate`` gives ``-1`` for experts whose logit is ``-inf``.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .table_batched_embeddings import _check_cuda, _require, _stream

MAX_EXPERTS = 1024
MAX_CHOICES = 32

_DTYPES = {torch.float32: _lib.TBE_F32, torch.float16: _lib.TBE_F16, torch.float64: _lib.TBE_F64,
           torch.bfloat16: _lib.TBE_BF16}


class ExpertPlan(NamedTuple):
    """Where every choice goes: ``offsets`` int32 ``[E+1]`` (rows of every expert), ``positions`` int32
    ``[N, k]`` (row of every choice) and ``order`` int32 ``[N*k]`` (the choice ``t*k + s`` in every row)."""
    offsets: torch.Tensor
    positions: torch.Tensor
    order: torch.Tensor


def _call(device, name, *args):
    """``_lib.call`` on the current stream of ``device``, whichever device is current."""
    if torch.cuda.current_device() == device.index:
        _lib.call(name, *args, _stream(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _stream(device))


def _weights_dtype(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _rows(name, t):
    """A detached view or copy of the 2-D ``t`` whose rows are dense."""
    _check_cuda(name, t)
    _require(t.dtype in _DTYPES, "%s must be float16, bfloat16, float32 or float64, got %s" % (name, t.dtype))
    _require(t.dim() == 2 and t.size(1) > 0, "%s must be two-dimensional with a non-empty row, got %s" % (name, tuple(t.shape)))
    t = t.detach()
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _check_plan(p, device):
    _require(isinstance(p, ExpertPlan), "expected an ExpertPlan, got %s" % type(p).__name__)
    for name, t in (("offsets", p.offsets), ("positions", p.positions)):
        _check_cuda("plan.%s" % name, t, torch.int32)
        _require(t.device == device, "plan.%s is on %s but the rows are on %s" % (name, t.device, device))
        _require(t.is_contiguous(), "plan.%s must be contiguous" % name)
    _require(p.offsets.dim() == 1 and p.offsets.numel() >= 2, "plan.offsets must be [num_experts + 1]")
    _require(p.positions.dim() == 2 and p.positions.size(1) > 0, "plan.positions must be [N, k]")


# ---------------------------------------------------------------------------- gate

def _gate_forward(logits, k, renormalize):
    rows = _rows("logits", logits)
    N, E = rows.shape
    weights = torch.empty((N, k), dtype=_weights_dtype(rows.dtype), device=rows.device)
    experts = torch.empty((N, k), dtype=torch.int32, device=rows.device)
    _call(rows.device, "tbe_expert_gate", rows.data_ptr(), rows.stride(0), weights.data_ptr(), experts.data_ptr(), N, E, k,
          _DTYPES[rows.dtype], renormalize)
    return weights, experts


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        weights, experts = _gate_forward(logits, k, renormalize)
        ctx.k, ctx.renormalize, ctx.shape, ctx.dtype = k, renormalize, logits.shape, logits.dtype
        # the renormalized weights are all their gradient needs; the softmax over the whole row is redone
        ctx.save_for_backward(weights, experts, None if renormalize else logits)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights, _):
        weights, experts, logits = ctx.saved_tensors
        grad_weights = grad_weights.contiguous()
        N, E = ctx.shape
        grad = torch.empty((N, E), dtype=ctx.dtype, device=weights.device)
        rows = grad if logits is None else _rows("logits", logits)
        _call(weights.device, "tbe_expert_gate_backward", grad_weights.data_ptr(), rows.data_ptr(), rows.stride(0),
              weights.data_ptr(), experts.data_ptr(), grad.data_ptr(), N, E, ctx.k, _DTYPES[ctx.dtype], ctx.renormalize)
        return grad, None, None


def gate(logits, k, renormalize=True):
    """The ``k`` largest of every row of ``logits`` ``[N, E]`` and their softmax weights: ``(weights [N, k],
    experts int32 [N, k])``, largest first, ties to the lowest index.

    ``renormalize=True``: softmax over the chosen; ``False``: softmax over the row, at the chosen.  A logit
    of ``-inf`` is never chosen: its slot gets id ``-1`` and weight 0, a row of nothing else is all that,
    with a gradient of 0.  ``E`` is at most 1024, ``k`` at most ``min(E, 32)``."""
    _check_cuda("logits", logits)
    k, renormalize = int(k), bool(renormalize)
    _require(logits.dim() == 2 and 1 <= logits.size(1) <= MAX_EXPERTS, "logits must be [N, E] with E in 1..%d" % MAX_EXPERTS)
    _require(1 <= k <= min(logits.size(1), MAX_CHOICES), "k must be in 1..min(E, %d), got %d" % (MAX_CHOICES, k))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Gate.apply(logits, k, renormalize)
    return _gate_forward(logits, k, renormalize)


# ---------------------------------------------------------------------------- plan

def plan(experts, num_experts):
    """Sorts the choices ``experts`` (int32 ``[N, k]``) by expert, stably: an :class:`ExpertPlan`.  Choices
    outside ``0 .. num_experts-1`` go behind all experts.  ``num_experts`` is at most 1024."""
    _check_cuda("experts", experts, torch.int32)
    num_experts = int(num_experts)
    _require(experts.dim() == 2 and experts.size(1) > 0, "experts must be [N, k]")
    _require(1 <= num_experts <= MAX_EXPERTS, "num_experts must be in 1..%d, got %d" % (MAX_EXPERTS, num_experts))
    experts = experts.contiguous()
    device, M = experts.device, experts.numel()
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    positions = torch.empty_like(experts)
    order = torch.empty(M, dtype=torch.int32, device=device)
    nbytes = _lib.lib().tbe_expert_plan_workspace_bytes(M, num_experts)
    _require(nbytes >= 0, _lib.last_error() if nbytes < 0 else "")
    # a buffer of this call: calls on other streams and captured graphs have their own
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call(device, "tbe_expert_plan", experts.data_ptr(), offsets.data_ptr(), positions.data_ptr(), order.data_ptr(), M,
          num_experts, workspace.data_ptr() if nbytes else None, nbytes)
    return ExpertPlan(offsets, positions, order)


# ---------------------------------------------------------------------------- dispatch and combine

def _dispatch_rows(x, offsets, positions):
    N, k = positions.shape
    y = torch.empty((N * k, x.size(1)), dtype=x.dtype, device=x.device)
    _call(x.device, "tbe_expert_dispatch", x.data_ptr(), x.stride(0), positions.data_ptr(), offsets.data_ptr(), y.data_ptr(),
          N, k, x.size(1), offsets.numel() - 1, _DTYPES[x.dtype])
    return y


def _combine_rows(y, offsets, positions, weights):
    N, k = positions.shape
    out = torch.empty((N, y.size(1)), dtype=y.dtype, device=y.device)
    _call(y.device, "tbe_expert_combine", y.data_ptr(), positions.data_ptr(), offsets.data_ptr(),
          None if weights is None else weights.data_ptr(), out.data_ptr(), N, k, y.size(1), offsets.numel() - 1,
          _DTYPES[y.dtype])
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, positions):
        ctx.save_for_backward(offsets, positions)
        return _dispatch_rows(_rows("x", x), offsets, positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        offsets, positions = ctx.saved_tensors
        return _combine_rows(grad.contiguous(), offsets, positions, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, offsets, positions):
        rows = _rows("y", y).contiguous()
        w = None if weights is None else weights.detach().contiguous()
        # the expert rows are only needed for the weights' gradient
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, w, offsets, positions)
        return _combine_rows(rows, offsets, positions, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        y, weights, offsets, positions = ctx.saved_tensors
        need_y, need_w = ctx.needs_input_grad[:2]
        grad = _rows("grad", grad)
        if weights is None:
            return (_dispatch_rows(grad, offsets, positions) if need_y else None), None, None, None
        N, k = positions.shape
        D = grad.size(1)
        grad_y = torch.empty((N * k, D), dtype=grad.dtype, device=grad.device) if need_y else None
        grad_w = torch.empty((N, k), dtype=weights.dtype, device=grad.device) if need_w else None
        _call(grad.device, "tbe_expert_combine_backward", grad.data_ptr(), grad.stride(0), y.data_ptr() if need_w else None,
              positions.data_ptr(), offsets.data_ptr(), weights.data_ptr(), grad_y.data_ptr() if need_y else None,
              grad_w.data_ptr() if need_w else None, N, k, D, offsets.numel() - 1, _DTYPES[grad.dtype])
        return grad_y, grad_w, None, None


def dispatch(x, plan):
    """The rows of ``x`` ``[N, D]`` in expert order: ``[N*k, D]``, row ``plan.positions[t, s]`` is ``x[t]``,
    rows behind ``plan.offsets[-1]`` are zero.  The gradient sums every sample's rows in slot order."""
    rows = _rows("x", x)
    _check_plan(plan, rows.device)
    _require(rows.size(0) == plan.positions.size(0), "x has %d rows but the plan was made for %d"
             % (rows.size(0), plan.positions.size(0)))
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, plan.offsets, plan.positions)
    return _dispatch_rows(rows, plan.offsets, plan.positions)


def combine(y, plan, weights=None):
    """The way back: ``out[t] = sum_s weights[t, s] * y[plan.positions[t, s]]`` over the choices that belong to
    an expert, ``[N, D]`` from ``[N*k, D]``; ``weights`` ``[N, k]`` or None for a plain sum.  Sums are kept in
    float32 (float64 for float64) in slot order and rounded once.  Rows of ``y`` behind
    ``plan.offsets[-1]`` are never read; their gradient is zero."""
    rows = _rows("y", y)
    _check_plan(plan, rows.device)
    N, k = plan.positions.shape
    _require(rows.size(0) == N * k, "y has %d rows but the plan was made for %d" % (rows.size(0), N * k))
    if weights is not None:
        _check_cuda("weights", weights, _weights_dtype(rows.dtype))
        _require(tuple(weights.shape) == (N, k), "weights must be [%d, %d], got %s" % (N, k, tuple(weights.shape)))
        _require(weights.device == rows.device, "weights are on %s but y is on %s" % (weights.device, rows.device))
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(y, weights, plan.offsets, plan.positions)
    return _combine_rows(rows.contiguous(), plan.offsets, plan.positions,
                         None if weights is None else weights.detach().contiguous())
