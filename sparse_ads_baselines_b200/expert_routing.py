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
enqueued on the current CUDA stream of the tensors' device.  There is no CPU path.  Forward-mode tangents are
refused, and so is recording by torch.jit.trace or make_fx; torch.compile leaves the graph around a call.

A choice of ``-1`` (or any id outside ``0 .. num_experts-1``, for instance an expert of another rank) is
nobody's: its row lies behind ``p.offsets[-1]``, ``dispatch`` fills it with zeros and ``combine`` leaves it
out.  ``gate`` gives ``-1`` for experts whose logit is ``-inf``.
"""
from typing import NamedTuple

import torch

from . import _lib

MAX_EXPERTS = 1024
MAX_CHOICES = 32


class ExpertPlan(NamedTuple):
    """Where every choice goes: ``offsets`` int32 ``[E+1]`` (rows of every expert), ``positions`` int32
    ``[N, k]`` (row of every choice) and ``order`` int32 ``[N*k]`` (the choice ``t*k + s`` in every row).
    :func:`plan` makes one; a plan of your own needs ``positions`` to be a permutation of ``0 .. N*k-1``."""
    offsets: torch.Tensor
    positions: torch.Tensor
    order: torch.Tensor


def _require_plan(plan):
    if not isinstance(plan, ExpertPlan):
        raise RuntimeError("expected an ExpertPlan, got %s" % type(plan).__name__)


def gate(logits, k, renormalize=True):
    """The ``k`` largest of every row of ``logits`` ``[N, E]`` and their softmax weights: ``(weights [N, k],
    experts int32 [N, k])``, largest first, ties to the lowest index.

    ``renormalize=True``: softmax over the chosen; ``False``: softmax over the row, at the chosen.  A logit
    of ``-inf`` is never chosen: its slot gets id ``-1`` and weight 0, a row of nothing else is all that,
    with a gradient of 0.  ``E`` is at most 1024, ``k`` at most ``min(E, 32)``."""
    return _lib.glue().gate(logits, k, bool(renormalize))


def plan(experts, num_experts):
    """Sorts the choices ``experts`` (int32 ``[N, k]``) by expert, stably: an :class:`ExpertPlan`.  Choices
    outside ``0 .. num_experts-1`` go behind all experts.  ``num_experts`` is at most 1024."""
    return ExpertPlan(*_lib.glue().plan(experts, num_experts))


def dispatch(x, plan):
    """The rows of ``x`` ``[N, D]`` in expert order: ``[N*k, D]``, row ``plan.positions[t, s]`` is ``x[t]``,
    rows behind ``plan.offsets[-1]`` are zero.  The gradient sums every sample's rows in slot order."""
    _require_plan(plan)
    return _lib.glue().dispatch(x, plan.offsets, plan.positions)


def combine(y, plan, weights=None):
    """The way back: ``out[t] = sum_s weights[t, s] * y[plan.positions[t, s]]`` over the choices that belong to
    an expert, ``[N, D]`` from ``[N*k, D]``; ``weights`` ``[N, k]`` or None for a plain sum.  Sums are kept in
    float32 (float64 for float64) in slot order and rounded once.  Rows of ``y`` behind
    ``plan.offsets[-1]`` are never read; their gradient is zero."""
    _require_plan(plan)
    return _lib.glue().combine(y, plan.offsets, plan.positions, weights)
