"""Gradients of the routing operators where digits cancel, and with gradients and inputs of unusual kinds.

Tolerances count roundings (u = 2^-24), as in the tests of the operators themselves.
"""
import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

import routing_testlib as ref
from routing_testlib import assert_within, f64, unit
from sparse_ads_baselines_b200 import _lib
from sparse_ads_baselines_b200 import expert_routing as er
from sparse_ads_baselines_b200 import gradient_clipping as gc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E", [2, 40, 256, 1000])
@pytest.mark.parametrize("k", [1, 2])
def test_whole_softmax_gradient_of_a_settled_router(cuda_device, E, k):
    """One weight nearly 1 (all other logits 0): the gradient keeps its relative accuracy in every column.

    A p_j carries 2 units (4 u) of exp (the differences are exact), 37 roundings of the sum and 4 u of its terms,
    one division: 46 u; a sum of them 37 more: 83 u.  p_s (sum over the chosen of w_j (g_s - g_j) + r g_s): the two
    terms have one sign, each carries at most 83 u and 2 operations; their sum 1, p_s and the product 47: 133 u.
    p_j c: c = w_1 g_1 + w_2 g_2 with |w_2 g_2| < w_1 |g_1| / 1000: 50 u, p_j and the product 47: 97 u."""
    rng = np.random.default_rng(E + k)
    x = torch.zeros(300, E, device=cuda_device)
    x[:, 1] = torch.from_numpy(rng.uniform(8, 20, 300)).float().to(cuda_device)
    x[0, 1], x[1, 1] = 20.0, 18.0
    x.requires_grad_()
    w, e = er.gate(x, k, renormalize=False)
    g = torch.from_numpy(np.stack([rng.uniform(1, 2, 300), rng.uniform(-2, -1, 300)], 1)[:, :k]).float().to(cuda_device)
    dx, = torch.autograd.grad(w, x, g)
    exact = f64(x).astype(np.longdouble)  # the formula loses digits too: 2^-53 / 2e-9 of the smallest value in float64
    weights, experts = ref.gate(exact, k, False)
    want = ref.gate_gradient(exact, weights, experts, f64(g), False)[0].astype(np.float64)
    assert np.array_equal(e.cpu().numpy(), experts)
    assert_within(dx, want, 133 * unit(torch.float32) * np.abs(want))


def _graph(op, device):
    """(output, inputs) of one operator with its graph."""
    torch.manual_seed(3)
    x = torch.randn(6, 8, device=device)
    if op.startswith("gate"):
        x.requires_grad_()
        return er.gate(x, 3, renormalize=op == "gate")[0], (x,)
    p = er.plan(er.gate(x, 3)[1], 7)
    if op == "dispatch":
        x.requires_grad_()
        return er.dispatch(x, p), (x,)
    y = torch.randn(18, 8, device=device, requires_grad=True)
    if op == "sum":
        return er.combine(y, p), (y,)
    w = torch.rand(6, 3, device=device, requires_grad=True)
    return er.combine(y, p, w), (y, w)


OPS = ["gate", "gate_whole", "dispatch", "sum", "combine"]


@pytest.mark.parametrize("op", OPS)
def test_lazily_negated_gradients(cuda_device, op):
    """An incoming gradient with the negative bit counts with its sign (the bits are the negated ones')."""
    out, inputs = _graph(op, cuda_device)
    g = torch.randn_like(out)
    want = torch.autograd.grad(out, inputs, -g, retain_graph=True)
    got = torch.autograd.grad(out, inputs, torch._neg_view(g))
    assert all(torch.equal(a, b) and a.any() for a, b in zip(got, want))


@pytest.mark.parametrize("op", OPS)
def test_forward_mode_over_a_backward_is_refused(cuda_device, op):
    """A gradient with a tangent would come back without one, which says that its derivative is zero."""
    out, inputs = _graph(op, cuda_device)
    with fwd.dual_level():
        g = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, inputs, g, retain_graph=True)
    assert all(t.isfinite().all() for t in torch.autograd.grad(out, inputs, torch.ones_like(out)))


def test_forward_mode_weights_and_out_are_refused(cuda_device):
    x, y, w = torch.randn(4, 6, device=cuda_device), torch.randn(8, 6, device=cuda_device), torch.rand(4, 2, device=cuda_device)
    p = er.plan(torch.arange(8, dtype=torch.int32, device=cuda_device).view(4, 2) % 3, 3)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            er.combine(y, p, fwd.make_dual(w, torch.ones_like(w)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gc.clip_grad_norm([x], 1.0, out=[fwd.make_dual(torch.zeros_like(x), torch.ones_like(x))])
    er.combine(y, p, w)


def test_recording_is_refused(cuda_device):
    x = torch.randn(4, 6, device=cuda_device)
    for f in (lambda t: er.gate(t, 2)[0], lambda t: er.gate(t.requires_grad_(), 2)[0], lambda t: gc.clip_grad_norm([t], 1.0)):
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(f, x.clone(), check_trace=False)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(f)(x.clone())
    out, inputs = _graph("gate", cuda_device)
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(lambda g: torch.autograd.grad(out, inputs, g, retain_graph=True)[0])(torch.ones_like(out))
    # a compiled function leaves the recorder around the call
    compiled = torch.compile(lambda t: er.gate(t * 2, 2)[0] * 3, backend="eager")
    assert torch.equal(compiled(x), er.gate(x * 2, 2)[0] * 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
def test_renormalized_gradient_without_logits(cuda_device, dtype):
    """The C entry takes no logits, or any, where it does not read them."""
    torch.manual_seed(5)
    x = torch.randn(33, 48, device=cuda_device, dtype=dtype, requires_grad=True)
    w, e = er.gate(x, 4)
    g = torch.randn_like(w)
    want, = torch.autograd.grad(w, x, g)
    kind = {torch.bfloat16: _lib.TBE_BF16, torch.float32: _lib.TBE_F32, torch.float64: _lib.TBE_F64}[dtype]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for logits, stride in ((None, 0), (None, -1), (x.data_ptr() + 1, 7)):
        out = torch.full_like(x, float("nan"))
        _lib.call("tbe_expert_gate_backward", g.data_ptr(), logits, stride, w.data_ptr(), e.data_ptr(), out.data_ptr(),
                  33, 48, 4, kind, 1, stream)
        assert torch.equal(out, want)


class _Weights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return er.gate(x, 2)[0]


@torch.library.custom_op("routing_tests::gate_weights", mutates_args=())
def _gate_weights(x: torch.Tensor) -> torch.Tensor:
    return er.gate(x, 2)[0]


@_gate_weights.register_fake
def _(x):
    return x.new_empty(x.shape[0], 2, dtype=torch.float32)


def test_operators_that_a_recorder_keeps_as_a_whole(cuda_device):
    """A call inside a Python autograd.Function or a custom operator is part of what is recorded, and runs again."""
    x, other = torch.randn(2, 5, 6, device=cuda_device)
    want = er.gate(other, 2)[0] * 2
    for f in (torch.jit.trace(lambda t: _Weights.apply(t) * 2, x, check_trace=False),
              torch.jit.trace(lambda t: _gate_weights(t) * 2, x, check_trace=False),
              make_fx(lambda t: _gate_weights(t) * 2)(x),
              torch.compile(lambda t: _gate_weights(t) * 2, backend="eager", fullgraph=True)):
        assert torch.equal(f(other), want)
