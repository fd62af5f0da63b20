"""Expert routing and gradient clipping under PyTorch's other modes, as far as no device is needed: what cannot be
computed there is refused before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from sparse_ads_baselines_b200 import expert_routing as er
from sparse_ads_baselines_b200 import gradient_clipping as gc


def _plan(device="cpu"):
    ints = dict(dtype=torch.int32, device=device)
    return er.ExpertPlan(torch.tensor([0, 4, 8], **ints), torch.arange(8, **ints).view(4, 2), torch.arange(8, **ints))


def _calls(dual):
    """Every call that would answer without a derivative, with a tangent on one of its arguments."""
    x, y, w = torch.randn(4, 6), torch.randn(8, 6), torch.rand(4, 2)
    p = _plan()
    return [lambda: er.gate(dual(x), 2), lambda: er.gate(dual(x), 2, renormalize=False), lambda: er.dispatch(dual(x), p),
            lambda: er.combine(dual(y), p), lambda: er.combine(dual(y), p, w), lambda: gc.grad_norm([dual(x)]),
            lambda: gc.grad_norm(dual(x)), lambda: gc.clip_grad_norm([dual(x)], 1.0),
            lambda: gc.clip_grad_norm([None, dual(x)], 1.0, out=[None, torch.empty_like(x)])]


@pytest.mark.parametrize("call", range(9))
def test_forward_mode_is_refused(call):
    """A dual tensor need not have requires_grad, so no autograd node would say so."""
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            _calls(lambda t: fwd.make_dual(t, torch.ones_like(t)))[call]()
    with pytest.raises(RuntimeError, match="CUDA tensor"):  # the same call without a tangent
        _calls(lambda t: t)[call]()


RECORDED = {
    "gate": lambda x: er.gate(x, 2)[0],
    "plan": lambda x: er.plan(x.int(), 3).order,
    "dispatch": lambda x: er.dispatch(x, _plan(x.device)),
    "combine": lambda x: er.combine(x.repeat(2, 1), _plan(x.device)),
    "grad_norm": lambda x: gc.grad_norm([x]),
    "clip_grad_norm": lambda x: gc.clip_grad_norm([x], 1.0),
    "clip_grad_norm out": lambda x: gc.clip_grad_norm([x], 1.0, out=[torch.empty_like(x)]),
}
RECORDERS = {"trace": lambda f, x: torch.jit.trace(f, x, check_trace=False), "make_fx": lambda f, x: make_fx(f)(x)}


@pytest.mark.parametrize("recorder", RECORDERS)
@pytest.mark.parametrize("op", RECORDED)
def test_recording_is_refused(op, recorder):
    """A recorder would keep the allocation of the result and nothing of what fills it."""
    with pytest.raises(RuntimeError, match="recorded"):
        RECORDERS[recorder](RECORDED[op], torch.zeros(4, 6))
    with pytest.raises(RuntimeError, match="CUDA tensor"):  # and not refused once the recorder is gone
        RECORDED[op](torch.zeros(4, 6))


class _Wrapped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return er.gate(x, 2)[0]


def test_a_recorded_function_is_not_refused():
    """torch.jit.trace keeps a Python autograd.Function as a whole and calls it again, so its result is computed."""
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch.jit.trace(_Wrapped.apply, torch.zeros(4, 6), check_trace=False)


class _WithTangent(torch.autograd.Function):
    @staticmethod
    def forward(x):
        return er.gate(x, 2)[0]

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def jvp(ctx, t):
        return t[:, :2]


def test_a_function_with_its_own_forward_mode_is_not_refused():
    """Inside its forward the tangents are its own business."""
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(4, 6), torch.ones(4, 6))
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            _WithTangent.apply(x)
