"""Expert routing and gradient clipping under PyTorch's other modes, as far as no device is needed: what cannot be
computed there is refused before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

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
