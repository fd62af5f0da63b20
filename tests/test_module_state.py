"""Modules that were saved by an earlier version of the package."""
import torch
from torch import nn

from sparse_ads_baselines_b200 import table_batched_embeddings_ops as ops


def test_a_module_from_before_the_gradient_limit(monkeypatch):
    """Unpickling restores the attributes that were saved; one without max_grad_norm has no limit."""
    m = ops.TableBatchedEmbeddingBags.__new__(ops.TableBatchedEmbeddingBags)
    nn.Module.__init__(m)
    m.embedding_weights = nn.Parameter(torch.zeros(4, 8))
    for name in ("table_offsets", "optimizer_state"):
        m.register_buffer(name, torch.zeros(4))
    m.__setstate__(dict(m.__dict__, optimizer=ops.Optimizer.SGD, learning_rate=0.1, eps=None, stochastic_rounding=False,
                        pooling_mode="sum", plan_ahead=False))
    seen = []
    monkeypatch.setattr(ops.LookupFunction, "apply", lambda *args: seen.append(args))
    m(torch.zeros(1), torch.zeros(2))
    assert seen[0][9:] == (False, "sum", False, None)
