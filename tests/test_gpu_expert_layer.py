"""The routing operators together, as a model uses them, against float64 autograd on the CPU: pooled table
rows -> router -> gate -> plan -> dispatch -> the experts' layers -> combine -> loss -> backward -> clipping ->
step of everything, tables included."""
import numpy as np
import pytest
import torch

from oracle import tbe_oracle as oracle
from sparse_ads_baselines_b200 import expert_routing as er
from sparse_ads_baselines_b200 import gradient_clipping as gc
from sparse_ads_baselines_b200 import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

T, ROWS, D, B, L, E, K, H, LR = 3, 50, 8, 37, 4, 6, 2, 5, 0.1


def _make(seed):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64) * 0.5

    dense = dict(router=rand(T * D, E), up=rand(E, T * D, H), down=rand(E, H, T * D), head=rand(T * D, 1))
    indices = torch.randint(0, ROWS, (T, B, L), generator=g)
    return rand(T * ROWS, D), dense, indices, rand(B, 1)


def _experts(y, offsets, dense):
    """The experts' two layers on their blocks of rows."""
    blocks = [torch.tanh(y[a:b] @ dense["up"][e]) @ dense["down"][e]
              for e, (a, b) in enumerate(zip(offsets[:-1], offsets[1:]))]
    return torch.cat(blocks + [torch.zeros_like(y[offsets[-1]:])])


def _reference(tables, dense, indices, target, renormalize, away, max_norm, max_pooled):
    """One step in plain float64 torch on the CPU: a loop over the choices."""
    tables, dense = tables.clone(), {n: t.clone().requires_grad_() for n, t in dense.items()}
    pooled = torch.stack([tables[t * ROWS:(t + 1) * ROWS][indices[t]].sum(1) for t in range(T)], 1).requires_grad_()
    x = pooled.reshape(B, T * D)
    logits = x @ dense["router"]
    if away is not None:
        logits = logits.masked_fill(torch.arange(E) == away, -float("inf"))
    p = torch.softmax(logits, 1)
    order = np.lexsort((np.broadcast_to(np.arange(E), (B, E)), -logits.detach().numpy()), axis=1)[:, :K]
    chosen = torch.from_numpy(order.copy())
    w = p.gather(1, chosen)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    rows = []
    for b in range(B):
        rows.append(sum(w[b, s] * (torch.tanh(x[b] @ dense["up"][e]) @ dense["down"][e]) for s, e in enumerate(order[b])))
    out = x + torch.stack(rows)
    loss = (out @ dense["head"] - target).square().sum()
    loss.backward()
    norm = torch.sqrt(sum(t.grad.square().sum() for t in dense.values()))
    factor = min(1.0, max_norm / (float(norm) + 1e-6))
    step = {n: t.detach() - LR * factor * t.grad for n, t in dense.items()}
    g = pooled.grad
    g = g * min(1.0, max_pooled / (float(g.norm()) + 1e-6))
    for t in range(T):
        for b in range(B):
            for r in indices[t, b]:
                tables[t * ROWS + r] -= LR * g[b, t]
    return loss.detach(), norm, step, tables


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("away", [None, 3], ids=["all", "one expert off"])
def test_training_step(cuda_device, renormalize, away):
    """In float64 throughout, so that both sides choose the same experts: 1e-9 is far above the few thousand
    roundings of 2^-53 of a step and far below anything else."""
    tables, dense, indices, target = _make(7)
    max_norm, max_pooled = 2.0, 1.5  # both below what the step has: both are clipped
    ref_loss, ref_norm, ref_dense, ref_tables = _reference(tables, dense, indices, target, renormalize, away, max_norm,
                                                           max_pooled)
    assert ref_norm > max_norm

    m = ops.TableBatchedEmbeddingBags(T, ROWS, D, learning_rate=LR, max_grad_norm=max_pooled).cuda().double()
    m.embedding_weights.data.copy_(tables)
    p = {n: t.to(cuda_device).requires_grad_() for n, t in dense.items()}
    idx, off = oracle.get_table_batched_offsets_from_dense(indices.numpy())
    pooled = m(torch.from_numpy(idx).to(cuda_device), torch.from_numpy(off).to(cuda_device))
    x = pooled.reshape(B, T * D)
    logits = x @ p["router"]
    if away is not None:
        logits = logits.masked_fill(torch.arange(E, device=cuda_device) == away, -float("inf"))
    weights, experts = er.gate(logits, K, renormalize=renormalize)
    plan = er.plan(experts, E)
    y = _experts(er.dispatch(x, plan), plan.offsets.tolist(), p)
    out = x + er.combine(y, plan, weights)
    loss = (out @ p["head"] - target.to(cuda_device)).square().sum()
    loss.backward()
    grads = [t.grad for t in p.values()]
    norm = gc.clip_grad_norm(grads, max_norm)
    close = dict(rtol=1e-9, atol=1e-9)
    torch.testing.assert_close(loss.detach().cpu(), ref_loss, **close)
    torch.testing.assert_close(norm.cpu().double(), ref_norm, rtol=2.0 ** -23, atol=0)
    for n, t in p.items():
        torch.testing.assert_close((t.detach() - LR * t.grad).cpu(), ref_dense[n], **close)
    torch.testing.assert_close(m.embedding_weights.detach().cpu(), ref_tables, **close)
    if away is not None:
        assert (experts != away).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_a_few_steps_run(cuda_device, dtype):
    """In the training types: the step runs, everything stays finite, a clipped list has its norm."""
    tables, dense, indices, target = _make(3)
    p = {n: t.to(cuda_device, dtype).requires_grad_() for n, t in dense.items()}
    x = torch.randn(B, T * D, device=cuda_device).to(dtype)
    for _ in range(3):
        weights, experts = er.gate((x @ p["router"]).float(), K)
        plan = er.plan(experts, E)
        y = _experts(er.dispatch(x, plan), plan.offsets.tolist(), p)
        out = x + er.combine(y, plan, weights)
        loss = (out @ p["head"] - target.to(cuda_device, dtype)).float().square().mean()
        loss.backward()
        grads = [t.grad for t in p.values()]
        gc.clip_grad_norm(grads, 0.01)
        assert all(torch.isfinite(g).all() for g in grads)
        assert float(gc.grad_norm(grads)) <= 0.01 * (1 + 2 ** -8)
        with torch.no_grad():
            for t in p.values():
                t -= 0.1 * t.grad
                t.grad = None


def test_one_expert_per_rank(cuda_device):
    """Experts spread over ranks: every rank plans only its own ids, and the ranks' results add up."""
    torch.manual_seed(0)
    N, k, dim, ranks = 200, 3, 40, 2
    logits = torch.randn(N, E, device=cuda_device)
    x = torch.randn(N, dim, device=cuda_device, dtype=torch.float64)
    weights, experts = er.gate(logits.double(), k)
    scale = torch.arange(1, E + 1, device=cuda_device, dtype=torch.float64)

    def run(ids, count, first):
        plan = er.plan(ids, count)
        y = er.dispatch(x, plan)
        for e, (a, b) in enumerate(zip(plan.offsets.tolist()[:-1], plan.offsets.tolist()[1:])):
            y[a:b] *= scale[first + e]
        return er.combine(y, plan, weights)

    whole = run(experts, E, 0)
    per = E // ranks
    parts = sum(run(experts - r * per, per, r * per) for r in range(ranks))
    torch.testing.assert_close(parts, whole, rtol=1e-12, atol=1e-12)
