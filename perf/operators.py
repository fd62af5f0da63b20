"""Cases of the expert-routing and gradient-clipping operators, with the operators in plain form.

A case names one operator (``op``) and its sizes:

  gate      a router's logits ``[rows, experts]`` -> the k largest of every row with their softmax weights
  dispatch  samples sorted by expert: the plan (sort) and the rows copied into that order, gradient included
  combine   expert outputs brought back to sample order with the gate's weights, gradients included
  clip      the 2-norm over a list of gradients (views of one flat bucket) and the clipped gradients

``prepare`` makes what a training or serving program has in hand, ``run`` is one pass, ``exact`` the same
outputs from the definition in 64 bits.  With ``own`` set, ``run`` calls the package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request at a time: a single row through the router
        dict(name="gate 1x64", op="gate", rows=1, experts=64, k=6, dtype="bf16", renormalize=True, masked=False, train=False),
        # an expert count that is no power of two, some experts switched off per row and padding rows without any
        dict(name="gate 4097x60 masked", op="gate", rows=4097, experts=60, k=4, dtype="fp32", renormalize=False, masked=True,
             train=True),
        # the largest batch of this repository's configurations through many small experts
        dict(name="gate 65536x256", op="gate", rows=65536, experts=256, k=8, dtype="bf16", renormalize=True, masked=False,
             train=True),
        # a handful of requests in flight
        dict(name="dispatch 8x2048", op="dispatch", rows=8, experts=128, k=8, dim=2048, dtype="bf16", dropped=0.0, train=False),
        # odd sizes, with a quarter of the choices belonging to experts of another rank
        dict(name="dispatch 5003x1001", op="dispatch", rows=5003, experts=61, k=6, dim=1001, dtype="fp32", dropped=0.25,
             train=True),
        # the headline batch with its 64 pooled rows of 128 side by side
        dict(name="dispatch 2048x8192", op="dispatch", rows=2048, experts=16, k=2, dim=8192, dtype="fp16", dropped=0.0,
             train=True),
        # the way back of the small call
        dict(name="combine 8x2048", op="combine", rows=8, experts=128, k=8, dim=2048, dtype="bf16", dropped=0.0, train=False),
        # rows that are only 8-byte aligned, some choices not served here
        dict(name="combine 2999x1004", op="combine", rows=2999, experts=37, k=3, dim=1004, dtype="fp16", dropped=0.1, train=True),
        # a long training batch with many choices per sample
        dict(name="combine 16384x2048", op="combine", rows=16384, experts=256, k=8, dim=2048, dtype="bf16", dropped=0.0,
             train=True),
        # the dense part of a small model: launch latency counts
        dict(name="clip 40 small", op="clip", tensors=40, elements=60_000, dtype="fp32", odd=True, clipped=True),
        # a model's gradients in one bucket, above the limit
        dict(name="clip 200M", op="clip", tensors=120, elements=200_000_000, dtype="bf16", odd=False, clipped=True),
        # fp32 gradients below the limit: the usual step late in a training run
        dict(name="clip 300M below", op="clip", tensors=160, elements=300_000_000, dtype="fp32", odd=False, clipped=False),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["gate", "dispatch", "combine", "clip"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "gate":
        experts = _log_int(rng, 2, 512)
        rows = _log_int(rng, 1, min(65536, 16_000_000 // experts))
        return dict(op=op, rows=rows, experts=experts, k=min(experts, rng.randint(1, 8)), dtype=dtype,
                    renormalize=rng.random() < 0.5, masked=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "clip":
        elements = _log_int(rng, 5_000, 200_000_000)
        return dict(op=op, tensors=_log_int(rng, 1, 200), elements=elements, dtype=dtype, odd=rng.random() < 0.5,
                    clipped=rng.random() < 0.7)
    k, dim = rng.randint(1, 8), _log_int(rng, 32, 8192)
    if rng.random() < 0.7:
        dim -= dim % 8
    rows = _log_int(rng, 1, min(65536, 120_000_000 // (k * dim)))
    return dict(op=op, rows=rows, experts=_log_int(rng, max(2, k), 256), k=k, dim=dim, dtype=dtype,
                dropped=rng.choice([0.0, 0.0, 0.1, 0.5]), train=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _choices(g, case):
    """Distinct experts per row, unevenly liked; a share of them switched to ids that are not served here."""
    rows, experts, k = case["rows"], case["experts"], case["k"]
    liked = torch.randn(experts, generator=g, device="cuda")
    scores = liked + torch.randn(rows, experts, generator=g, device="cuda")
    ids = torch.sort(scores, dim=1, descending=True).indices[:, :k].to(torch.int32)
    away = torch.rand(rows, k, generator=g, device="cuda") < case["dropped"]
    return torch.where(away, torch.full_like(ids, -1), ids).contiguous()


def _sizes(case):
    """Lengths of the gradients of one bucket: a few large matrices, many small vectors."""
    r = np.random.RandomState(case["tensors"] * 7 + case["elements"] % 1000)
    share = np.exp(r.uniform(0, 6, case["tensors"]))
    n = np.maximum(1, (case["elements"] * share / share.sum()).astype(np.int64))
    return (n | 1 if case["odd"] else (n + 63) // 64 * 64).tolist()


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "gate":
        s["logits"] = _randn(g, (case["rows"], case["experts"]), dtype)
        if case["masked"]:
            off = torch.rand(case["rows"], case["experts"], generator=g, device="cuda") < 0.2
            off |= torch.rand(case["rows"], 1, generator=g, device="cuda") < 0.05
            s["logits"].masked_fill_(off, -math.inf)
        s["logits"].requires_grad_(case["train"])
        s["grad"] = _randn(g, (case["rows"], case["k"]), torch.float32)
    elif case["op"] == "dispatch":
        s["experts"] = _choices(g, case)
        s["x"] = _randn(g, (case["rows"], case["dim"]), dtype).requires_grad_(case["train"])
        s["grad"] = _randn(g, (case["rows"] * case["k"], case["dim"]), dtype) if case["train"] else None
    elif case["op"] == "combine":
        s["offsets"], s["positions"], s["order"] = _plan(_choices(g, case), case["experts"])
        s["y"] = _randn(g, (case["rows"] * case["k"], case["dim"]), dtype).requires_grad_(case["train"])
        w = torch.rand(case["rows"], case["k"], generator=g, device="cuda") + 0.05
        s["weights"] = (w / w.sum(1, keepdim=True)).requires_grad_(case["train"])
        s["grad"] = _randn(g, (case["rows"], case["dim"]), dtype) if case["train"] else None
    else:
        sizes = _sizes(case)
        total = sum(sizes)
        s["flat"] = _randn(g, (total,), dtype, 1e-2)
        s["grads"] = list(s["flat"].split(sizes))
        s["max_norm"] = 1e-2 * math.sqrt(total) * (0.3 if case["clipped"] else 2.0)
        if case["clipped"]:
            s["flat_out"] = torch.empty_like(s["flat"])
            s["out"] = list(s["flat_out"].split(sizes))
    return s


# ------------------------------------------------------------------------------------------ plain forms

def _gate(logits, k, renormalize, grad):
    x = logits.detach().float()
    ranked = torch.sort(x, dim=1, descending=True, stable=True)
    chosen, index = ranked.values[:, :k], ranked.indices[:, :k]
    none = chosen == -math.inf
    top = x.amax(1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    e, e_all = torch.exp(chosen - top), torch.exp(x - top)
    total = (e if renormalize else e_all).sum(1, keepdim=True)
    dead = total == 0
    total = torch.where(dead, torch.ones_like(total), total)
    weights = e / total
    experts = torch.where(none, torch.full_like(index, -1), index).to(torch.int32)
    if grad is None:
        return {"weights": weights, "experts": experts}
    wg = weights * grad
    mean = wg.sum(1, keepdim=True)
    dx = torch.zeros_like(x).scatter_(1, index, wg)
    if renormalize:
        dx -= torch.zeros_like(x).scatter_(1, index, weights) * mean
    else:
        dx -= e_all / total * mean
    return {"weights": weights, "experts": experts, "grad_logits": dx.to(logits.dtype)}


def _plan(experts, num_experts):
    ids = experts.flatten().long()
    bins = torch.where((ids >= 0) & (ids < num_experts), ids, torch.full_like(ids, num_experts))
    ranked = torch.sort(bins, stable=True)
    positions = torch.empty_like(ids)
    positions[ranked.indices] = torch.arange(ids.numel(), device=ids.device)
    offsets = torch.searchsorted(ranked.values, torch.arange(num_experts + 1, device=ids.device))
    return offsets.to(torch.int32), positions.to(torch.int32).view(experts.shape), ranked.indices.to(torch.int32)


def _dispatch(x, experts, num_experts, grad):
    offsets, positions, order = _plan(experts, num_experts)
    kept, k = offsets[-1], experts.shape[1]
    rows = torch.arange(order.numel(), device=x.device)[:, None]
    zero = torch.zeros((), dtype=x.dtype, device=x.device)
    y = torch.where(rows < kept, x.detach()[order.long() // k], zero)
    out = {"offsets": offsets, "positions": positions, "order": order, "y": y}
    if grad is not None:
        terms = torch.where((positions < kept)[:, :, None], grad[positions.long()].float(), zero.float())
        out["grad_x"] = terms.sum(1).to(x.dtype)
    return out


def _combine(y, offsets, positions, order, weights, grad):
    kept, k = offsets[-1], positions.shape[1]
    here = positions < kept
    zero = torch.zeros((), device=y.device)
    rows = torch.where(here[:, :, None], y.detach()[positions.long()].float(), zero)
    w = weights.detach()
    out = {"out": (rows * w[:, :, None]).sum(1).to(y.dtype)}
    if grad is not None:
        g = grad.float()
        out["grad_weights"] = (rows * g[:, None, :]).sum(2)
        del rows
        entry = order.long()
        dy = w.flatten()[entry][:, None] * g[entry // k]
        at = torch.arange(entry.numel(), device=y.device)[:, None]
        out["grad_y"] = torch.where(at < kept, dy, zero).to(y.dtype)
    return out


def _clip(flat, max_norm):
    x = flat.float()
    norm = (x * x).sum(dtype=torch.float64).sqrt()
    scale = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    return {"norm": norm.float(), "grads": (x * scale).to(flat.dtype)}


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "gate":
        return _gate(s["logits"], case["k"], case["renormalize"], s["grad"] if case["train"] else None)
    if case["op"] == "dispatch":
        return _dispatch(s["x"], s["experts"], case["experts"], s["grad"])
    if case["op"] == "combine":
        return _combine(s["y"], s["offsets"], s["positions"], s["order"], s["weights"], s["grad"])
    return _clip(s["flat"], s["max_norm"])


def _run_own(s, case):
    from sparse_ads_baselines_b200 import expert_routing, gradient_clipping
    if case["op"] == "gate":
        weights, experts = expert_routing.gate(s["logits"], case["k"], renormalize=case["renormalize"])
        out = {"weights": weights, "experts": experts}
        if case["train"]:
            out["grad_logits"], = torch.autograd.grad(weights, s["logits"], s["grad"])
        return out
    if case["op"] == "dispatch":
        plan = expert_routing.plan(s["experts"], case["experts"])
        y = expert_routing.dispatch(s["x"], plan)
        out = {"offsets": plan.offsets, "positions": plan.positions, "order": plan.order, "y": y}
        if case["train"]:
            out["grad_x"], = torch.autograd.grad(y, s["x"], s["grad"])
        return out
    if case["op"] == "combine":
        plan = expert_routing.ExpertPlan(s["offsets"], s["positions"], s["order"])
        y = expert_routing.combine(s["y"], plan, s["weights"])
        out = {"out": y}
        if case["train"]:
            out["grad_y"], out["grad_weights"] = torch.autograd.grad(y, (s["y"], s["weights"]), s["grad"])
        return out
    if case["clipped"]:
        return {"norm": gradient_clipping.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"]), "grads": s["flat_out"]}
    return {"norm": gradient_clipping.clip_grad_norm(s["grads"], s["max_norm"]), "grads": s["flat"]}


# ------------------------------------------------------------------------------------------ work and the exact values

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "clip":
        n = sum(_sizes(case))
        return {"bytes": n * size * 2, "flops": 3 * n}
    entries = case["rows"] * case["k"]
    if case["op"] == "gate":
        table = case["rows"] * case["experts"]
        train = entries * 4 + table * size if case["train"] else 0
        return {"bytes": table * size + entries * 8 + train, "flops": table * (6 if case["train"] else 3)}
    one, many = case["rows"] * case["dim"] * size, entries * case["dim"] * size
    if case["op"] == "dispatch":
        sort = entries * 12 + (case["experts"] + 1) * 4
        return {"bytes": sort + (one + many) * (2 if case["train"] else 1), "flops": entries * case["dim"] if case["train"] else 0}
    back = one + many + entries * 4 if case["train"] else 0
    return {"bytes": many + one + entries * 8 + back, "flops": entries * case["dim"] * (5 if case["train"] else 2)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gate":
        return _exact_gate(s, case)
    if case["op"] == "clip":
        n2 = sum(float(torch.dot(p, p)) for p in (q.double() for q in s["flat"].split(1 << 26)))
        factor = min(1.0, s["max_norm"] / (math.sqrt(n2) + 1e-6))
        return {"norm": math.sqrt(n2), "grads": s["flat"].double().mul_(factor)}
    k = case["k"]
    if case["op"] == "dispatch":
        ids = s["experts"].flatten()
        groups = [(ids == e).nonzero().flatten() for e in range(case["experts"])]
        kept = sum(len(v) for v in groups)
        order = torch.cat(groups + [(ids < 0).nonzero().flatten()])
        positions = torch.argsort(order)
        counts = [0] + [len(v) for v in groups]
        y = torch.zeros(ids.numel(), case["dim"], dtype=torch.float64, device="cuda")
        y[:kept] = s["x"].detach().double()[torch.div(order[:kept], k, rounding_mode="floor")]
        out = {"offsets": torch.tensor(np.cumsum(counts), dtype=torch.int32), "y": y, "order": order.to(torch.int32),
               "positions": positions.to(torch.int32).view(-1, k)}
        if case["train"]:
            dx = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
            dx.index_add_(0, order[:kept] // k, s["grad"][:kept].double())
            out["grad_x"] = dx
        return out
    kept, w = int(s["offsets"][-1]), s["weights"].detach().double()
    out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
    y, dw, dy = s["y"].detach(), torch.zeros_like(w), torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    for j in range(k):
        p = s["positions"][:, j].long()
        t = (p < kept).nonzero().flatten()
        rows = y[p[t]].double()
        out[t] += w[t, j, None] * rows
        if case["train"]:
            dw[t, j] = torch.linalg.vecdot(rows, s["grad"][t].double())
            dy[p[t]] = w[t, j, None] * s["grad"][t].double()
    return {"out": out, "grad_y": dy, "grad_weights": dw} if case["train"] else {"out": out}


def _exact_gate(s, case):
    x = s["logits"].detach().double().cpu().numpy()
    index = np.argsort(-x, axis=1, kind="stable")[:, :case["k"]]
    chosen = np.take_along_axis(x, index, 1)
    live = np.isfinite(chosen)
    high = np.where(live[:, :1], chosen[:, :1], 0.0)
    p = np.exp(x - high)
    picked = np.take_along_axis(p, index, 1)
    mass = picked.sum(1, keepdims=True) if case["renormalize"] else p.sum(1, keepdims=True)
    mass[mass == 0] = 1.0
    weights = picked / mass
    out = {"weights": weights, "experts": np.where(live, index, -1).astype(np.int32)}
    if case["train"]:
        g = s["grad"].double().cpu().numpy()
        full, spread = np.zeros_like(x), np.zeros_like(x)
        np.put_along_axis(full, index, g, 1)
        np.put_along_axis(spread, index, weights, 1)
        if not case["renormalize"]:
            spread = p / mass
        out["grad_logits"] = spread * (full - (weights * g).sum(1, keepdims=True))
    return out
