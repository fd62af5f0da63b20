"""Gradient norm and clipping against float64.

Tolerances: sixteen-bit values are summed eight at a time in float32, seven additions and eight squares of
positive terms: 2^-21 relative in the squared norm, 2^-22 in the norm; everything else is float64, and the
norm is rounded once to float32 (2^-24).  A scaled element carries the factor's error (2^-22, and 2^-24 for
its rounding to float32), one product (2^-24) and the rounding to its type.  In float64 a thread adds up
to 64 squares of a chunk and the tree above it has 13 levels, here and in the reference: 256 units.
"""
import math

import numpy as np
import pytest
import torch

from routing_testlib import HALF_STEP, TINY, assert_within, f64, name
from sparse_ads_baselines_b200 import gradient_clipping as gc
from sparse_ads_baselines_b200 import table_batched_embeddings_ops as ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]
NORM_TOL = 2.0 ** -22 + 2.0 ** -23
SCALE_TOL = 2.0 ** -22 + 3 * 2.0 ** -24


def _norm(tensors):
    return math.sqrt(sum(float(np.square(f64(t)).sum()) for t in tensors))


def _make(sizes, dtype, device, seed=0, scale=1.0):
    rng = np.random.default_rng(seed)
    return [torch.from_numpy(rng.standard_normal(n) * scale).to(dtype).to(device) for n in sizes]


def _check(before, after, norm, max_norm, eps=1e-6):
    n = _norm(before)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    # the returned float32 is inf where the norm passes its range (2^128, less a rounding); the factor is not
    assert math.isinf(float(norm)) if n >= 2.0 ** 128 else abs(float(norm) - n) <= NORM_TOL * n + 2.0 ** -150
    c = min(1.0, max_norm / (n + eps))
    for b, a in zip(before, after):
        d = name(a.dtype)
        want = f64(b) * c
        tol = 2.0 ** -22 if d == "float64" else SCALE_TOL
        if all(t.dtype in (torch.float32, torch.float64) for t in before):
            tol = 256 * 2.0 ** -53 if d == "float64" else 3 * 2.0 ** -24
        assert_within(a, want, (tol + HALF_STEP[d] * (1 + tol)) * np.abs(want) + TINY[d] * 1.01, "scaled")


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [7, 8, 9, 1023], [16383, 16384, 16385], [100_003, 3, 65_536, 1]],
                         ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("factor", [0.25, 1.5, 0.0])
def test_clip(cuda_device, dtype, sizes, factor):
    before = _make(sizes, dtype, cuda_device)
    max_norm = factor * _norm(before)
    g = [t.clone() for t in before]
    norm = gc.clip_grad_norm(g, max_norm)
    _check(before, g, norm, max_norm)
    if factor > 1:
        assert all(torch.equal(a, b) for a, b in zip(g, before))
    out = [torch.full_like(t, float("nan")) for t in before]
    source = [t.clone() for t in before]
    norm2 = gc.clip_grad_norm(source, max_norm, out=out)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(out, g))
    assert all(torch.equal(a, b) for a, b in zip(source, before))
    assert torch.equal(gc.grad_norm(before), norm)


@pytest.mark.parametrize("count", [64, 65, 1024, 1025, 2500])
def test_many_tensors_of_mixed_types(cuda_device, count):
    rng = np.random.default_rng(count)
    before = [torch.from_numpy(rng.standard_normal(int(rng.integers(0, 400)))).to(DTYPES[i % 4]).to(cuda_device)
              for i in range(count)]
    before[count // 2] = torch.from_numpy(rng.standard_normal(70_000)).to(torch.bfloat16).to(cuda_device)
    g = [t.clone() for t in before]
    norm = gc.clip_grad_norm(g, 3.0)
    _check(before, g, norm, 3.0)
    mixed = [None if i % 3 == 0 else t for i, t in enumerate(before)]
    assert abs(float(gc.grad_norm(mixed)) - _norm([t for t in mixed if t is not None])) <= NORM_TOL * float(norm)


@pytest.mark.parametrize("sizes", [[2 ** 17], [2 ** 17 + 1], [2 ** 17 - 64] + [1] * 64, [127] * 1000, [255] * 1000,
                                   [2000] * 130, [10 ** 6] + [3] * 70],
                         ids=["one", "one more", "65", "1000 short", "1000", "130", "71"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=name)
def test_around_the_one_kernel_limit(cuda_device, sizes, dtype):
    before = _make(sizes, dtype, cuda_device)
    g = [t.clone() for t in before]
    norm = gc.clip_grad_norm(g, 7.0)
    _check(before, g, norm, 7.0)
    assert torch.equal(gc.grad_norm(before), norm)
    assert torch.equal(gc.clip_grad_norm(before, float("inf")), norm)  # nothing to do: the same bits again
    assert torch.equal(gc.grad_norm(before), norm)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_views_of_a_bucket_at_any_alignment(cuda_device, dtype):
    """Neighbouring views; what lies between and around them keeps its bytes."""
    rng = np.random.default_rng(1)
    flat = torch.from_numpy(rng.standard_normal(200_000)).to(dtype).to(cuda_device)
    cuts = [(1, 6), (6, 7), (9, 1034), (1037, 40_000), (40_000, 100_001), (100_003, 199_999)]
    keep = flat.clone()
    views = [flat[a:b] for a, b in cuts]
    before = [v.clone() for v in views]
    norm = gc.clip_grad_norm(views, 2.0)
    _check(before, views, norm, 2.0)
    mask = torch.ones(200_000, dtype=torch.bool, device=cuda_device)
    for a, b in cuts:
        mask[a:b] = False
    assert torch.equal(flat[mask], keep[mask])
    # an output that lies otherwise in its vectors than its source
    other = torch.zeros(200_003, dtype=dtype, device=cuda_device)
    out = [other[a + 3:b + 3] for a, b in cuts]
    # (not the views' bits: the alignment decides which thread squares what, so the two norms are two sums)
    _check(before, out, gc.clip_grad_norm(before, 2.0, out=out), 2.0)
    assert not other[:4].any() and not other[100_004:100_006].any()


def test_permuted_memory(cuda_device):
    a = torch.randn(30, 50, device=cuda_device)
    b = torch.randn(2, 8, 5, 6, device=cuda_device).to(memory_format=torch.channels_last)
    before = [a.clone(), b.clone()]
    _check(before, [a, b], gc.clip_grad_norm([a.t(), b], 1.0), 1.0)
    with pytest.raises(RuntimeError, match="gaps or repeats"):
        gc.grad_norm([a[:, ::2]])
    with pytest.raises(RuntimeError, match="gaps or repeats"):
        gc.clip_grad_norm([a[:1].expand(4, 50)], 1.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_range(cuda_device, dtype):
    """Squares that leave the type's or float32's range, on both sides."""
    for scale in (1e-30, 1e-22, 1e25, 1e36) if dtype != torch.float16 else (1e-6, 1e4):
        before = _make([1000, 77], dtype, cuda_device, scale=scale)
        n = _norm(before)
        g = [t.clone() for t in before]
        _check(before, g, gc.clip_grad_norm(g, n / 3, eps=0.0), n / 3, eps=0.0)
    if dtype != torch.float16:  # a factor below float32's range, elements that are not
        for high, low in ((1e30, 1e-20), (1e20, 1e-24), (1e36, 1e-10)):
            before = _make([1000, 300_000], dtype, cuda_device, scale=high)
            g = [t.clone() for t in before]
            _check(before, g, gc.clip_grad_norm(g, low, eps=0.0), low, eps=0.0)
    zero = [torch.zeros(5000, dtype=dtype, device=cuda_device)]
    assert float(gc.clip_grad_norm(zero, 1.0)) == 0.0 and not zero[0].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_not_finite(cuda_device, dtype):
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([1.0, inf, -2.0] + [0.5] * 30, dtype=dtype, device=cuda_device)
    h = torch.ones(20_000, dtype=dtype, device=cuda_device)
    assert float(gc.clip_grad_norm([g, h], 1.0)) == inf
    assert torch.isnan(g[1]) and not g[[0, 2]].any() and not h.any()
    g = torch.tensor([1.0, nan], dtype=dtype, device=cuda_device)
    h = torch.ones(20_000, dtype=dtype, device=cuda_device)
    assert math.isnan(float(gc.clip_grad_norm([g, h], 1.0)))
    assert torch.isnan(g).all() and torch.isnan(h).all()
    h = torch.ones(100, dtype=dtype, device=cuda_device)
    assert float(gc.clip_grad_norm([h], inf)) == 10.0 and (h == 1).all()


def test_empty_lists(cuda_device):
    assert float(gc.grad_norm([])) == 0.0 and float(gc.clip_grad_norm([None], 1.0)) == 0.0
    e = torch.empty(0, device=cuda_device)
    assert float(gc.grad_norm([e, e])) == 0.0 and float(gc.clip_grad_norm([e, e], 1.0)) == 0.0
    t = torch.full((), 3.0, device=cuda_device)
    assert float(gc.clip_grad_norm(t, 1.5, eps=0.0)) == 3.0 and float(t) == 1.5


def test_refusals(cuda_device):
    a = torch.ones(100, device=cuda_device)
    b = torch.ones(100, device=cuda_device)
    for call in (lambda: gc.grad_norm([a.cpu()]), lambda: gc.grad_norm([a.int()]), lambda: gc.clip_grad_norm([a], -1.0),
                 lambda: gc.clip_grad_norm([a], float("nan")), lambda: gc.clip_grad_norm([a], 1.0, eps=-1.0),
                 lambda: gc.grad_norm([a.to_sparse()]), lambda: gc.clip_grad_norm([a], 1.0, out=[b[:50]]),
                 lambda: gc.clip_grad_norm([a], 1.0, out=[b.half()]), lambda: gc.clip_grad_norm([a], 1.0, out=[]),
                 lambda: gc.clip_grad_norm([a], 1.0, out=b), lambda: gc.clip_grad_norm([a, b], 1.0, out=[a.clone(), None]),
                 # an element that would be scaled twice, or read after it was written
                 lambda: gc.clip_grad_norm([a, a], 1.0), lambda: gc.clip_grad_norm([a, a[40:60]], 1.0),
                 lambda: gc.clip_grad_norm([a, b], 1.0, out=[b, a]), lambda: gc.clip_grad_norm([a[:60]], 1.0, out=[a[40:]]),
                 lambda: gc.clip_grad_norm([a, b], 1.0, out=[torch.ones_like(a)] * 2)):
        with pytest.raises(RuntimeError):
            call()
    assert (a == 1).all() and (b == 1).all()
    assert abs(float(gc.grad_norm([a, a])) - math.sqrt(200)) < 1e-5  # read twice is fine
    gc.clip_grad_norm([a[:50], a[50:]], 1.0)  # neighbours are
    assert abs(float(gc.grad_norm(a)) - 1.0) < 1e-5


def test_writes_are_noticed(cuda_device):
    """A tensor that autograd has saved must not be scaled behind its back."""
    a = torch.ones(10, device=cuda_device, requires_grad=True)
    g = torch.full((10,), 3.0, device=cuda_device)
    loss = (a * g).sum()
    gc.clip_grad_norm([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        t = torch.ones(10, device=cuda_device)
        assert float(gc.clip_grad_norm(t, 1.0)) > 3.0
    with pytest.raises(RuntimeError):
        gc.clip_grad_norm(t, 0.1)
    assert float(t[0]) > 0.3


def test_stream_and_graphs(cuda_device):
    """On another stream; captured twice with the two graphs replayed together on new values."""
    sizes = [3_000_000, 17, 65_000]
    sets = [_make(sizes, torch.float32, cuda_device, seed=s) for s in range(2)]
    want = [gc.clip_grad_norm([t.clone() for t in s], 1.0) for s in sets]
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        got = gc.grad_norm(sets[0])
    both = gc.grad_norm(sets[1])
    torch.cuda.synchronize(cuda_device)
    assert torch.equal(got, want[0]) and torch.equal(both, want[1])
    graphs, norms, outs = [], [], []
    for s in sets:
        graph, out = torch.cuda.CUDAGraph(), [torch.empty_like(t) for t in s]
        with torch.cuda.graph(graph):
            norms.append(gc.clip_grad_norm(s, 1.0, out=out))
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream(cuda_device) for _ in sets]
    for r in range(3):
        for i, s in enumerate(sets):
            for t, v in zip(s, _make(sizes, torch.float32, cuda_device, seed=10 * r + i + 5)):
                t.copy_(v)
        torch.cuda.synchronize(cuda_device)
        for graph, stream in zip(graphs * 2, streams * 2):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize(cuda_device)
        for s, n, out in zip(sets, norms, outs):
            expect = [torch.empty_like(t) for t in s]
            assert torch.equal(n, gc.clip_grad_norm(s, 1.0, out=expect))
            assert all(torch.equal(x, y) for x, y in zip(out, expect))


def test_large_tensor(cuda_device):
    """More than 2^31 elements in one tensor."""
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    n = 2 ** 31 + 12_345
    t = torch.ones(n, dtype=torch.bfloat16, device=cuda_device)
    t[-5:] = 256.0
    norm = math.sqrt(n - 5 + 5 * 65536)
    assert abs(float(gc.clip_grad_norm(t, norm / 2, eps=0.0)) - norm) <= NORM_TOL * norm
    assert (t[:-5] == 0.5).all() and (t[-5:] == 128.0).all()


# ---------------------------------------------------------------------------- in front of the tables

@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("optimizer", [ops.Optimizer.SGD, ops.Optimizer.EXACT_ROWWISE_ADAGRAD])
def test_max_grad_norm_of_the_tables(cuda_device, fp16, optimizer):
    """The module with a limit does what the module without does on the scaled gradient; without a limit
    that is reached, the same bits."""
    T, E, D, B, L = 3, 200, 16, 32, 4
    torch.manual_seed(0)
    idx = torch.randint(0, E, (T * B * L,), dtype=torch.int32, device=cuda_device)
    off = torch.arange(0, T * B * L + 1, L, dtype=torch.int32, device=cuda_device)
    w0 = torch.randn(T * E, D, device=cuda_device)
    go = torch.randn(B, T, D, device=cuda_device, dtype=torch.float16 if fp16 else torch.float32)

    def trained(grad, **kw):
        m = ops.TableBatchedEmbeddingBags(T, E, D, optimizer=optimizer, learning_rate=0.1, eps=0.1, fp16=fp16, **kw).cuda()
        m.embedding_weights.data.copy_(w0)
        m(idx, off).backward(grad)
        return m.embedding_weights.detach().clone(), m.optimizer_state.clone()

    plain = trained(go)
    for grad in (go, go.transpose(0, 1).contiguous().transpose(0, 1)):  # the view the exchange hands over
        scaled = grad.clone()  # in the same memory order, which is the order of the sum
        gc.clip_grad_norm(scaled, 5.0)
        got, want = trained(grad, max_grad_norm=5.0), trained(scaled)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert not torch.equal(got[0], plain[0])
        high = trained(grad, max_grad_norm=1e6)
        assert torch.equal(high[0], plain[0]) and torch.equal(high[1], plain[1])
    kept = go.clone()
    trained(kept, max_grad_norm=5.0)
    assert torch.equal(kept, go)  # autograd's gradient is not written to
    one = torch.ones((), device=cuda_device, dtype=go.dtype).expand(B, T, D)  # out.sum().backward()
    got, want = trained(one, max_grad_norm=2.0), trained(one.contiguous(), max_grad_norm=2.0)
    assert torch.equal(got[0], want[0])


def test_max_grad_norm_of_a_lazily_negated_gradient(cuda_device):
    """A gradient with the negative bit is limited like any other."""
    idx = torch.arange(6, dtype=torch.int32, device=cuda_device)
    off = torch.arange(0, 7, 2, dtype=torch.int32, device=cuda_device)
    go = torch.randn(3, 1, 8, device=cuda_device)
    w0 = torch.randn(10, 8, device=cuda_device)
    rows = []
    for grad in (-go, torch._neg_view(go)):
        m = ops.TableBatchedEmbeddingBags(1, 10, 8, learning_rate=0.5, max_grad_norm=0.25).cuda()
        m.embedding_weights.data.copy_(w0)
        m(idx, off).backward(grad)
        rows.append(m.embedding_weights.detach().clone())
    assert torch.equal(rows[0], rows[1]) and not torch.equal(rows[0], w0)
