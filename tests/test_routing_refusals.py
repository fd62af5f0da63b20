"""What the routing and clipping entry points refuse before they touch a device, and the oracle of their
GPU tests against a second way of writing it down."""
import ctypes

import numpy as np
import pytest
import torch

import routing_testlib as ref
from sparse_ads_baselines_b200 import _lib
from sparse_ads_baselines_b200 import expert_routing as er
from sparse_ads_baselines_b200 import gradient_clipping as gc


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from sparse_ads_baselines_b200 import build
        build.build()
    return _lib.lib()


def test_there_is_no_cpu_path(lib):
    x = torch.zeros(4, 8)
    e = torch.zeros(4, 2, dtype=torch.int32)
    p = er.ExpertPlan(torch.zeros(3, dtype=torch.int32), e, torch.zeros(8, dtype=torch.int32))
    for call in (lambda: er.gate(x, 2), lambda: er.plan(e, 2), lambda: er.dispatch(x, p), lambda: er.combine(x, p),
                 lambda: gc.grad_norm([x]), lambda: gc.clip_grad_norm([x], 1.0)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_bad_arguments_of_the_c_entries(lib):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) & ~63
    f32, bad = _lib.TBE_F32, -1

    def refused(rc, text):
        assert rc < 0 and text in lib.tbe_last_error_string(), lib.tbe_last_error_string()

    refused(lib.tbe_expert_gate(None, 4, p, p, 1, 4, 1, f32, 1, None), b"null")
    refused(lib.tbe_expert_gate(p, 4, p, p, 1, 1025, 1, f32, 1, None), b"1..1024")
    refused(lib.tbe_expert_gate(p, 4, p, p, 1, 4, 0, f32, 1, None), b"k 1..32")
    refused(lib.tbe_expert_gate(p, 4, p, p, 1, 4, 5, f32, 1, None), b"k must be")
    refused(lib.tbe_expert_gate(p, 4, p, p, -1, 4, 1, f32, 1, None), b"tbe_expert_gate")
    refused(lib.tbe_expert_gate(p, 4, p, p, 1, 4, 1, 9, 1, None), b"bad dtype")
    refused(lib.tbe_expert_gate(p, -4, p, p, 2, 4, 1, f32, 1, None), b"stride")
    refused(lib.tbe_expert_gate_backward(None, p, 4, p, p, p, 1, 4, 1, f32, 1, None), b"null")
    refused(lib.tbe_expert_plan_workspace_bytes(-1, 4), b"M must be")
    refused(lib.tbe_expert_plan_workspace_bytes(1 << 31, 4), b"M must be")
    refused(lib.tbe_expert_plan_workspace_bytes(8, 0), b"E 1..1024")
    refused(lib.tbe_expert_plan_workspace_bytes((1 << 31) - 1024, 4), b"M must be")
    assert lib.tbe_expert_plan_workspace_bytes((1 << 31) - 1025, 4) > 0
    assert lib.tbe_expert_plan_workspace_bytes(131_072, 1024) == 0
    need = lib.tbe_expert_plan_workspace_bytes(200_000, 1024)
    assert need > 0
    refused(lib.tbe_expert_plan(p, p, p, p, 200_000, 1024, p, need - 1, None), b"workspace")
    refused(lib.tbe_expert_plan(p, None, p, p, 8, 4, None, 0, None), b"null")
    refused(lib.tbe_expert_dispatch(None, 4, p, p, p, 1, 1, 4, 2, f32, None), b"null")
    refused(lib.tbe_expert_dispatch(p, 4, p, p, p, 1, 0, 4, 2, f32, None), b"k and D > 0")
    refused(lib.tbe_expert_dispatch(p, 4, p, p, p, 1 << 30, 2, 4, 2, f32, None), b"2^31")
    refused(lib.tbe_expert_dispatch(p, 4, p, p, p, 1, 1, 4, 0, f32, None), b"E must be")
    refused(lib.tbe_expert_combine(p, p, p, None, p, 1, 1, 0, 2, f32, None), b"k and D > 0")
    refused(lib.tbe_expert_combine(p, p, p, None, p, 1, 1, 4, 2, bad, None), b"bad dtype")
    refused(lib.tbe_expert_combine_backward(p, 4, None, p, p, p, None, p, 1, 1, 4, 2, f32, None), b"null")
    ptrs = (ctypes.c_void_p * 2)(p, p)
    sizes, types = (ctypes.c_int64 * 2)(4, 4), (ctypes.c_int32 * 2)(f32, f32)
    need = lib.tbe_grad_norm_workspace_bytes(2)
    big = ctypes.create_string_buffer(need + 64)
    ws = (ctypes.addressof(big) + 63) & ~63
    refused(lib.tbe_grad_norm(ptrs, sizes, types, 2, None, ws, need, None), b"null")
    refused(lib.tbe_grad_norm(ptrs, sizes, types, 2, p, ws, need - 1, None), b"workspace")
    refused(lib.tbe_grad_norm(ptrs, sizes, types, -1, p, ws, need, None), b"number of tensors")
    refused(lib.tbe_grad_clip(ptrs, ptrs, sizes, types, 2, 1.0, 1e-6, p, ws, need, None), b"shares memory")
    refused(lib.tbe_grad_clip(ptrs, None, sizes, types, 2, 1.0, 1e-6, p, ws, need, None), b"null")
    refused(lib.tbe_grad_clip(ptrs, ptrs, sizes, types, 1, -1.0, 1e-6, p, ws, need, None), b"negative")
    refused(lib.tbe_grad_clip(ptrs, ptrs, sizes, types, 1, float("nan"), 1e-6, p, ws, need, None), b"negative")
    types[1] = 7
    refused(lib.tbe_grad_norm(ptrs, sizes, types, 2, p, ws, need, None), b"bad dtype")
    odd = (ctypes.c_void_p * 1)(p + 2)
    refused(lib.tbe_grad_norm(odd, sizes, types, 1, p, ws, need, None), b"aligned")


def test_misaligned_pointers_of_the_c_entries(lib):
    """An address that is no multiple of its elements' size faults on the GPU; the host refuses it."""
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 63) & ~63
    types = [(_lib.TBE_F16, 2, 4), (_lib.TBE_BF16, 2, 4), (_lib.TBE_F32, 4, 4), (_lib.TBE_F64, 8, 8)]

    def refused_one_by_one(call, sizes):
        for i, size in enumerate(sizes):
            args = [p] * len(sizes)
            args[i] = p + size // 2
            assert call(*args) == -1 and b"aligned" in lib.tbe_last_error_string(), (i, lib.tbe_last_error_string())

    for t, es, ws in types:
        refused_one_by_one(lambda x, w, e: lib.tbe_expert_gate(x, 4, w, e, 1, 4, 1, t, 1, None), [es, ws, 4])
        for ren in (0, 1):
            refused_one_by_one(lambda g, w, e, d: lib.tbe_expert_gate_backward(g, p, 4, w, e, d, 1, 4, 1, t, ren, None),
                               [ws, ws, 4, es])
        refused_one_by_one(lambda x: lib.tbe_expert_gate_backward(p, x, 4, p, p, p, 1, 4, 1, t, 0, None), [es])
        refused_one_by_one(lambda x, q, o, y: lib.tbe_expert_dispatch(x, 4, q, o, y, 1, 1, 4, 2, t, None), [es, 4, 4, es])
        refused_one_by_one(lambda y, q, o, w, d: lib.tbe_expert_combine(y, q, o, w, d, 1, 1, 4, 2, t, None),
                           [es, 4, 4, ws, es])
        refused_one_by_one(
            lambda g, y, q, o, w, dy, dw: lib.tbe_expert_combine_backward(g, 4, y, q, o, w, dy, dw, 1, 1, 4, 2, t, None),
            [es, es, 4, 4, ws, es, ws])
    refused_one_by_one(lambda e, o, q, r: lib.tbe_expert_plan(e, o, q, r, 8, 4, None, 0, None), [4] * 4)
    need = lib.tbe_expert_plan_workspace_bytes(200_000, 4)
    refused_one_by_one(lambda w: lib.tbe_expert_plan(p, p, p, p, 200_000, 4, w, need, None), [4])
    ptrs, one = (ctypes.c_void_p * 1)(p), (ctypes.c_void_p * 1)(p + 64)
    sizes, kinds = (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(_lib.TBE_F32)
    need = lib.tbe_grad_norm_workspace_bytes(1)
    refused_one_by_one(lambda n, w: lib.tbe_grad_norm(ptrs, sizes, kinds, 1, n, w, need, None), [4, 8])
    refused_one_by_one(lambda n, w: lib.tbe_grad_clip(ptrs, one, sizes, kinds, 1, 1.0, 0.0, n, w, need, None), [4, 8])


def test_the_gates_renormalized_gradient_needs_no_logits(lib):
    """As the header says: a call is refused for what it reads."""
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) & ~63
    for logits, stride in ((None, 4), (p + 1, 4), (p, -4)):
        rc = lib.tbe_expert_gate_backward(p, logits, stride, p, p, p, 2, 4, 1, _lib.TBE_F32, 0, None)
        assert rc == -1  # the other gradient reads them
        rc = lib.tbe_expert_gate_backward(p, logits, stride, p, p, p, 0, 4, 1, _lib.TBE_F32, 1, None)
        assert rc == 0, lib.tbe_last_error_string()
        rc = lib.tbe_expert_gate_backward(p, logits, stride, p, p, None, 2, 4, 1, _lib.TBE_F32, 1, None)
        assert rc == -1 and b"null" in lib.tbe_last_error_string()


def test_dense_memory_is_recognised():
    a = torch.zeros(4, 6, 5)
    assert all(gc._dense(t) for t in (a, a.permute(2, 0, 1), a[:1], a[2:3, 1:2], torch.zeros(()), torch.zeros(0, 3)))
    assert not any(gc._dense(t) for t in (a[:, ::2], a[:, :, :4], a[:1].expand(3, 6, 5)))


def test_the_oracle_against_loops():
    rng = np.random.default_rng(0)
    N, k, E, D = 9, 3, 5, 4
    x = np.round(rng.standard_normal((N, E)) * 2) / 2  # ties
    x[2] = -np.inf
    x[3, 1:] = -np.inf
    for renormalize in (True, False):
        w, e = ref.gate(x, k, renormalize)
        g = rng.standard_normal((N, k))
        d, _ = ref.gate_gradient(x, w, e, g, renormalize)
        for t in range(N):
            chosen = sorted((j for j in range(E) if x[t, j] > -np.inf), key=lambda j: (-x[t, j], j))[:k]
            assert list(e[t]) == chosen + [-1] * (k - len(chosen))
            over = chosen if renormalize else [j for j in range(E) if x[t, j] > -np.inf]
            total = sum(np.exp(x[t, j]) for j in over)
            assert np.allclose(w[t], [np.exp(x[t, j]) / total for j in chosen] + [0] * (k - len(chosen)))
            row = torch.tensor(x[t], requires_grad=True)  # the gradient by autograd
            if chosen:
                p = torch.softmax(row[over], 0)
                (p[[over.index(j) for j in chosen]] * torch.tensor(g[t, :len(chosen)])).sum().backward()
                assert np.allclose(d[t], row.grad.numpy())
            else:
                assert not d[t].any()
    ids = rng.integers(-1, E + 1, (N, k))
    offsets, positions, order = ref.plan(ids, E)
    flat = list(ids.reshape(-1))
    want = [i for b in range(E) for i in range(N * k) if flat[i] == b]
    want += [i for i in range(N * k) if not 0 <= flat[i] < E]
    assert list(order) == want and list(positions.reshape(-1)[want]) == list(range(N * k))
    assert list(offsets) == [sum(0 <= f < b for f in flat) for b in range(E + 1)]
    kept = offsets[-1]
    xs, y, w, g = (rng.standard_normal(s) for s in ((N, D), (N * k, D), (N, k), (N, D)))
    assert np.array_equal(ref.dispatch(xs, positions, kept),
                          np.array([xs[order[p] // k] if p < kept else np.zeros(D) for p in range(N * k)]))
    out = np.array([sum((w[t, s] * y[positions[t, s]] for s in range(k) if positions[t, s] < kept), np.zeros(D))
                    for t in range(N)])
    assert np.allclose(ref.combine(y, positions, kept, w), out)
    dy, dw = ref.combine_gradient(g, y, positions, kept, w)
    for t in range(N):
        for s in range(k):
            p = positions[t, s]
            assert np.allclose(dy[p], w[t, s] * g[t] if p < kept else 0)
            assert np.isclose(dw[t, s], g[t] @ y[p] if p < kept else 0)
