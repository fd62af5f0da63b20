"""Gate, plan, dispatch and combine against their definition in float64.

Tolerances count roundings (u = 2^-24 for accumulations in float32, 2^-53 in float64; h = half a step of
the result's type):

* gate weights: e = exp(l - top) carries the rounding of the difference, |l - top| u <= 64 u for the
  logits drawn here, and 2 units (4 u) of exp itself; the sum of E <= 1024 positive terms adds at most
  32 + 5 roundings (32 values per lane, five levels of the tree) and the errors of its terms; one division:
  64 + 4 + (64 + 4 + 37) + 1 < 180 u relative.
* gate gradient p (g - c): 180 u from p and w each, k + 5 roundings in c, three more operations: 450 u of
  the formula over absolute values, and h of the result.
* combine: k products and additions, (k + 1) u of the sum over absolute values, and h of the result.
* combine's weight gradient: a lane adds up to D/8 terms, then five levels, then four warps:
  (D/8 + 12) u of the sum over absolute values.
"""
import numpy as np
import pytest
import torch

import routing_testlib as ref
from routing_testlib import HALF_STEP, TINY, assert_within, f64, name, unit
from sparse_ads_baselines_b200 import expert_routing as er

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def _randn(rng, shape, dtype, device, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(dtype).to(device)


def _wdtype(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _choices(rng, N, k, E, dropped, device):
    ids = rng.integers(0, E, size=(N, k)).astype(np.int32)
    away = rng.random((N, k)) < dropped
    odd = rng.choice(np.array([-1, E, 2 ** 31 - 1, -2 ** 31], dtype=np.int64), size=(N, k)).astype(np.int32)
    return torch.from_numpy(np.where(away, odd, ids)).to(device)


# ---------------------------------------------------------------------------- gate

GATE_SIZES = [(1, 1, 1), (1, 64, 6), (3, 2, 2), (5, 7, 3), (33, 8, 2), (64, 60, 4), (17, 61, 8), (100, 256, 8), (9, 257, 5),
              (7, 512, 32), (5, 1000, 1), (6, 1024, 32), (3, 32, 32), (1025, 16, 1)]


def _gate_logits(rng, N, E, dtype, masked):
    x = rng.standard_normal((N, E)) * 3
    if masked:
        x[rng.random((N, E)) < 0.3] = -np.inf
        x[rng.random(N) < 0.2] = -np.inf
        x[0] = -np.inf
    else:
        x.reshape(-1)[::7] = np.round(x.reshape(-1)[::7])  # ties, in every type
        x.reshape(-1)[::11] = 0.0
        x.reshape(-1)[5::11] = -0.0  # equal to +0: the lower index goes first
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("N,E,k", GATE_SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_gate(cuda_device, N, E, k, dtype, renormalize, masked):
    rng = np.random.default_rng(N * 1000 + E + k)
    x = _gate_logits(rng, N, E, dtype, masked).to(cuda_device).requires_grad_()
    w, e = er.gate(x, k, renormalize=renormalize)
    assert w.dtype == _wdtype(dtype) and e.dtype == torch.int32 and w.shape == e.shape == (N, k)
    wr, exr = ref.gate(f64(x), k, renormalize)
    assert np.array_equal(e.cpu().numpy(), exr)
    u = unit(dtype)
    assert_within(w, wr, 180 * u * np.abs(wr) + TINY[name(w.dtype)], "weights")
    g = _randn(rng, (N, k), w.dtype, cuda_device)
    dx, = torch.autograd.grad(w, x, g)
    assert dx.dtype == dtype and dx.shape == x.shape
    dr, scale = ref.gate_gradient(f64(x), wr, exr, f64(g), renormalize)
    assert_within(dx, dr, 450 * u * scale + HALF_STEP[name(dtype)] * np.abs(dr) * (1 + 2 ** -7) + TINY[name(dtype)] * 1.01, "gradient")
    # without autograd: the same bits
    with torch.no_grad():
        w2, e2 = er.gate(x, k, renormalize=renormalize)
    assert torch.equal(w2, w) and torch.equal(e2, e)


@pytest.mark.parametrize("N,E,k", [(16384, 256, 8), (16387, 130, 5), (16385, 512, 8), (16386, 999, 4), (16391, 256, 32),
                                   (16384, 256, 9)])
@pytest.mark.parametrize("dtype,renormalize,masked", [(torch.bfloat16, True, True), (torch.float16, False, False)],
                         ids=["bfloat16-masked", "float16-whole"])
def test_gate_many_rows(cuda_device, N, E, k, dtype, renormalize, masked):
    test_gate(cuda_device, N, E, k, dtype, renormalize, masked)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_gate_strides(cuda_device, dtype):
    rng = np.random.default_rng(3)
    wide = _randn(rng, (40, 100), dtype, cuda_device)
    for x in (wide[:, 3:67], wide[:, 8:72], wide.t(), wide[5:6].expand(30, 100), wide[::3]):
        base = x.contiguous()
        for renormalize in (True, False):
            a, b = x.detach().requires_grad_(), base.detach().requires_grad_()
            (wa, ea), (wb, eb) = er.gate(a, 5, renormalize), er.gate(b, 5, renormalize)
            assert torch.equal(ea, eb)
            g = _randn(rng, wa.shape, wa.dtype, cuda_device)
            da, = torch.autograd.grad(wa, a, g.t().contiguous().t())
            db, = torch.autograd.grad(wb, b, g)
            if renormalize:
                assert torch.equal(wa, wb) and torch.equal(da, db)
            else:  # the alignment decides which lane sums which columns
                u, h = unit(dtype), HALF_STEP[name(dtype)]
                assert_within(wa, f64(wb), 360 * u * f64(wb))
                dr, scale = ref.gate_gradient(f64(b), f64(wb), eb.cpu().numpy(), f64(g), False)
                assert_within(da, f64(db), 900 * u * scale + 2 * h * np.abs(dr) * (1 + 2 ** -7) + 2.02 * TINY[name(dtype)])


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("renormalize", [True, False])
def test_gate_not_a_number(cuda_device, dtype, renormalize):
    """NaN and +inf make their own row's weights NaN; ids stay distinct and other rows whole."""
    x = torch.zeros(4, 40, dtype=dtype, device=cuda_device)
    x[:, 3], x[:, 9] = 2.0, 1.0
    x[1, 20] = float("nan")
    x[2, 30] = float("inf")
    x.requires_grad_()
    w, e = er.gate(x, 3, renormalize=renormalize)
    assert e.tolist() == [[3, 9, 0], [20, 3, 9], [30, 3, 9], [3, 9, 0]]
    assert torch.isnan(w[1:3]).all() and torch.isfinite(w[0]).all() and torch.equal(w[0], w[3])
    dx, = torch.autograd.grad(w.sum(), x)
    assert torch.isfinite(dx[0]).all() and torch.isnan(dx[1, 20]) and torch.isnan(dx[2, 30])
    assert torch.isnan(dx[1:3]).all() == (not renormalize)


def test_gate_lowest_values(cuda_device):
    """The lowest finite value is a value, not a mask."""
    for dtype in DTYPES:
        low = torch.finfo(dtype).min
        x = torch.full((2, 12), low, dtype=dtype, device=cuda_device)
        x[1, 4:] = float("-inf")
        w, e = er.gate(x, 6)
        assert e.tolist() == [[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, -1, -1]]
        assert_within(w, np.array([[1 / 6] * 6, [0.25] * 4 + [0.0] * 2]), 1e-6)


def test_gate_gradient_of_a_settled_router(cuda_device):
    """One weight nearly 1: the renormalized gradient keeps its relative accuracy (every term of w_s sum_j w_j
    (g_s - g_j) has the errors of two weights, 360 u, and of its operations; the gradients differ by more than an
    eighth of the larger, so their difference costs no more than 16 u)."""
    rng = np.random.default_rng(8)
    x = torch.zeros(500, 40, device=cuda_device)
    x[:, 7] = torch.from_numpy(rng.uniform(8, 14, 500)).float().to(cuda_device)
    x.requires_grad_()
    w, e = er.gate(x, 2)
    g = torch.from_numpy(np.stack([rng.uniform(1, 2, 500), rng.uniform(-2, -1, 500)], 1)).float().to(cuda_device)
    dx, = torch.autograd.grad(w, x, g)
    wr, exr = ref.gate(f64(x), 2, True)
    # the reference in the same form: in float64 the other one would do as well
    first = wr[:, 0] * wr[:, 1] * (f64(g)[:, 0] - f64(g)[:, 1])
    want = np.zeros((500, 40))
    want[np.arange(500), exr[:, 0]], want[np.arange(500), exr[:, 1]] = first, -first
    assert float(w.detach()[:, 0].min()) > 0.999
    assert_within(dx, want, 400 * unit(torch.float32) * np.abs(want))


def test_gate_gradcheck(cuda_device):
    torch.manual_seed(0)
    x = torch.randn(6, 20, dtype=torch.float64, device=cuda_device, requires_grad=True)
    for renormalize in (True, False):
        assert torch.autograd.gradcheck(lambda t: er.gate(t, 4, renormalize)[0], (x,))


# ---------------------------------------------------------------------------- plan

@pytest.mark.parametrize("N,k", [(0, 3), (1, 1), (1, 8), (7, 1), (128, 8), (129, 8), (1025, 1), (512, 8), (4097, 1), (1025, 8),
                                 (2731, 3), (20000, 2), (16384, 8), (131073, 1), (50001, 7), (200000, 8)])
@pytest.mark.parametrize("E", [1, 2, 61, 256, 1024])
def test_plan(cuda_device, N, k, E):
    rng = np.random.default_rng(N + k + E)
    experts = _choices(rng, N, k, E, 0.1, cuda_device)
    p = er.plan(experts, E)
    offsets, positions, order = ref.plan(experts.cpu().numpy(), E)
    assert np.array_equal(p.offsets.cpu().numpy(), offsets)
    assert np.array_equal(p.positions.cpu().numpy(), positions)
    assert np.array_equal(p.order.cpu().numpy(), order)


def test_plan_all_alike(cuda_device):
    """One expert takes everything; nobody takes anything; a transposed view."""
    for value in (3, -1):
        ids = torch.full((9000, 4), value, dtype=torch.int32, device=cuda_device)
        p = er.plan(ids, 5)
        assert torch.equal(p.positions.view(-1).cpu(), torch.arange(36000, dtype=torch.int32))
        assert p.offsets.tolist() == ([0, 0, 0, 0, 36000, 36000] if value == 3 else [0] * 6)
    ids = torch.randint(0, 9, (3, 500), dtype=torch.int32, device=cuda_device).t()
    a, b = er.plan(ids, 9), er.plan(ids.contiguous(), 9)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------------------- dispatch

ROW_SIZES = [(1, 1, 1, 1), (3, 2, 4, 3), (5, 3, 2, 4), (65, 8, 16, 7), (40, 6, 61, 1001), (33, 5, 8, 1004), (300, 1, 3, 8),
             (257, 7, 9, 100), (64, 12, 32, 64), (20, 33, 40, 128), (130, 8, 128, 768), (16, 2, 4, 4096), (9, 3, 4, 10000)]


def _cases(N, k, E, D, dtype, dropped, device, seed=0):
    rng = np.random.default_rng(N + k + E + D + seed)
    experts = _choices(rng, N, k, E, dropped, device)
    p = er.plan(experts, E)
    offsets, positions, _ = ref.plan(experts.cpu().numpy(), E)
    return rng, p, positions, int(offsets[-1])


@pytest.mark.parametrize("N,k,E,D", ROW_SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
def test_dispatch(cuda_device, N, k, E, D, dtype, dropped):
    rng, p, positions, kept = _cases(N, k, E, D, dtype, dropped, cuda_device)
    x = _randn(rng, (N, D), dtype, cuda_device).requires_grad_()
    y = er.dispatch(x, p)
    assert np.array_equal(f64(y), ref.dispatch(f64(x), positions, kept))
    g = _randn(rng, (N * k, D), dtype, cuda_device)
    g[kept:] = float("nan")  # what lies behind the kept rows belongs to nobody
    dx, = torch.autograd.grad(y, x, g)
    gr = np.nan_to_num(f64(g))
    dr = ref.combine(gr, positions, kept)
    bound = (k + 1) * unit(dtype) * ref.combine(np.abs(gr), positions, kept)
    assert_within(dx, dr, bound + HALF_STEP[name(dtype)] * (np.abs(dr) + bound) + TINY[name(dtype)], "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=name)
def test_dispatch_strides(cuda_device, dtype):
    rng, p, positions, kept = _cases(24, 3, 5, 40, dtype, 0.2, cuda_device)
    wide = _randn(rng, (72, 99), dtype, cuda_device)
    for x in (wide[:24, 1:41], wide[:24, 8:48], wide[::3, :40], wide[:40, :24].t(), wide[3:4, :40].expand(24, 40)):
        x = x.detach().requires_grad_()
        y = er.dispatch(x, p)
        assert np.array_equal(f64(y), ref.dispatch(f64(x), positions, kept))
        wide_g = _randn(rng, (72, 45), dtype, cuda_device)
        a, = torch.autograd.grad(er.dispatch(x, p), x, wide_g[:, 2:42])
        b, = torch.autograd.grad(y, x, wide_g[:, 2:42].contiguous())
        assert torch.equal(a, b)


def test_positions_outside_are_skipped(cuda_device):
    """A plan that was tampered with reaches no memory outside the tensors."""
    rng, p, positions, kept = _cases(16, 2, 4, 32, torch.float32, 0.0, cuda_device)
    bad = p.positions.clone()
    bad[3, 0], bad[4, 1], bad[5, 0] = -1, 32, 2 ** 31 - 1
    q = er.ExpertPlan(p.offsets, bad, p.order)
    x = _randn(rng, (16, 32), torch.float32, cuda_device).requires_grad_()
    w = torch.ones(16, 2, device=cuda_device, requires_grad=True)
    er.dispatch(x, q)
    y = _randn(rng, (32, 32), torch.float32, cuda_device).requires_grad_()
    out = er.combine(y, q, w)
    assert torch.equal(out[3], y[positions[3, 1]]) and torch.equal(out[4], y[positions[4, 0]])
    dy, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert dw[3, 0] == 0 and dw[4, 1] == 0 and dw[5, 0] == 0
    far = er.ExpertPlan(torch.full_like(p.offsets, 2 ** 30), p.positions, p.order)
    assert torch.equal(er.dispatch(x, far), er.dispatch(x, p))
    none = er.ExpertPlan(torch.full_like(p.offsets, -5), p.positions, p.order)
    assert not er.dispatch(x, none).any() and not er.combine(y, none, w).any()


# ---------------------------------------------------------------------------- combine

@pytest.mark.parametrize("N,k,E,D", ROW_SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(cuda_device, N, k, E, D, dtype, dropped, weighted):
    rng, p, positions, kept = _cases(N, k, E, D, dtype, dropped, cuda_device)
    y = _randn(rng, (N * k, D), dtype, cuda_device)
    y[kept:] = float("nan")
    y.requires_grad_()
    w = torch.from_numpy(rng.standard_normal((N, k))).to(_wdtype(dtype)).to(cuda_device)
    w[(torch.from_numpy(positions).to(cuda_device) >= kept)] = float("inf")  # nobody's: never multiplied
    w.requires_grad_()
    out = er.combine(y, p, w if weighted else None)
    yr = np.nan_to_num(f64(y))
    wr = np.where(positions < kept, f64(w), 0.0) if weighted else np.ones((N, k))
    o, u, h = ref.combine(yr, positions, kept, wr), unit(dtype), HALF_STEP[name(dtype)]
    bound = (k + 1) * u * ref.combine(np.abs(yr), positions, kept, np.abs(wr))
    assert_within(out, o, bound + h * (np.abs(o) + bound) + TINY[name(dtype)], "out")
    g = _randn(rng, (N, D), dtype, cuda_device)
    dyr, dwr = ref.combine_gradient(f64(g), yr, positions, kept, wr)
    if weighted:
        dy, dw = torch.autograd.grad(out, (y, w), g)
        _, dw_scale = ref.combine_gradient(np.abs(f64(g)), np.abs(yr), positions, kept, wr)
        assert_within(dw, dwr, (D / 8 + 12) * u * dw_scale + TINY[name(dw.dtype)], "weights' gradient")
    else:
        dy, = torch.autograd.grad(out, y, g)
    bound = u * np.abs(dyr)
    assert_within(dy, dyr, bound + h * (np.abs(dyr) + bound) + TINY[name(dtype)], "rows' gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=name)
def test_combine_one_gradient_at_a_time(cuda_device, dtype):
    rng, p, _, _ = _cases(50, 3, 7, 200, dtype, 0.1, cuda_device)
    y, w = _randn(rng, (150, 200), dtype, cuda_device), _randn(rng, (50, 3), torch.float32, cuda_device)
    g = _randn(rng, (50, 200), dtype, cuda_device)
    ya, wa = y.clone().requires_grad_(), w.clone().requires_grad_()
    dy, dw = torch.autograd.grad(er.combine(ya, p, wa), (ya, wa), g)
    assert torch.equal(torch.autograd.grad(er.combine(ya, p, w), ya, g)[0], dy)
    assert torch.equal(torch.autograd.grad(er.combine(y, p, wa), wa, g)[0], dw)
    # a gradient that is a view of something wider, or one row for all
    wide = torch.zeros(50, 333, dtype=dtype, device=cuda_device)
    wide[:, 100:300] = g
    dy2, dw2 = torch.autograd.grad(er.combine(ya, p, wa), (ya, wa), wide[:, 100:300])
    # the strided rows are aligned to fewer bytes: another order of the same sum, each side within its bound
    dw_bound = 2 * (200 / 8 + 12) * unit(dtype) * ref.combine_gradient(
        np.abs(f64(g)), np.abs(f64(y)), p.positions.cpu().numpy(), int(p.offsets[-1]), f64(w))[1]
    assert torch.equal(dy2, dy)
    assert_within(dw2, f64(dw), dw_bound)
    one = g[:1].expand(50, 200)
    dy3, dw3 = torch.autograd.grad(er.combine(ya, p, wa), (ya, wa), one)
    dy4, dw4 = torch.autograd.grad(er.combine(ya, p, wa), (ya, wa), one.contiguous())
    assert torch.equal(dy3, dy4) and torch.equal(dw3, dw4)
    # rows and weights that are not contiguous
    yt = torch.empty(200, 150, dtype=dtype, device=cuda_device).t()
    yt.copy_(y)
    assert torch.equal(er.combine(yt, p, w.t().contiguous().t()), er.combine(y, p, w))


def test_rows_gradcheck(cuda_device):
    _, p, _, _ = _cases(7, 3, 4, 5, torch.float64, 0.3, cuda_device)
    torch.manual_seed(1)
    x = torch.randn(7, 5, dtype=torch.float64, device=cuda_device, requires_grad=True)
    y = torch.randn(21, 5, dtype=torch.float64, device=cuda_device, requires_grad=True)
    w = torch.randn(7, 3, dtype=torch.float64, device=cuda_device, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: er.dispatch(t, p), (x,))
    assert torch.autograd.gradcheck(lambda a, b: er.combine(a, p, b), (y, w))
    assert torch.autograd.gradcheck(lambda a: er.combine(a, p), (y,))


def test_no_rows(cuda_device):
    w, e = er.gate(torch.empty(0, 8, device=cuda_device, requires_grad=True), 2)
    assert w.shape == e.shape == (0, 2)
    w.sum().backward()
    p = er.plan(e, 8)
    x = torch.empty(0, 16, device=cuda_device, requires_grad=True)
    y = er.dispatch(x, p)
    out = er.combine(y, p, w.detach())
    assert y.shape == out.shape == (0, 16) and p.offsets.tolist() == [0] * 9
    out.sum().backward()
    assert x.grad.shape == (0, 16)


def test_past_32_bit_offsets(cuda_device):
    """2.5 G elements in expert order: addresses, and pair indices of unaligned rows, pass 32 bits."""
    free, _ = torch.cuda.mem_get_info()
    if free < 80 << 30:
        pytest.skip("needs 80 GB of free device memory")
    for N, k, D in ((620_000, 2, 2048), (2_200_000, 1, 2049)):
        g = torch.Generator(device=cuda_device).manual_seed(1)
        experts = torch.randint(0, 64, (N, k), generator=g, device=cuda_device, dtype=torch.int32)
        p = er.plan(experts, 64)
        x = torch.randint(-8, 8, (N, D), generator=g, device=cuda_device, dtype=torch.int8).to(torch.bfloat16)
        y = er.dispatch(x, p)
        assert y.numel() > 2 ** 31
        for t in range(0, N, 100_000):
            n = min(N, t + 100_000)
            assert torch.equal(y[p.positions[t:n].long()], x[t:n, None].expand(-1, k, -1))
        w = torch.full((N, k), 0.5, device=cuda_device, requires_grad=True)
        y.requires_grad_()
        out = er.combine(y, p, w)
        assert torch.equal(out, x * (k * 0.5))
        dy, dw = torch.autograd.grad(out, (y, w), x)
        for t in range(0, N, 100_000):
            n = min(N, t + 100_000)
            assert torch.equal(dy[p.positions[t:n].long()], (x[t:n, None] * 0.5).expand(-1, k, -1))
            # whole numbers below 2^24: the sums are exact
            assert torch.equal(dw[t:n], x[t:n].float().square().sum(1, keepdim=True).expand(-1, k))
        del x, y, out, dy, dw, w
        torch.cuda.empty_cache()


def test_several_launches(cuda_device):
    """Calls beyond 2^32 threads are cut by samples; the knob makes small ones take the same way."""
    from sparse_ads_baselines_b200 import _lib
    for D, dtype in ((64, torch.bfloat16), (33, torch.float32), (1001, torch.float32), (1024, torch.float16)):
        rng, p, _, _ = _cases(100, 3, 8, D, dtype, 0.2, cuda_device)
        x = _randn(rng, (100, D + 3), dtype, cuda_device)[:, 1:D + 1]
        y = _randn(rng, (300, D), dtype, cuda_device)
        w = _randn(rng, (100, 3), torch.float32, cuda_device)
        a, b, c = er.dispatch(x, p), er.combine(y, p, w), er.combine(y, p)
        try:
            for most in (1, 7, 100, 333):
                _lib.call("tbe_set_tuning", b"row_threads", most)
                assert torch.equal(er.dispatch(x, p), a) and torch.equal(er.combine(y, p, w), b)
                assert torch.equal(er.combine(y, p), c)
        finally:
            _lib.call("tbe_set_tuning", b"row_threads", 0)


# ---------------------------------------------------------------------------- streams, graphs, repeats

def _step(logits, x, k, E):
    w, e = er.gate(logits, k)
    p = er.plan(e, E)
    y = er.dispatch(x, p)
    return er.combine(y * 2, p, w), p


def test_another_stream(cuda_device):
    rng = np.random.default_rng(0)
    logits, x = _randn(rng, (3000, 64), torch.float32, cuda_device), _randn(rng, (3000, 256), torch.float32, cuda_device)
    expected, _ = _step(logits, x, 4, 64)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        got, _ = _step(logits, x, 4, 64)
    again, _ = _step(logits, x, 4, 64)  # at the same time, on the first stream
    torch.cuda.synchronize(cuda_device)
    assert torch.equal(got, expected) and torch.equal(again, expected)


def test_two_captured_graphs_replay_together(cuda_device):
    """Captured, replayed on new inputs, two graphs at once on two streams: nothing is shared."""
    rng = np.random.default_rng(1)
    sizes = [(4000, 64, 4, 96), (2500, 256, 8, 128)]
    states, graphs, outs = [], [], []
    for N, E, k, D in sizes:
        logits, x = _randn(rng, (N, E), torch.bfloat16, cuda_device), _randn(rng, (N, D), torch.bfloat16, cuda_device)
        _step(logits, x, k, E)
        torch.cuda.synchronize(cuda_device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = _step(logits, x, k, E)
        states.append((logits, x))
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream(cuda_device) for _ in sizes]
    for r in range(3):
        for (logits, x), (N, E, k, D) in zip(states, sizes):
            logits.copy_(_randn(rng, (N, E), torch.bfloat16, cuda_device))
            x.copy_(_randn(rng, (N, D), torch.bfloat16, cuda_device))
        torch.cuda.synchronize(cuda_device)
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize(cuda_device)
        for (logits, x), (N, E, k, D), out in zip(states, sizes, outs):
            assert torch.equal(out, _step(logits, x, k, E)[0])


def test_captured_training_step(cuda_device):
    """Forward and backward captured together, from tensors that have no eager graph."""
    rng = np.random.default_rng(4)
    N, E, k, D = 600, 32, 3, 64
    logits = _randn(rng, (N, E), torch.float32, cuda_device).requires_grad_()
    x = _randn(rng, (N, D), torch.float32, cuda_device).requires_grad_()
    g = _randn(rng, (N, D), torch.float32, cuda_device)

    def step(a, b):
        out, _ = _step(a, b, k, E)
        return (out.detach(),) + torch.autograd.grad(out, (a, b), g)

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        step(logits, x)
    torch.cuda.synchronize(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(logits, x)
    for _ in range(2):
        with torch.no_grad():
            logits.copy_(_randn(rng, (N, E), torch.float32, cuda_device))
            x.copy_(_randn(rng, (N, D), torch.float32, cuda_device))
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        want = step(logits.detach().clone().requires_grad_(), x.detach().clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [100, 5000, 200_000])
def test_captured_plan_of_many_experts(cuda_device, M):
    """More shared memory than a kernel has without asking, in every form of the plan, captured and replayed."""
    ids = torch.randint(0, 1024, (M, 1), dtype=torch.int32, device=cuda_device)
    er.plan(ids, 1024)
    torch.cuda.synchronize(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = er.plan(ids, 1024)
    for _ in range(2):
        ids.copy_(torch.randint(-1, 1025, (M, 1), dtype=torch.int32, device=cuda_device))
        graph.replay()
        want = ref.plan(ids.cpu().numpy(), 1024)
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, want))


def test_broadcast_inputs(cuda_device):
    """One row or one weight for all samples: the gradient is summed over what was broadcast."""
    rng, p, positions, kept = _cases(30, 2, 4, 24, torch.float64, 0.2, cuda_device)
    row = _randn(rng, (24,), torch.float64, cuda_device).requires_grad_()
    weight = _randn(rng, (2,), torch.float64, cuda_device).requires_grad_()
    y = er.dispatch(row.expand(30, 24), p)
    out = er.combine(y, p, weight.expand(30, 2))
    g = _randn(rng, (30, 24), torch.float64, cuda_device)
    d_row, d_weight = torch.autograd.grad(out, (row, weight), g)
    here = torch.from_numpy(positions < kept).to(cuda_device).double()
    # out[t] = (here[t] . weight) row
    torch.testing.assert_close(d_row, ((here @ weight.detach())[:, None] * g).sum(0), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(d_weight, (here * (g @ row.detach())[:, None]).sum(0), rtol=1e-12, atol=1e-12)


def test_saved_tensors_that_change_are_noticed(cuda_device):
    _, p, _, _ = _cases(10, 2, 4, 8, torch.float32, 0.0, cuda_device)
    y = torch.randn(20, 8, device=cuda_device, requires_grad=True) * 1.0
    w = torch.rand(10, 2, device=cuda_device, requires_grad=True)
    out = er.combine(y, p, w)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_same_bits_every_time(cuda_device):
    rng = np.random.default_rng(2)
    logits = _randn(rng, (20000, 128), torch.bfloat16, cuda_device).requires_grad_()
    x = _randn(rng, (20000, 512), torch.bfloat16, cuda_device).requires_grad_()
    g = _randn(rng, (20000, 512), torch.bfloat16, cuda_device)
    first = None
    for _ in range(4):
        out, p = _step(logits, x, 6, 128)
        now = [out.detach(), *p, *torch.autograd.grad(out, (logits, x), g)]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_noncurrent_grad_modes(cuda_device):
    x = torch.randn(4, 8, device=cuda_device, requires_grad=True)
    with torch.no_grad():
        w, e = er.gate(x, 2)
    assert not w.requires_grad
    p = er.plan(e, 8)
    with torch.no_grad():
        assert not er.dispatch(x, p).requires_grad
    y = er.dispatch(x, p)
    assert y.requires_grad and not e.requires_grad
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|differentiat"):
        d, = torch.autograd.grad(y.sum(), x, create_graph=True)
        d.sum().backward()


# ---------------------------------------------------------------------------- refusals that need a device

def test_refusals(cuda_device):
    x = torch.zeros(4, 8, device=cuda_device)
    e = torch.zeros(4, 2, dtype=torch.int32, device=cuda_device)
    p = er.plan(e, 3)
    w = torch.ones(4, 2, device=cuda_device)
    y = er.dispatch(x, p)
    bad = [
        lambda: er.gate(x, 0), lambda: er.gate(x, 9), lambda: er.gate(x.int(), 2), lambda: er.gate(x[0], 2),
        lambda: er.gate(torch.zeros(2, 1025, device=cuda_device), 2), lambda: er.gate(torch.zeros(2, 64, device=cuda_device), 33),
        lambda: er.plan(e.long(), 3), lambda: er.plan(e, 0), lambda: er.plan(e, 1025), lambda: er.plan(e.view(-1), 3),
        lambda: er.dispatch(x[:3], p), lambda: er.dispatch(x.int(), p), lambda: er.dispatch(x, tuple(p)),
        lambda: er.dispatch(x, p._replace(positions=p.positions.long())),
        lambda: er.dispatch(x, p._replace(positions=p.positions.t())),
        lambda: er.dispatch(x, p._replace(positions=p.positions.cpu())),
        lambda: er.dispatch(x, p._replace(offsets=p.offsets[:1])),
        lambda: er.dispatch(torch.zeros(4, 0, device=cuda_device), p),
        lambda: er.combine(y[:-1], p, w), lambda: er.combine(y, p, w[:3]), lambda: er.combine(y, p, w.half()),
        lambda: er.combine(y, p, w.cpu()), lambda: er.combine(y, None, w),
        lambda: er.dispatch(torch._neg_view(x), p), lambda: er.combine(y, p, torch._neg_view(w)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError("refusal %d was accepted" % i)
