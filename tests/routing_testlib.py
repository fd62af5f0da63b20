"""Expert routing and gradient clipping restated in float64 numpy, for the tests."""
import numpy as np

U32 = 2.0 ** -24  # half a unit in the last place of float32, relative
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
# half of the smallest subnormal: what rounding a value near zero may cost in absolute terms
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150, "float64": 0.0}


def f64(t):
    return t.detach().double().cpu().numpy()


def name(dtype):
    return str(dtype).replace("torch.", "")


def unit(dtype):
    """The rounding of one operation in the accumulator of `dtype`."""
    return 2.0 ** -53 if name(dtype) == "float64" else U32


def gate(x, k, renormalize):
    """(weights, experts) of finite or -inf logits."""
    index = np.argsort(-x, axis=1, kind="stable")[:, :k]  # ties keep the order of the columns
    chosen = np.take_along_axis(x, index, 1)
    live = chosen > -np.inf
    top = np.where(live[:, :1], chosen[:, :1], 0.0)
    e = np.exp(x - top)
    picked = np.take_along_axis(e, index, 1)
    total = picked.sum(1, keepdims=True) if renormalize else e.sum(1, keepdims=True)
    total[total == 0] = 1
    return picked / total, np.where(live, index, -1)


def gate_gradient(x, weights, experts, g, renormalize):
    """(gradient, the same formula over absolute values) -- the second is what its errors scale with."""
    n = np.arange(len(x))[:, None]
    slot = np.where(experts >= 0, experts, 0)
    g = np.where(experts >= 0, g, 0.0)
    c, c_abs = (weights * g).sum(1, keepdims=True), (weights * np.abs(g)).sum(1, keepdims=True)
    if renormalize:
        p, full, full_abs = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
        np.add.at(p, (n, slot), weights)
    else:
        top = np.max(x, 1, keepdims=True)
        e = np.exp(x - np.where(np.isfinite(top), top, 0.0))
        total = e.sum(1, keepdims=True)
        p = e / np.where(total == 0, 1, total)
        full, full_abs = np.zeros_like(x), np.zeros_like(x)
    np.add.at(full, (n, slot), g)
    np.add.at(full_abs, (n, slot), np.abs(g))
    return p * (full - c), p * (full_abs + c_abs)


def plan(experts, num_experts):
    flat = experts.reshape(-1).astype(np.int64)
    bins = np.where((flat >= 0) & (flat < num_experts), flat, num_experts)
    order = np.argsort(bins, kind="stable")
    positions = np.empty_like(order)
    positions[order] = np.arange(len(order))
    offsets = np.searchsorted(bins[order], np.arange(num_experts + 1))
    return offsets, positions.reshape(experts.shape), order


def dispatch(x, positions, kept):
    N, k = positions.shape
    y = np.zeros((N * k, x.shape[1]))
    y[positions.reshape(-1)] = np.repeat(x, k, axis=0)
    y[kept:] = 0
    return y


def combine(y, positions, kept, weights=None):
    here = positions < kept
    rows = np.where(here[:, :, None], y[np.where(here, positions, 0)], 0.0)
    return (rows if weights is None else rows * np.where(here, weights, 0.0)[:, :, None]).sum(1)


def combine_gradient(grad, y, positions, kept, weights):
    """(grad_y, grad_weights)"""
    here = positions < kept
    rows = np.where(here[:, :, None], y[np.where(here, positions, 0)], 0.0)
    dy = np.zeros_like(y)
    dy[positions.reshape(-1)] = (np.where(here, weights, 0.0)[:, :, None] * grad[:, None, :]).reshape(-1, y.shape[1])
    return dy, (rows * grad[:, None, :]).sum(2)


def assert_within(actual, expected, bound, what=""):
    """|actual - expected| <= bound everywhere; NaN only where expected is."""
    a = f64(actual) if hasattr(actual, "detach") else np.asarray(actual, dtype=np.float64)
    assert a.shape == expected.shape, "%s: shape %s, expected %s" % (what, a.shape, expected.shape)
    same = (a == expected) | (np.isnan(a) & np.isnan(expected))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(a - expected) <= bound)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d values are off; at %s got %r, expected %r, bound %r" % (
            what, bad.sum(), bad.size, i, a[i], expected[i], np.broadcast_to(bound, a.shape)[i]))
