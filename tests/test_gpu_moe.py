"""Routing to experts, the plan, the experts' layers and the weighted sum, against float64 and whole numbers; and a whole
feed-forward layer of experts."""
import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce
from test_gpu_w8a8 import DTYPES, FILL, KINDS, blank, check, choice, make, untouched, up  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- routing -----------------------------------------------------------------------------------

def route(lh, store, dtype, router, pad=0, with_plan=True):
    T, E = store.shape
    padded = np.zeros((T, E + pad), store.dtype)
    padded[:, :E] = store
    X = up(lh, padded)
    k = router.top_k
    ids, w = blank(lh, "i32", T, k), blank(lh, "f32", T, k)
    p = lh.MoePlan(T, E, k) if with_plan else None
    if p is not None:
        for a in (p.offsets, p.order, p.workspace):
            a.fill_bytes(FILL)
    lh.moe_route_raw(router.desc, dtype, X.ptr, E + pad, T, ids.ptr, w.ptr, p.desc if p is not None else None)
    lh.synchronize()
    return ids.to_numpy().T, w.to_numpy().T, p


def check_route(got, store, dtype, k, scale=1.0, **kw):
    ids, w, p = got
    want, ww = ref.route(ref.to_float(store, dtype), k, scale=scale, **kw)
    np.testing.assert_array_equal(ids, want)
    nan = np.isnan(ww)
    np.testing.assert_array_equal(np.isnan(w), nan)
    # exp's argument is rounded once (|x| below 128: 2^-17 of the result), exp, sums of up to 1024 in a tree of 26, quotients
    assert (np.abs(w - ww)[~nan] <= (np.abs(ww) * (2.0 ** -17 + 40 * ref.U) + 2.0 ** -140)[~nan]).all()
    if p is not None:
        offsets, order = ref.plan(want, store.shape[1])
        np.testing.assert_array_equal(p.offsets.to_numpy(), offsets)
        np.testing.assert_array_equal(p.order.to_numpy(), order)
        p.close()


CASES = [  # T, E, k, score, bias, groups, top_groups, group_best, renormalize, scale
    (1, 1, 1, "softmax", False, 1, 1, 1, True, 1.0), (1, 8, 2, "softmax", False, 1, 1, 1, True, 1.0),
    (3, 7, 7, "sigmoid", False, 1, 1, 1, False, 2.5), (63, 64, 8, "softmax", False, 1, 1, 1, False, 1.0),
    (64, 64, 8, "softmax", True, 1, 1, 1, True, 1.0), (65, 60, 4, "softmax", False, 1, 1, 1, True, 1.0),
    (130, 128, 6, "sigmoid", True, 1, 1, 1, True, 1.0), (200, 160, 6, "softmax", False, 8, 3, 1, False, 16.0),
    (100, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5), (70, 256, 32, "sigmoid", False, 8, 4, 2, True, 2.5),
    (33, 96, 3, "softmax", True, 4, 1, 2, False, 1.0), (50, 384, 6, "sigmoid", True, 1, 1, 1, True, 1.0),
    (20, 1024, 32, "softmax", True, 64, 16, 2, True, 1.0), (40, 257, 9, "softmax", False, 257 // 257, 1, 1, True, 1.0),
    (90, 64, 4, "sigmoid", False, 64, 5, 1, True, 1.0), (300, 66, 5, "sigmoid", True, 33, 7, 2, True, 1.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_route(gpu, dtype, i):
    lh = gpu
    T, E, k, score, biased, groups, top_groups, best, renorm, scale = CASES[i]
    announce(f"route {CASES[i]} {dtype}")
    rng = np.random.default_rng(200 + i)
    store = ref.to_store(rng.standard_normal((T, E)) * 2, dtype)
    bias = (rng.standard_normal(E) * 0.2).astype(np.float32) if biased else None
    B = up(lh, bias) if biased else None
    r = lh.MoeRouter(E, k, score, B, groups, top_groups, best, renorm, scale)
    check_route(route(lh, store, dtype, r, pad=i % 3), store, dtype, k, scale, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_best=best, renormalize=renorm)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,top,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_route_of_equal_and_nearly_equal_scores(gpu, score, biased, groups, top, best):
    """Logits of a few values only: equal ones go to the lower number; and logits one step apart, whose scores 32 bits round
    to the same or to the wrong order, with biases that make up for the difference."""
    lh = gpu
    announce(f"route ties {score} bias={biased} {groups} {top} {best}")
    rng = np.random.default_rng(5)
    T, E, k = 150, 64, 6
    x = rng.integers(-2, 3, (T, E)).astype(np.float32)
    x[50:] = (rng.standard_normal((100, 1)) + rng.integers(0, 3, (100, E)) * 2.0 ** -22).astype(np.float32)
    x[100:, ::2] += np.float32(0.5)
    bias = None
    if biased:
        p = 1 / (1 + np.exp(-0.5))
        bias = (rng.integers(0, 2, E) * 0.25 + rng.integers(-2, 3, E) * 2.0 ** -24 + p * 0).astype(np.float32)
    B = up(lh, bias) if biased else None
    r = lh.MoeRouter(E, k, score, B, groups, top, best)
    check_route(route(lh, x, "f32", r), x, "f32", k, score=score, bias=bias, groups=groups, top_groups=top, group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(8, 4), (24, 12), (400, 50)])
@pytest.mark.parametrize("most", [0.5, 64.0, 2.0 ** 20])
def test_route_of_groups_whose_biases_cancel(gpu, score, E, groups, most):
    """Runs that count their two highest, one far above and one far below zero: 32 bits round each by more than the counts differ,
    2^-18 of a logit a step, which is far more than 64 bits lose."""
    lh = gpu
    announce(f"route groups with biases of {most} and {-most}, {score} {groups} runs")
    rng = np.random.default_rng(21)
    T, size = 120, E // groups
    x = np.full((T, groups, size), -3.0)
    x[:, :, :2] = 0.3
    steps = rng.integers(0, 64, (T, groups))
    x[:, :, 0] += steps * 2.0 ** -18
    x[:, :, 1] += (np.argsort(rng.random((T, groups)), axis=1) + 64 - steps) * 2.0 ** -18
    x = x.reshape(T, E).astype(np.float32)
    bias = np.full((groups, size), -2 * most, np.float32)
    bias[:, 0], bias[:, 1] = most, -most
    bias = bias.ravel()
    r = lh.MoeRouter(E, 2, score, up(lh, bias), groups, 2, 2)
    check_route(route(lh, x, "f32", r), x, "f32", 2, score=score, bias=bias, groups=groups, top_groups=2, group_best=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,E,k,groups,top", [("f32", 40, 8, 1, 1), ("bf16", 40, 8, 5, 2), ("f16", 300, 9, 1, 1)])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_of_masked_and_bad_logits(gpu, score, dtype, E, k, groups, top, renorm):
    lh = gpu
    announce(f"route masks {score} {dtype} {E}")
    rng = np.random.default_rng(6)
    x = rng.standard_normal((70, E))
    x[1] = -np.inf                      # nothing left
    x[2, 1:] = -np.inf                  # one left
    x[3, rng.random(E) < 0.7] = -np.inf
    x[4, 5] = np.nan
    x[5, E - 1] = np.inf
    x[6, ::2] = -np.inf
    x[7] = np.finfo(np.float32).min if dtype != "f16" else -65504.0    # the type's lowest value is no mask
    x[8, 3:] = -80.0                    # scores below the least float
    x[9] = -np.linspace(90, 300, E)
    x[66, 0] = -np.inf
    store = ref.to_store(x, dtype)
    for bias in (None, np.where(np.arange(E) % 5 == 1, -np.inf, 0.1).astype(np.float32)):
        B = up(lh, bias) if bias is not None else None
        r = lh.MoeRouter(E, k, score, B, groups, top, 1, renorm)
        check_route(route(lh, store, dtype, r), store, dtype, k, score=score, bias=bias, groups=groups, top_groups=top,
                    renormalize=renorm)


def test_route_without_a_plan_and_of_bad_biases(gpu):
    lh = gpu
    announce("route bad biases")
    x = np.random.default_rng(7).standard_normal((9, 16)).astype(np.float32)
    r = lh.MoeRouter(16, 3)
    check_route(route(lh, x, "f32", r, with_plan=False), x, "f32", 3, score="softmax")
    for value in (np.nan, np.inf):
        bias = np.zeros(16, np.float32)
        bias[4] = value
        B = up(lh, bias)
        ids, w, p = route(lh, x, "f32", lh.MoeRouter(16, 3, bias=B))
        assert (ids == -1).all() and np.isnan(w).all()
        assert not p.offsets.to_numpy().any() and (p.order.to_numpy() == -1).all()


# ---- plans of given ids ------------------------------------------------------------------------

@pytest.mark.parametrize("T,E,k", [(0, 5, 3), (1, 1, 1), (1, 1024, 32), (7, 3, 2), (63, 60, 4), (64, 64, 8), (65, 64, 8), (700, 17, 5),
                                   (1024, 256, 8), (5003, 60, 4), (16385, 128, 6), (40000, 9, 3)])
def test_sort(gpu, T, E, k):
    lh = gpu
    announce(f"sort {T} tokens, {k} of {E}")
    rng = np.random.default_rng(T + E)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < 0.1] = -1
    if T > 5:
        ids[3] = E            # no expert either
        ids[4] = 2 ** 31 - 1
        ids[5] = -2 ** 31
        ids[T // 2:T // 2 + 3] = 0
    I, p = up(lh, ids), lh.MoePlan(T, E, k)
    for a in (p.offsets, p.order, p.workspace):
        a.fill_bytes(FILL)
    for _ in range(2):
        lh.moe_sort(p, I)
        lh.synchronize()
        offsets, order = ref.plan(ids, E)
        np.testing.assert_array_equal(p.offsets.to_numpy(), offsets)
        np.testing.assert_array_equal(p.order.to_numpy(), order)


# ---- the experts' layers -----------------------------------------------------------------------

def experts_case(rng, T, E, k, N, K, masked=0.1, favourite=False):
    ids = np.argsort(rng.random((T, E)), axis=1)[:, :k].astype(np.int32)
    if favourite:
        ids[:] = np.arange(k)          # the rest of the experts have no row
    ids[rng.random((T, k)) < masked] = -1
    x, xs, _, _, _ = make(rng, T * k, 1, K)
    w = rng.integers(-127, 128, (E, N, K)).astype(np.int8)
    ws = ((rng.random((E, N)) + 0.5) / (70 * np.sqrt(K + 1.0))).astype(np.float32)
    return ids, x, xs, w, ws, (rng.standard_normal((E, N)) * 0.3).astype(np.float32)


def run_experts(lh, ids, x, xs, w, ws, bias, act, gated, dtype, x_sorted, y_sorted, pad=(0, 0, 0), offsets=None, order=None):
    """Y (T * k, columns) for x of T or T * k rows; rows that no assignment has must stay."""
    (T, k), (E, N, K) = ids.shape, w.shape
    cols = N // 2 if gated else N
    if offsets is None:
        offsets, order = ref.plan(ids, E)

    def rows(a, extra):
        out = np.full(a.shape[:-1] + (K + extra,), 77, np.int8)
        out[..., :K] = a
        return up(lh, np.concatenate((out.ravel(), np.full(32, 99, np.int8))))

    X, W, Y = rows(x, pad[0]), rows(w, pad[1]), blank(lh, dtype, T * k, cols + pad[2])
    XS, WS, B = up(lh, xs), up(lh, ws), up(lh, bias) if bias is not None else None
    O, R = up(lh, offsets), up(lh, order)
    layer = lh.w8_layer_raw(W.ptr, WS.ptr, N, K, K + pad[1], bias=B.ptr if B is not None else 0, act=act, gated=gated, experts=E,
                            expert_stride=N * (K + pad[1]))
    lh.experts_w8a8_raw(lh.moe_plan_raw(T, E, k, O.ptr, R.ptr), layer, X.ptr, XS.ptr, K + pad[0], dtype, Y.ptr, cols + pad[2],
                        x_sorted=x_sorted, y_sorted=y_sorted)
    lh.synchronize()
    got = Y.to_numpy().T
    assert untouched(got[:, cols:])
    return got[:, :cols]


def check_experts(got, ids, x, xs, w, ws, bias, act, gated, dtype, x_sorted, y_sorted):
    (T, k), E = ids.shape, w.shape[0]
    offsets, order = ref.plan(ids, E)
    written = np.zeros(T * k, bool)
    for e in range(E):
        at = np.arange(offsets[e], offsets[e + 1])
        if not at.size:
            continue
        src = at if x_sorted else order[at] // k
        dst = at if y_sorted else order[at]
        written[dst] = True
        check(got[dst], ref.layer(x[src], xs[src], w[e], ws[e], bias[e] if bias is not None else None, act, gated, dtype), dtype)
    assert untouched(got[~written])


EXPERTS = [  # T, E, k, N, K
    (1, 1, 1, 16, 16), (1, 8, 2, 64, 128), (1, 64, 8, 128, 256), (3, 5, 2, 30, 33), (16, 4, 1, 96, 64), (20, 60, 4, 66, 208), (64, 64, 8, 64, 80),
    (70, 3, 2, 130, 272), (100, 7, 3, 258, 144), (300, 4, 2, 256, 128), (520, 2, 2, 384, 320), (257, 130, 6, 40, 64)]


@pytest.mark.parametrize("sorted_", [(False, True), (True, False), (False, False), (True, True)])
@pytest.mark.parametrize("i", range(len(EXPERTS)))
def test_experts(gpu, choice, i, sorted_):  # noqa: F811
    lh = gpu
    T, E, k, N, K = EXPERTS[i]
    (act, gated), dtype = KINDS[(i + 2 * sorted_[0] + 3 * sorted_[1]) % len(KINDS)], DTYPES[(i + sorted_[0]) % 3]
    announce(f"experts {EXPERTS[i]} {act} gated={gated} {dtype} sorted={sorted_} choice {choice}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(300 + i), T, E, k, N, K, favourite=i % 4 == 2)
    if not sorted_[0]:
        x, xs = x[:T], xs[:T]
    b = bias if i % 2 else None
    args = (ids, x, xs, w, ws, b, act, gated, dtype, *sorted_)
    check_experts(run_experts(lh, *args), *args)


@pytest.mark.parametrize("K", [65, 80])
@pytest.mark.parametrize("sorted_", [(False, True), (True, False)])
def test_experts_of_many_tiles(gpu, K, sorted_):
    lh = gpu
    announce(f"experts of many tiles, K = {K}, sorted={sorted_}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(20), 2000, 4, 2, 1100, K)
    if not sorted_[0]:
        x, xs = x[:2000], xs[:2000]
    args = (ids, x, xs, w, ws, bias, "silu", True, "bf16", *sorted_)
    for c in (0, 1):
        lh.set_kernel_override(lh.FAMILY_W8A8, c)
        try:
            got = run_experts(lh, *args)
        finally:
            lh.set_kernel_override(lh.FAMILY_W8A8, 0)
        check_experts(got, *args)


@pytest.mark.parametrize("pad", [(16, 32, 4), (1, 0, 1), (0, 3, 0)])
def test_experts_strides(gpu, choice, pad):  # noqa: F811
    lh = gpu
    announce(f"experts, rows {pad} longer, choice {choice}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(17), 90, 6, 2, 70, 160)
    args = (ids, x[:90], xs[:90], w, ws, bias, "silu", True, "bf16", False, False)
    check_experts(run_experts(lh, *args, pad=pad), *args)


def test_experts_without_tokens_of_their_own(gpu, choice):  # noqa: F811
    """All assignments masked: nothing is written; and all to the last expert."""
    lh = gpu
    announce(f"experts with none, choice {choice}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(18), 20, 9, 2, 64, 128)
    ids[:] = -1
    args = (ids, x, xs, w, ws, bias, "none", False, "f16", True, True)
    check_experts(run_experts(lh, *args), *args)
    ids[:, 1] = 8
    check_experts(run_experts(lh, *args), *args)


@pytest.mark.parametrize("sorted_", [(False, True), (True, False)])
def test_experts_of_a_bad_plan_stay_inside(gpu, choice, sorted_):  # noqa: F811
    """Offsets and entries of the plan that are none: what they name is left out, the rest stands."""
    lh = gpu
    announce(f"experts bad plan {sorted_} choice {choice}")
    T, E, k, N, K = 40, 6, 2, 64, 128
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(19), T, E, k, N, K, masked=0.0)
    if not sorted_[0]:
        x, xs = x[:T], xs[:T]
    offsets, order = ref.plan(ids, E)
    bad_order = order.copy()
    out = [0, 7, T * k - 1]
    bad_order[out] = [-1, T * k, -2 ** 31]
    args = (ids, x, xs, w, ws, bias, "none", False, "f32", *sorted_)
    got = run_experts(lh, *args, offsets=offsets, order=bad_order)
    full = run_experts(lh, *args)
    lost = np.zeros(T * k, bool)
    lost[out if sorted_[1] else order[out]] = True
    assert untouched(got[lost])
    np.testing.assert_array_equal(got[~lost], full[~lost])
    for o in (np.array([0, -5, 2 ** 31 - 1, 10, -2 ** 31, 3, 2 ** 31 - 1]), np.full(E + 1, 2 ** 31 - 1), np.full(E + 1, -1)):
        run_experts(lh, *args, offsets=o.astype(np.int32), order=order)   # stays inside its buffers, writes what it will


# ---- the weighted sum --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,N,pad", [(1, 1, 1, 0), (1, 8, 64, 0), (3, 2, 7, 1), (5, 10, 1000, 0), (64, 8, 2048, 8), (130, 6, 1026, 0),
                                       (9, 0, 40, 0), (2, 32, 5000, 4)])
@pytest.mark.parametrize("base", ["none", "own", "in place"])
def test_combine(gpu, dtype, T, k, N, pad, base):
    lh = gpu
    announce(f"combine {dtype} {T} x {k} x {N} base {base}")
    rng = np.random.default_rng(T * 31 + N)
    y, b = (ref.to_store(rng.standard_normal(s), dtype) for s in ((T * k, N + pad), (T, N + pad)))
    ids = rng.integers(0, 9, (T, k)).astype(np.int32)
    dead = rng.random((T, k)) < 0.2
    ids[dead] = -1
    nan = {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "bf16": np.uint16(0x7FC0)}[dtype]
    y[dead.ravel()] = nan                            # rows that are not read
    w = rng.random((T, k)).astype(np.float32)
    Y, I, W, B, O = up(lh, y) if k else None, up(lh, ids) if k else None, up(lh, w) if k else None, up(lh, b), blank(lh, dtype, T, N + pad)
    if base == "in place":
        O = B
    lh.moe_combine_raw(dtype, Y.ptr if k else 0, N + pad, I.ptr if k else 0, W.ptr if k else 0, T, k, N, O.ptr, N + pad,
                       base=0 if base == "none" else B.ptr, ldb=N + pad)
    lh.synchronize()
    got = O.to_numpy().T
    assert untouched(got[:, N:]) if base != "in place" else (got[:, N:] == b[:, N:]).all()
    yf = np.where(dead.reshape(T, k, 1), 0.0, ref.to_float(y, dtype).reshape(T, k, N + pad)[:, :, :N])
    check(got[:, :N], ref.combine(yf, w.astype(np.float64), ids, None if base == "none" else ref.to_float(b, dtype)[:, :N], dtype), dtype)


def test_combine_shows_weights_that_are_nan(gpu):
    lh = gpu
    announce("combine NaN weights")
    y, w, ids = np.ones((6, 8), np.float32), np.full((3, 2), 0.5, np.float32), np.zeros((3, 2), np.int32)
    w[1], ids[1] = np.nan, -1
    O = blank(lh, "f32", 3, 8)
    lh.moe_combine(O, up(lh, y), up(lh, w), up(lh, ids))
    lh.synchronize()
    got = O.to_numpy().T
    assert np.isnan(got[1]).all() and (got[[0, 2]] == 1).all()


# ---- a whole layer -----------------------------------------------------------------------------

class Block:
    """A feed-forward layer of experts as a program runs it: routed, quantised, gate and up, quantised, down, summed."""

    def __init__(self, lh, rng, T, E, k, D, F):
        self.lh, self.shape = lh, (T, E, k, D, F)
        self.w1, self.w2 = (rng.integers(-127, 128, s).astype(np.int8) for s in ((E, 2 * F, D), (E, D, F)))
        self.s1, self.s2 = ((rng.random((E, n)) * 1e-3 + 5e-4).astype(np.float32) for n in (2 * F, D))
        self.bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
        self.W = [up(lh, a) for a in (self.w1, self.s1, self.w2, self.s2, self.bias)]
        self.gate_up, self.down = lh.W8Layer(self.W[0], self.W[1], act="silu", gated=True), lh.W8Layer(self.W[2], self.W[3])
        self.router = lh.MoeRouter(E, k, "sigmoid", self.W[4])
        self.plan = lh.MoePlan(T, E, k)
        new = lh.HIPDeviceArray
        self.x, self.logits = new("bf16", (D, T)), new("f32", (E, T))
        self.ids, self.weights = new("i32", (k, T)), new("f32", (k, T))
        self.q, self.qs, self.h = new("i8", (D, T)), new("f32", (T,)), new("bf16", (F, T * k))
        self.hq, self.hs, self.y, self.out = new("i8", (F, T * k)), new("f32", (T * k,)), new("bf16", (D, T * k)), new("bf16", (D, T))

    def set(self, x, logits):
        self.x.copy_from(ref.to_store(x, "bf16").T)
        self.logits.copy_from(logits.T)

    def run(self, stream=None):
        lh = self.lh
        lh.moe_route(self.ids, self.weights, self.router, self.logits, self.plan, stream=stream)
        lh.quantize_i8(self.q, self.qs, self.x, stream=stream)
        lh.experts_w8a8(self.h, self.plan, self.gate_up, self.q, self.qs, y_sorted=True, stream=stream)
        lh.quantize_i8(self.hq, self.hs, self.h, stream=stream)
        lh.experts_w8a8(self.y, self.plan, self.down, self.hq, self.hs, x_sorted=True, stream=stream)
        lh.moe_combine(self.out, self.y, self.weights, self.ids, base=self.x, stream=stream)

    def want(self, x, logits):
        """The layer in float64 from the rounded tokens, nothing quantised, and what quantising may move."""
        T, E, k, D, F = self.shape
        xf = ref.to_float(ref.to_store(x, "bf16"), "bf16")
        ids, w = ref.route(logits.astype(np.float64), k, "sigmoid", self.bias)
        out, slack = xf.copy(), np.zeros((T, D))
        for t in range(T):
            step = np.abs(xf[t]).max() / 127 / 2
            for j, e in enumerate(ids[t]):
                w1, w2 = self.w1[e] * self.s1[e][:, None].astype(np.float64), self.w2[e] * self.s2[e][:, None].astype(np.float64)
                z = w1 @ xf[t]
                dz = np.abs(w1).sum(1) * step
                g, u = z[:F], z[F:]
                h = ref.act("silu", g) * u
                dh = 1.13 * dz[:F] * (np.abs(u) + dz[F:]) + np.abs(ref.act("silu", g)) * dz[F:] + np.abs(h) * 2.0 ** -7
                dh += (np.abs(h) + dh).max() / 127 / 2
                out[t] += w[t, j] * (w2 @ h)
                slack[t] += w[t, j] * (np.abs(w2) @ dh + np.abs(w2 @ h) * 2.0 ** -7)
        return out, slack + np.abs(out) * 2.0 ** -7


@pytest.mark.parametrize("T,E,k,D,F", [(1, 8, 2, 64, 32), (37, 16, 4, 128, 96), (130, 5, 3, 80, 64)])
def test_a_layer_of_experts(gpu, T, E, k, D, F):
    lh = gpu
    announce(f"a layer of experts {T} tokens, {k} of {E}, {D} x {F}")
    rng = np.random.default_rng(T)
    b = Block(lh, rng, T, E, k, D, F)
    x, logits = rng.standard_normal((T, D)), rng.standard_normal((T, E)).astype(np.float32)
    b.set(x, logits)
    b.run()
    lh.synchronize()
    out, slack = b.want(x, logits)
    off = np.abs(ref.to_float(b.out.to_numpy().T, "bf16") - out)
    assert (off <= slack).all(), f"{(off / slack).max()} of what quantising may move"
    # and exactly what the parts, each checked above, give: nothing depends on who ran before
    first = b.out.to_numpy()
    b.run()
    lh.synchronize()
    np.testing.assert_array_equal(b.out.to_numpy(), first)


@pytest.mark.parametrize("T", [1, 3, 200])
def test_a_captured_layer_of_experts(gpu, T):
    """Captured on a fresh stream without an eager call first (no call allocates), replayed on new tokens with eager work of
    another layer between the replays."""
    lh = gpu
    announce(f"a captured layer of experts, {T} tokens")
    rng = np.random.default_rng(T)
    a, b = Block(lh, rng, T, 12, 3, 64, 48), Block(lh, rng, T, 12, 3, 64, 48)
    for block in (a, b):
        block.set(rng.standard_normal((T, 64)), rng.standard_normal((T, 12)).astype(np.float32))
    lh.synchronize()
    st = lh.Stream()
    g = lh.Graph(st)
    with g.capture():
        a.run(st.handle)
    for _ in range(4):
        x, logits = rng.standard_normal((T, 64)), rng.standard_normal((T, 12)).astype(np.float32)
        a.set(x, logits)
        a.out.fill_bytes(FILL)
        lh.synchronize()
        g.launch()
        b.run()
        st.synchronize()
        got = a.out.to_numpy()
        a.out.fill_bytes(FILL)
        lh.synchronize()
        a.run()
        lh.synchronize()
        np.testing.assert_array_equal(got, a.out.to_numpy())
        out, slack = a.want(x, logits)
        assert (np.abs(ref.to_float(got.T, "bf16") - out) <= slack).all()
    g.close()
    st.close()


def test_two_layers_of_experts_at_once(gpu):
    """On two streams, each with a plan of its own: the bits of one behind the other."""
    lh = gpu
    announce("two layers of experts at once")
    rng = np.random.default_rng(31)
    blocks = [Block(lh, rng, T, 16, 4, 256, 128) for T in (300, 170)]
    streams = [lh.Stream() for _ in blocks]
    for b in blocks:
        T, E, _, D, _ = b.shape
        b.set(rng.standard_normal((T, D)), rng.standard_normal((T, E)).astype(np.float32))
    want = []
    for b in blocks:
        b.run()
        lh.synchronize()
        want.append(b.out.to_numpy())
        b.out.fill_bytes(FILL)
    lh.synchronize()
    for _ in range(10):
        for b, st in zip(blocks, streams):
            b.run(st.handle)
    for b, st, w in zip(blocks, streams, want):
        st.synchronize()
        np.testing.assert_array_equal(b.out.to_numpy(), w)
        st.close()


@pytest.mark.parametrize("T,E,k", [(16500, 16, 4), (33000, 130, 2), (66000, 7, 2)])
def test_route_of_more_tokens_than_a_workgroup_has_at_once(gpu, T, E, k):
    """Workgroups of 128, 192 and 320 tokens."""
    lh = gpu
    announce(f"route {T} tokens, {k} of {E}")
    x = np.random.default_rng(32).standard_normal((T, E)).astype(np.float32)
    check_route(route(lh, x, "f32", lh.MoeRouter(E, k, "sigmoid")), x, "f32", k, score="sigmoid")


# ---- sizes past 32 bits ------------------------------------------------------------------------

def put(lh, a, at, b):
    b = np.ascontiguousarray(b)
    lh._lib.call("lava_hip_memcpy_h2d", a.ptr + at, b.ctypes.data, b.nbytes)


@pytest.mark.parametrize("x_sorted", [False, True])
def test_experts_whose_tokens_and_weights_pass_32_bits(gpu, choice, x_sorted):  # noqa: F811
    """Rows 65536 bytes apart: the last token and the second expert lie 2 GiB behind the first."""
    lh = gpu
    announce(f"experts past 2 GiB, x_sorted={x_sorted}, choice {choice}")
    T, N, K, ld, stride = 32790, 40, 128, 65536, 2 ** 31 + 65536
    rng = np.random.default_rng(33)
    seen = [0, 1, 70, T - 2, T - 1]
    x, w = rng.integers(-127, 128, (len(seen), K)).astype(np.int8), rng.integers(-127, 128, (2, N, K)).astype(np.int8)
    X, W = lh.HIPDeviceArray("i8", (ld * T,)), lh.HIPDeviceArray("i8", (stride + N * ld,))
    Y = blank(lh, "f32", T, N)
    ids = np.full((T, 1), -1, np.int32)
    ids[seen, 0] = [0, 1, 1, 0, 1]
    offsets, order = ref.plan(ids, 2)
    at = [int(np.flatnonzero(order == t)[0]) if x_sorted else t for t in seen]
    if x_sorted:      # the plan's rows moved to the end, so that they lie far from X
        order = np.concatenate((np.full(T - 5, -1), order[:5])).astype(np.int32)
        offsets = np.array([T - 5, T - 3, T], np.int32)
        at = [T - 5 + a for a in at]
    for a, row in zip(at, x):
        put(lh, X, a * ld, row)
    for e in range(2):
        for n in range(N):
            put(lh, W, e * stride + n * ld, w[e, n])
    XS, WS, O, R = up(lh, np.ones(T, np.float32)), up(lh, np.ones((2, N), np.float32)), up(lh, offsets), up(lh, order)
    layer = lh.w8_layer_raw(W.ptr, WS.ptr, N, K, ld, experts=2, expert_stride=stride)
    try:
        lh.experts_w8a8_raw(lh.moe_plan_raw(T, 2, 1, O.ptr, R.ptr), layer, X.ptr, XS.ptr, ld, "f32", Y.ptr, N, x_sorted=x_sorted)
        lh.synchronize()
        got = Y.to_numpy().T
    finally:
        for a in (X, W, Y):
            a.close()
    for i, t in enumerate(seen):
        np.testing.assert_array_equal(got[t], w[ids[t, 0]].astype(np.float64) @ x[i].astype(np.float64))
    assert untouched(np.delete(got, seen, 0))
