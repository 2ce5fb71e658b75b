"""What the layers with 8-bit weights, the routing and the experts refuse, on the host: every call here fails, or has nothing
to do, before a device is touched."""
import ctypes as C

import numpy as np
import pytest

import lava_hip as lh
import w8a8_reference as ref

A = 1 << 20   # a 16-byte aligned address that nothing reads


def layer(**kw):
    d = dict(w=A, scale=A, n=64, k=128, ldw=128)
    d.update(kw)
    return lh.w8_layer_raw(**d)


def linear(l=None, X=A, xs=A, tokens=5, ldx=128, dtype="f16", Y=A, ldy=64):
    lh.w8a8_raw(l or layer(), X, xs, tokens, ldx, dtype, Y, ldy)


def plan(**kw):
    d = dict(tokens=5, experts=4, top_k=2, offsets=A, order=A)
    d.update(kw)
    return lh.moe_plan_raw(**d)


def experts(p=None, l=None, X=A, xs=A, ldx=128, dtype="f16", Y=A, ldy=64, **kw):
    lh.experts_w8a8_raw(p or plan(), l or layer(experts=4, expert_stride=64 * 128), X, xs, ldx, dtype, Y, ldy, **kw)


def router(**kw):
    d = dict(experts=8, top_k=2)
    d.update(kw)
    return lh.moe_router_raw(**d)


def route(r=None, dtype="f32", logits=A, ldl=8, tokens=5, ids=A, weights=A, plan=None):
    lh.moe_route_raw(r or router(), dtype, logits, ldl, tokens, ids, weights, plan)


@pytest.mark.parametrize("change,words", [
    (dict(k=-1), "negative"), (dict(tokens=-1), "negative"), (dict(X=0), "null"), (dict(Q=0), "null"), (dict(scale=0), "null"),
    (dict(ldx=63), "ldx"), (dict(ldq=63), "ldq"), (dict(X=A + 1), "aligned"), (dict(scale=A + 2), "aligned")])
def test_quantisations_that_are_refused(change, words):
    d = dict(dtype="f16", X=A, Q=A, scale=A, k=64, tokens=3, ldx=64, ldq=64)
    d.update(change)
    with pytest.raises(lh.InvalidArgument, match=words):
        lh.quantize_i8_raw(**d)


BAD_LAYERS = {
    "negative n": (dict(n=-1), "negative"), "negative k": (dict(k=-1), "negative"), "no weights": (dict(w=0), "null"),
    "no scales": (dict(scale=0), "null"), "short rows": (dict(ldw=127), "ldw"), "odd scales": (dict(scale=A + 2), "aligned"),
    "odd bias": (dict(bias=A + 1), "aligned"), "odd gated": (dict(n=63, gated=True), "odd number"),
}


@pytest.mark.parametrize("name", list(BAD_LAYERS))
def test_layers_that_are_refused(name):
    change, words = BAD_LAYERS[name]
    with pytest.raises(lh.InvalidArgument, match=words):
        linear(layer(**change))
    with pytest.raises(lh.InvalidArgument, match=words):
        experts(l=layer(**dict(dict(experts=4, expert_stride=64 * 128), **change)))


@pytest.mark.parametrize("change,words", [
    (dict(X=0), "null"), (dict(xs=0), "null"), (dict(Y=0), "null"), (dict(tokens=-1), "negative"), (dict(ldx=127), "ldx"),
    (dict(ldy=63), "ldy"), (dict(xs=A + 1), "aligned"), (dict(Y=A + 1), "aligned"), (dict(dtype="f32", Y=A + 2), "aligned"),
    (dict(l=layer(experts=2, expert_stride=64 * 128)), "2 experts")])
def test_linear_arguments_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        linear(**change)


def test_layers_that_are_not_supported():
    with pytest.raises(lh.Unsupported, match="131071"):
        linear(layer(k=131072, ldw=131072), ldx=131072)
    with pytest.raises(lh.Unsupported, match="too large"):
        linear(layer(n=2 ** 31), ldy=2 ** 31)
    with pytest.raises(lh.Unsupported, match="too many"):
        linear(tokens=2 ** 31)
    with pytest.raises(lh.Unsupported, match="f32, f16 or bf16"):
        linear(dtype="i32")
    with pytest.raises(ValueError, match="act"):
        layer(act="swish")
    with pytest.raises(ValueError, match="64 bits"):
        layer(n=2 ** 63)
    with pytest.raises(ValueError, match="32 bits"):
        layer(experts=2 ** 32 + 1)


@pytest.mark.parametrize("change,words", [
    (dict(p=plan(tokens=-1)), "negative"), (dict(p=plan(experts=0)), "0 experts"), (dict(p=plan(top_k=0)), "plan of 0"),
    (dict(p=plan(offsets=0)), "null"), (dict(p=plan(order=0)), "null"), (dict(p=plan(order=A + 2)), "misaligned"),
    (dict(p=plan(experts=5)), "a plan of 5"), (dict(l=layer(experts=4, expert_stride=64 * 128 - 1)), "expert_stride"),
    (dict(l=layer(experts=4, expert_stride=-64 * 128)), "expert_stride"), (dict(X=0), "null"), (dict(Y=0), "null"),
    (dict(ldx=127), "ldx"), (dict(ldy=63), "ldy")])
def test_experts_arguments_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        experts(**change)


def test_plans_that_are_not_supported():
    for change in (dict(experts=1025), dict(top_k=33), dict(tokens=2 ** 30)):
        with pytest.raises(lh.Unsupported):
            experts(p=plan(**change))
        with pytest.raises(lh.Unsupported):
            lh.moe_sort_raw(A, plan(**change))


@pytest.mark.parametrize("change,words", [
    (dict(experts=0), "0 experts"), (dict(top_k=0), "0 of"), (dict(top_k=9), "top_k"), (dict(groups=3, top_groups=1), "groups"),
    (dict(groups=0, top_groups=0), "groups"), (dict(groups=2, top_groups=3), "top_groups"), (dict(groups=2, top_groups=0), "top_groups"),
    (dict(group_best=3), "group_best"), (dict(group_best=0), "group_best"), (dict(groups=8, top_groups=8, group_best=2), "group_best"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(bias=A + 1), "misaligned")])
def test_routers_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        route(router(**change))


def test_routers_that_are_not_supported():
    with pytest.raises(lh.Unsupported, match="1024"):
        route(router(experts=1025), ldl=1025)
    with pytest.raises(lh.Unsupported, match="32"):
        route(router(experts=64, top_k=33), ldl=64)
    with pytest.raises(lh.Unsupported, match="groups"):
        route(router(experts=130, groups=65, top_groups=2), ldl=130)
    with pytest.raises(ValueError, match="score"):
        router(score="tanh")


@pytest.mark.parametrize("change,words", [
    (dict(logits=0), "null"), (dict(ids=0), "null"), (dict(weights=0), "null"), (dict(tokens=-1), "negative"),
    (dict(ldl=7), "ldl"), (dict(logits=A + 2), "aligned"), (dict(ids=A + 1), "aligned"), (dict(weights=A + 2), "aligned"),
    (dict(plan=plan(experts=8, tokens=6)), "a plan of 6"), (dict(plan=plan(experts=4)), "a plan of 5"),
    (dict(plan=plan(experts=8, top_k=3)), "a plan of 5"), (dict(plan=plan(experts=8, offsets=0)), "null")])
def test_route_arguments_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        route(**change)


def test_plans_whose_workspace_is_too_small():
    n = lh.moe_plan_workspace_bytes(5000, 8, 2)
    assert n > 0
    for p in (plan(tokens=5000, experts=8), plan(tokens=5000, experts=8, workspace=A, workspace_bytes=n - 1)):
        with pytest.raises(lh.InvalidArgument, match="workspace"):
            lh.moe_sort_raw(A, p)
        with pytest.raises(lh.InvalidArgument, match="workspace"):
            route(tokens=5000, plan=p)
    with pytest.raises(lh.InvalidArgument, match="misaligned"):
        lh.moe_sort_raw(A, plan(tokens=5000, experts=8, workspace=A + 2, workspace_bytes=n))
    with pytest.raises(lh.InvalidArgument, match="null ids"):
        lh.moe_sort_raw(0, plan())


def test_workspace_bytes():
    assert lh.moe_plan_workspace_bytes(0, 1024, 32) == 0 and lh.moe_plan_workspace_bytes(1, 8, 2) == 0
    assert lh.moe_plan_workspace_bytes(1 << 20, 1024, 32) <= 1 << 20   # it does not grow with the tokens for ever
    with pytest.raises(lh.InvalidArgument, match="null"):
        lh._lib.call("lava_hip_moe_plan_workspace_bytes", 5, 8, 2, None)


@pytest.mark.parametrize("change,words", [
    (dict(tokens=-1), "negative"), (dict(n=-1), "negative"), (dict(top_k=-1), "negative"), (dict(Y=0), "null"),
    (dict(weights=0), "null"), (dict(out=0), "null"), (dict(ldy=63), "stride"), (dict(ldo=63), "stride"),
    (dict(base=A, ldb=63), "stride"), (dict(Y=A + 1), "aligned"), (dict(ids=A + 2), "aligned"),
    (dict(base=2 * A, out=2 * A, ldb=128), "another stride")])
def test_combine_arguments_that_are_refused(change, words):
    d = dict(dtype="bf16", Y=A, ldy=64, ids=A, weights=A, tokens=5, top_k=2, n=64, out=A, ldo=64)
    d.update(change)
    with pytest.raises(lh.InvalidArgument, match=words):
        lh.moe_combine_raw(**d)


def test_null_descriptors_are_refused():
    call = lh._lib.call
    with pytest.raises(lh.InvalidArgument, match="null layer"):
        call("lava_hip_gemm_w8a8", None, A, A, 5, 128, 0, A, 64, None)
    with pytest.raises(lh.InvalidArgument, match="null plan"):
        call("lava_hip_experts_w8a8", None, C.byref(layer()), A, A, 128, 0, A, 64, 0, None)
    with pytest.raises(lh.InvalidArgument, match="null layer"):
        call("lava_hip_experts_w8a8", C.byref(plan()), None, A, A, 128, 0, A, 64, 0, None)
    with pytest.raises(lh.InvalidArgument, match="flags"):
        call("lava_hip_experts_w8a8", C.byref(plan()), C.byref(layer(experts=4, expert_stride=8192)), A, A, 128, 0, A, 64, 4, None)
    with pytest.raises(lh.InvalidArgument, match="null router"):
        call("lava_hip_moe_route", None, 0, A, 8, 5, A, A, None, None)
    with pytest.raises(lh.InvalidArgument, match="null plan"):
        call("lava_hip_moe_sort", A, None, None)


def test_calls_with_nothing_to_do():
    """No tokens or no channels: nothing is read, pointers may be null."""
    linear(tokens=0, X=0, xs=0, Y=0)
    linear(layer(n=0, w=0, scale=0), X=0, xs=0, Y=0)
    experts(p=plan(tokens=0, offsets=0, order=0), X=0, xs=0, Y=0)
    route(tokens=0, logits=0, ids=0, weights=0)
    lh.quantize_i8_raw("f32", 0, 0, 0, 64, 0, 64, 64)
    lh.moe_combine_raw("f32", 0, 64, 0, 0, 0, 2, 64, 0, 64)
    lh.moe_combine_raw("f32", 0, 0, 0, 0, 5, 2, 0, 0, 0)


def test_descriptors_have_the_header_s_layout():
    L = lh._lib
    assert C.sizeof(L.W8LayerDesc) == 72 and L.W8LayerDesc.n.offset == 24 and L.W8LayerDesc.experts.offset == 56
    assert C.sizeof(L.MoeRouterDesc) == 40 and L.MoeRouterDesc.scale.offset == 28 and L.MoeRouterDesc.bias.offset == 32
    assert C.sizeof(L.MoePlanDesc) == 48 and L.MoePlanDesc.offsets.offset == 16 and L.MoePlanDesc.workspace_bytes.offset == 40


# ---- the reference itself, and the mistakes that the tests have to see --------------------------

def test_the_reference_quantises_borders_to_even():
    x = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5]])
    q, s = ref.quantize(x)
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, 126]] and s[0] == 1.0


def test_the_reference_sees_a_lost_scale_and_a_swapped_gate():
    rng = np.random.default_rng(0)
    x, w = rng.integers(-127, 128, (3, 40)).astype(np.int8), rng.integers(-127, 128, (8, 40)).astype(np.int8)
    xs, ws = np.float32([0.01, 0.02, 0.03]), np.linspace(0.001, 0.002, 8).astype(np.float32)
    y, err = ref.layer(x, xs, w, ws, None, "silu", True, "f32")
    swapped, _ = ref.layer(x, xs, np.roll(w, 4, 0), np.roll(ws, 4), None, "silu", True, "f32")
    lost, _ = ref.layer(x, xs[[0, 0, 0]], w, ws, None, "silu", True, "f32")
    assert (np.abs(swapped - y) > 100 * err).any() and (np.abs(lost - y) > 100 * err).any()


def test_the_reference_routes_as_written():
    x = np.array([[1.0, 3.0, 3.0, -np.inf, 2.0, 0.0]])
    ids, w = ref.route(x, 2, "softmax")
    assert ids.tolist() == [[1, 2]] and np.allclose(w, 0.5)
    ids, _ = ref.route(x, 2, "sigmoid", groups=3, top_groups=1, group_best=2)   # (1, 3), (3, masked), (2, 0)
    assert ids.tolist() == [[1, 0]]
    ids, _ = ref.route(x, 2, "sigmoid", bias=np.float32([9, 0, 0, 9, 0, 0]))
    assert ids.tolist() == [[0, 1]]
    ids, w = ref.route(np.full((1, 4), -np.inf), 2, "softmax")
    assert ids.tolist() == [[-1, -1]] and not w.any()


def test_the_last_tiles_rows_and_channels_are_counted_in_32_bits():
    """A tile begun at 2^31 - 256 or behind ends past 2^31."""
    top = 2 ** 31 - 256
    with pytest.raises(lh.Unsupported, match="too large"):
        linear(layer(n=top + 1), ldy=top + 1)
    with pytest.raises(lh.Unsupported, match="too many"):
        linear(tokens=top + 1)
    with pytest.raises(lh.Unsupported, match="too many"):
        lh.moe_plan_workspace_bytes(top // 8 + 1, 64, 8)
    assert lh.moe_plan_workspace_bytes(top // 8, 64, 8) == 256 * 64 * 4
