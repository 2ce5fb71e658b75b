"""Tokens routed to experts, the experts' layers and their weighted sum: `moe_route`, `moe_sort`, `experts_w8a8` and
`moe_combine`, destination-first like the other kernels, over HIPDeviceArrays or raw device addresses.

Arrays keep the order of `w8a8`, the features fastest: logits are an (experts, T) array, the chosen experts and their weights
(top_k, T) ones, an assignment's number is its place in those, token * top_k + rank.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib
from .device import HIPDeviceArray
from .kernels import _DCODE
from .paged import _fits_size
from .w8a8 import W8Layer, _code, _cut, _fits, _matrix, _scales

_SCORES = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}


def moe_router_raw(experts: int, top_k: int, score: str = "softmax", bias: int = 0, groups: int = 1, top_groups: int = 1,
                   group_best: int = 1, renormalize: bool = True, scale: float = 1.0) -> _lib.MoeRouterDesc:
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}")
    _fits(32, experts=experts, top_k=top_k, groups=groups, top_groups=top_groups, group_best=group_best)
    return _lib.MoeRouterDesc(experts, top_k, _SCORES[score], groups, top_groups, group_best, int(bool(renormalize)), scale,
                              bias or None)


def moe_plan_raw(tokens: int, experts: int, top_k: int, offsets: int, order: int, workspace: int = 0,
                 workspace_bytes: int = 0) -> _lib.MoePlanDesc:
    _fits(64, tokens=tokens)
    _fits(32, experts=experts, top_k=top_k)
    _fits_size(workspace_bytes=workspace_bytes)
    return _lib.MoePlanDesc(tokens, experts, top_k, offsets or None, order or None, workspace or None, workspace_bytes)


def moe_plan_workspace_bytes(tokens: int, experts: int, top_k: int) -> int:
    """Bytes of workspace for writing a plan of these sizes."""
    _fits(64, tokens=tokens)
    _fits(32, experts=experts, top_k=top_k)
    n = C.c_size_t()
    _lib.call("lava_hip_moe_plan_workspace_bytes", tokens, experts, top_k, C.byref(n))
    return int(n.value)


def moe_route_raw(router: _lib.MoeRouterDesc, dtype: str, logits: int, ldl: int, tokens: int, ids: int, weights: int,
                  plan: Optional[_lib.MoePlanDesc] = None, stream: Optional[int] = None) -> None:
    if _cut(ldl, tokens):
        _fits(64, ldl=ldl, tokens=tokens)
    _lib.call("lava_hip_moe_route", C.byref(router), _code(dtype), logits or None, ldl, tokens, ids or None, weights or None,
              C.byref(plan) if plan is not None else None, stream)


def moe_sort_raw(ids: int, plan: _lib.MoePlanDesc, stream: Optional[int] = None) -> None:
    _lib.call("lava_hip_moe_sort", ids or None, C.byref(plan), stream)


def experts_w8a8_raw(plan: _lib.MoePlanDesc, layer: _lib.W8LayerDesc, X: int, x_scale: int, ldx: int, y_dtype: str, Y: int,
                     ldy: int, x_sorted: bool = False, y_sorted: bool = False, stream: Optional[int] = None) -> None:
    if _cut(ldx, ldy):
        _fits(64, ldx=ldx, ldy=ldy)
    flags = (_lib.X_SORTED if x_sorted else 0) | (_lib.Y_SORTED if y_sorted else 0)
    _lib.call("lava_hip_experts_w8a8", C.byref(plan), C.byref(layer), X or None, x_scale or None, ldx, _code(y_dtype),
              Y or None, ldy, flags, stream)


def moe_combine_raw(dtype: str, Y: int, ldy: int, ids: int, weights: int, tokens: int, top_k: int, n: int, out: int,
                    ldo: int, base: int = 0, ldb: int = 0, stream: Optional[int] = None) -> None:
    if _cut(ldy, tokens, n, ldo, ldb, top_k << 32):
        _fits(64, ldy=ldy, tokens=tokens, n=n, ldo=ldo, ldb=ldb)
        _fits(32, top_k=top_k)
    _lib.call("lava_hip_moe_combine", _code(dtype), Y or None, ldy, ids or None, weights or None, tokens, top_k, n,
              base or None, ldb, out or None, ldo, stream)


class MoeRouter:
    """How tokens are routed (`lava_hip_moe_router`); bias: f32, one an expert."""

    def __init__(self, experts: int, top_k: int, score: str = "softmax", bias: Optional[HIPDeviceArray] = None,
                 groups: int = 1, top_groups: int = 1, group_best: int = 1, renormalize: bool = True, scale: float = 1.0):
        if bias is not None:
            _scales("bias", bias, experts)
        self.bias, self.experts, self.top_k = bias, experts, top_k
        self.desc = moe_router_raw(experts, top_k, score, bias.ptr if bias is not None else 0, groups, top_groups,
                                   group_best, renormalize, scale)


class MoePlan:
    """The tokens of each expert: i32 device arrays `offsets` (experts + 1) and `order` (tokens * top_k), and the workspace for
    writing them.  Calls that may run at once write plans of their own."""

    def __init__(self, tokens: int, experts: int, top_k: int):
        n = moe_plan_workspace_bytes(tokens, experts, top_k)
        self.tokens, self.experts, self.top_k = tokens, experts, top_k
        self.offsets = HIPDeviceArray("i32", (experts + 1,))
        self.order = HIPDeviceArray("i32", (tokens * top_k,))
        self.workspace = HIPDeviceArray("u8", (n,))
        self.desc = moe_plan_raw(tokens, experts, top_k, self.offsets.ptr, self.order.ptr, self.workspace.ptr, n)

    def close(self) -> None:
        for a in (self.offsets, self.order, self.workspace):
            a.close()


def moe_route(ids: HIPDeviceArray, weights: HIPDeviceArray, router: MoeRouter, logits: HIPDeviceArray,
              plan: Optional[MoePlan] = None, stream: Optional[int] = None) -> HIPDeviceArray:
    """Routes tokens by their logits (experts, T): ids (i32) and weights (f32), (top_k, T), and the plan if one is given."""
    _matrix("logits", logits, tuple(_DCODE), router.experts)
    T = logits.dims[1]
    _matrix("ids", ids, ("i32",), router.top_k, T)
    _matrix("weights", weights, ("f32",), router.top_k, T)
    moe_route_raw(router.desc, logits.dtype, logits.ptr, router.experts, T, ids.ptr, weights.ptr,
                  plan.desc if plan is not None else None, stream)
    return ids


def moe_sort(plan: MoePlan, ids: HIPDeviceArray, stream: Optional[int] = None) -> MoePlan:
    """The plan of given ids (top_k, T); numbers outside [0, experts) are no expert (negative ones, if `moe_combine` gets them too)."""
    _matrix("ids", ids, ("i32",), plan.top_k, plan.tokens)
    moe_sort_raw(ids.ptr, plan.desc, stream)
    return plan


def experts_w8a8(Y: HIPDeviceArray, plan: MoePlan, layer: W8Layer, X: HIPDeviceArray, x_scale: HIPDeviceArray,
                 x_sorted: bool = False, y_sorted: bool = False, stream: Optional[int] = None) -> HIPDeviceArray:
    """The experts' layers on quantised rows: X (K, T) of the tokens, or with x_sorted (K, T * top_k) in the plan's order; Y
    (columns, T * top_k) by assignment, or with y_sorted in the plan's order."""
    rows = plan.tokens * plan.top_k
    _matrix("X", X, ("i8",), layer.k, rows if x_sorted else plan.tokens)
    _matrix("Y", Y, tuple(_DCODE), layer.columns, rows)
    _scales("x_scale", x_scale, X.dims[1])
    experts_w8a8_raw(plan.desc, layer.desc, X.ptr, x_scale.ptr, layer.k, Y.dtype, Y.ptr, layer.columns, x_sorted, y_sorted,
                     stream)
    return Y


def moe_combine(out: HIPDeviceArray, Y: HIPDeviceArray, weights: HIPDeviceArray, ids: Optional[HIPDeviceArray] = None,
                base: Optional[HIPDeviceArray] = None, stream: Optional[int] = None) -> HIPDeviceArray:
    """out (N, T) = base + the sum of each token's rows of Y (N, T * top_k), weighted (top_k, T); rows whose id is negative
    are left out.  base may be out itself."""
    _matrix("out", out, tuple(_DCODE))
    N, T = out.dims
    _matrix("weights", weights, ("f32",), None, T)
    k = weights.dims[0]
    _matrix("Y", Y, (out.dtype,), N, T * k)
    if ids is not None:
        _matrix("ids", ids, ("i32",), k, T)
    if base is not None:
        _matrix("base", base, (out.dtype,), N, T)
    moe_combine_raw(out.dtype, Y.ptr, N, ids.ptr if ids is not None else 0, weights.ptr, T, k, N, out.ptr, N,
                    base.ptr if base is not None else 0, N, stream)
    return out
