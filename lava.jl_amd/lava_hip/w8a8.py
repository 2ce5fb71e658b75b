"""Linear layers with 8-bit weights on 8-bit tokens: `quantize_i8` and `w8a8`, destination-first like the other kernels,
over HIPDeviceArrays or raw device addresses.

Arrays keep the paged cache's order, the features fastest: tokens are (K, T) arrays with a scale a token, a layer's weights a
(K, N) array with a scale a channel, results (N, T).  The `*_raw` constructors make the descriptors of
include/lava_hip.h from addresses; a serving program makes them once.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib
from .device import HIPDeviceArray
from .kernels import _ACTS, _DCODE

_W8_ACTS = {**_ACTS, "silu": _lib.ACT_SILU}


def _fits(bits: int, **values: int) -> None:
    """Refuses what a descriptor's integers would cut off."""
    for name, x in values.items():
        if not -2 ** (bits - 1) <= x < 2 ** (bits - 1):
            raise ValueError(f"{name} = {x} does not fit {bits} bits")


def _cut(*values: int) -> bool:
    """Whether a 64-bit argument may be cut off: the bits of all together leave the range where one does, or are negative where one
    is, which would hide it."""
    together = 0
    for x in values:
        together |= x
    return not 0 <= together < 2 ** 63


def _code(dtype: str) -> int:
    if dtype not in _DCODE:
        raise _lib.Unsupported(_lib.ERR_UNSUPPORTED, f"{dtype!r} is not f32, f16 or bf16")
    return _DCODE[dtype]


def quantize_i8_raw(dtype: str, X: int, Q: int, scale: int, k: int, tokens: int, ldx: int, ldq: int,
                    stream: Optional[int] = None) -> None:
    if _cut(k, tokens, ldx, ldq):
        _fits(64, k=k, tokens=tokens, ldx=ldx, ldq=ldq)
    _lib.call("lava_hip_quantize_i8", _code(dtype), X or None, Q or None, scale or None, k, tokens, ldx, ldq, stream)


def w8_layer_raw(w: int, scale: int, n: int, k: int, ldw: int, bias: int = 0, act: str = "none", gated: bool = False,
                 experts: int = 1, expert_stride: int = 0) -> _lib.W8LayerDesc:
    """n channels of k weights at `w` (ldw apart, K contiguous) with a scale each; of several experts expert_stride apart."""
    if act not in _W8_ACTS:
        raise ValueError(f"act must be one of {sorted(_W8_ACTS)}")
    _fits(64, n=n, k=k, ldw=ldw, expert_stride=expert_stride)
    _fits(32, experts=experts)
    return _lib.W8LayerDesc(w or None, scale or None, bias or None, n, k, ldw, expert_stride, experts, _W8_ACTS[act],
                            int(bool(gated)))


def w8a8_raw(layer: _lib.W8LayerDesc, X: int, x_scale: int, tokens: int, ldx: int, y_dtype: str, Y: int, ldy: int,
             stream: Optional[int] = None) -> None:
    if _cut(tokens, ldx, ldy):
        _fits(64, tokens=tokens, ldx=ldx, ldy=ldy)
    _lib.call("lava_hip_gemm_w8a8", C.byref(layer), X or None, x_scale or None, tokens, ldx, _code(y_dtype), Y or None, ldy,
              stream)


class W8Layer:
    """A layer of int8 weights `w` (K, N) or, of several experts, (K, N, experts), with f32 `scale` (and `bias`) (N) or
    (N, experts).  A gated layer's first N / 2 channels are the gate's."""

    def __init__(self, w: HIPDeviceArray, scale: HIPDeviceArray, bias: Optional[HIPDeviceArray] = None, act: str = "none",
                 gated: bool = False):
        if w.dtype != "i8" or len(w.dims) not in (2, 3) or w.order != "F":
            raise ValueError("w must be a column-major i8 array (K, N) or (K, N, experts)")
        for name, a in (("scale", scale), ("bias", bias)):
            if a is not None and (a.dtype != "f32" or a.dims != w.dims[1:] or a.order != "F"):
                raise ValueError(f"{name} must be an f32 array {w.dims[1:]}, like w's channels")
        self.w, self.scale, self.bias = w, scale, bias
        self.k, self.n = w.dims[:2]
        self.experts = w.dims[2] if len(w.dims) == 3 else 1
        self.columns = self.n // 2 if gated else self.n
        self.desc = w8_layer_raw(w.ptr, scale.ptr, self.n, self.k, self.k, bias.ptr if bias is not None else 0, act, gated,
                                 self.experts, self.k * self.n)


def _matrix(name: str, a: HIPDeviceArray, dtypes, rows: Optional[int] = None, cols: Optional[int] = None) -> None:
    if a.dtype not in dtypes or len(a.dims) != 2 or a.order != "F":
        raise ValueError(f"{name} must be a column-major 2-D array of {' or '.join(dtypes)}")
    if (rows is not None and a.dims[0] != rows) or (cols is not None and a.dims[1] != cols):
        raise ValueError(f"shape mismatch: {name} {a.dims}, expected ({rows}, {cols})")


def _scales(name: str, a: HIPDeviceArray, n: int) -> None:
    if a.dtype != "f32" or a.size != n:
        raise ValueError(f"{name} must be an f32 vector of {n} scales")


def quantize_i8(Q: HIPDeviceArray, scale: HIPDeviceArray, X: HIPDeviceArray, stream: Optional[int] = None) -> HIPDeviceArray:
    """The tokens X (K, T) in 8 bits: Q (K, T), and a scale a token."""
    _matrix("X", X, tuple(_DCODE))
    _matrix("Q", Q, ("i8",), *X.dims)
    _scales("scale", scale, X.dims[1])
    quantize_i8_raw(X.dtype, X.ptr, Q.ptr, scale.ptr, X.dims[0], X.dims[1], X.dims[0], X.dims[0], stream)
    return Q


def w8a8(Y: HIPDeviceArray, layer: W8Layer, X: HIPDeviceArray, x_scale: HIPDeviceArray,
         stream: Optional[int] = None) -> HIPDeviceArray:
    """The layer on quantised tokens X (K, T) with their scales: Y (columns, T), f16, bf16 or f32."""
    _matrix("X", X, ("i8",), layer.k)
    _matrix("Y", Y, tuple(_DCODE), layer.columns, X.dims[1])
    _scales("x_scale", x_scale, X.dims[1])
    w8a8_raw(layer.desc, X.ptr, x_scale.ptr, X.dims[1], layer.k, Y.dtype, Y.ptr, layer.columns, stream)
    return Y
