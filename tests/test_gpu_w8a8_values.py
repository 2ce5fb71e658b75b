"""The activations of layers with 8-bit weights over all of their argument, infinities among it: a layer without K gives the
activation of its biases."""
import math

import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce
from test_gpu_w8a8 import blank, up

pytestmark = pytest.mark.gpu

U = ref.U


def activation(lh, act, x, kernel=0):
    """act(x) in f32 by a layer of one token, x its biases."""
    x = np.ascontiguousarray(x, np.float32)
    B, one, WS, Y = up(lh, x), up(lh, np.ones(1, np.float32)), up(lh, np.ones(x.size, np.float32)), blank(lh, "f32", 1, x.size)
    lh.set_kernel_override(lh.FAMILY_W8A8, kernel)
    try:
        lh.w8a8_raw(lh.w8_layer_raw(0, WS.ptr, x.size, 0, 0, bias=B.ptr, act=act), 0, one.ptr, 1, 0, "f32", Y.ptr, x.size)
        lh.synchronize()
    finally:
        lh.set_kernel_override(lh.FAMILY_W8A8, 0)
    return Y.to_numpy().ravel()


def everywhere():
    """Values of both signs: 4096 of each power of two from the subnormal ones to the largest, and all around where the tail ends."""
    m = np.random.default_rng(40).integers(0, 1 << 23, (255, 4096)).astype(np.uint32)
    x = ((np.arange(255, dtype=np.uint32)[:, None] << 23) | m).view(np.float32).ravel()
    near = np.concatenate([np.nextafter(np.float32(v), np.float32(to)).reshape(1) for v in (1, 2, 3, 6, 10, 13, 16) for to in (0, v, 99)])
    return np.concatenate((x, near, np.linspace(1e-3, 14.5, 200001).astype(np.float32)))


def test_gelu_erf_over_all_numbers(gpu):
    """Below zero the result is a product of x with e / 2, e = erfc(|x| / sqrt 2) = 2^-E, E = a (a log2(e) / 2 + G(t)), a = |x|.  In units of
    half a step, 2^-24, what it may be off by: t = 1 / (1 + c a) by its sum and the reciprocal 3, which moves G by t G' (at most 1.43) of
    that; G's seven fused steps 2.1; the constant a^2 log2(e) / 2 of itself; the sum and the product by a 2 E; ln 2 of all that times a;
    the fit and its coefficients 0.7 up to a = 1, 2.2 up to 6, 17.2 up to 14; 2^-E 2, the product with x 1: less than 3.5 + 6 a + 1.5 a^2
    (worked out at 200000 places up to 14, behind which e is below the least normal float and may come out as zero).  Above zero the
    factor is 1 - e / 2: that of e by e / 2 of the factor, and two roundings."""
    lh = gpu
    announce("gelu_erf over all numbers")
    a = everywhere()
    a64 = a.astype(np.float64)
    tail = np.vectorize(math.erfc, otypes=[float])(a64 * math.sqrt(0.5)) / 2
    steps = 3.5 + 6 * a64 + 1.5 * np.minimum(a64, 14) ** 2
    flush = a64 * 2.0 ** -126 * (a64 < 15) + 2.0 ** -148
    y = -a64 * tail
    off = np.abs(activation(lh, "gelu_erf", -a).astype(np.float64) - y)
    bad = ~(off <= steps * U * -y + flush)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax((off - flush) / (-y * U + 1e-300)):.1f} half steps, x = {-a[bad][0]}"
    y = a64 * (1 - tail)
    off = np.abs(activation(lh, "gelu_erf", a).astype(np.float64) - y)
    bad = ~(off <= (2 + (steps - 1) * tail / (1 - tail)) * U * y + flush)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, x = {a[bad][0]}, off {off[bad][0] / (y[bad][0] * U)} half steps"


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_silu_and_gelu_tanh_over_their_range(gpu, act):
    """Within the bound that the layers' tests use; results below zero and above -2^-119 may be 0: 1 / (1 + exp) is below the least
    normal float from 2^126 on, times |x| of up to 88."""
    lh = gpu
    announce(f"{act} over its range")
    a = everywhere()
    a = np.concatenate((a[a < 400], np.linspace(14, 130, 100001).astype(np.float32)))
    x = np.concatenate((-a, a))
    off = np.abs(activation(lh, act, x).astype(np.float64) - ref.act(act, x.astype(np.float64)))
    bad = ~(off <= ref.act_error(act, x.astype(np.float64), 0.0) + (x < 0) * 2.0 ** -119 + 2.0 ** -148)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, x = {x[bad][0]}, off {off[bad][0]}"


@pytest.mark.parametrize("act", ["none", "relu", "gelu_tanh", "gelu_erf", "silu"])
def test_activations_of_infinities_zeros_and_nan(gpu, act):
    """As their formulas have them: a product of -infinity with zero is NaN, and +infinity stays."""
    lh = gpu
    x = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 3e38, -3e38, 1e20, -1e20, 2.0 ** -149, -2.0 ** -149], np.float32)
    want = {"none": -np.inf, "relu": 0.0}.get(act, np.nan)
    low = {"none": x[[6, 8]]}.get(act, np.zeros(2))
    for kernel in (0, 1):
        announce(f"{act} of infinities, choice {kernel}")
        y = activation(lh, act, x, kernel)
        np.testing.assert_array_equal(y[:6], np.array([np.inf, want, np.nan, 0.0, 0.0, x[5]], np.float32))
        np.testing.assert_array_equal(y[[6, 8]], low)
        assert y[7] == x[7] and abs(y[9]) <= x[9] and abs(y[10]) <= x[9]


def test_a_bias_of_minus_infinity_in_a_layer(gpu):
    """A channel whose bias is -infinity, on the tile kernels: NaN where the activation's formula gives it, other channels untouched."""
    lh = gpu
    announce("a bias of -infinity on tiles")
    rng = np.random.default_rng(41)
    x, w = rng.integers(-127, 128, (70, 256)).astype(np.int8), rng.integers(-127, 128, (96, 256)).astype(np.int8)
    xs, ws, bias = np.full(70, 0.02, np.float32), np.full(96, 1e-3, np.float32), rng.standard_normal(96).astype(np.float32)
    X, W, XS, WS = up(lh, x), up(lh, w), up(lh, xs), up(lh, ws)
    for act in ("relu", "gelu_tanh", "gelu_erf", "silu"):
        got = []
        for low in (False, True):
            b = bias.copy()
            if low:
                b[5] = -np.inf
            B, Y = up(lh, b), blank(lh, "f32", 70, 96)
            lh.w8a8_raw(lh.w8_layer_raw(W.ptr, WS.ptr, 96, 256, 256, bias=B.ptr, act=act), X.ptr, XS.ptr, 70, 256, "f32", Y.ptr, 96)
            lh.synchronize()
            got.append(Y.to_numpy().T)
        keep = [n for n in range(96) if n != 5]
        np.testing.assert_array_equal(got[1][:, keep], got[0][:, keep])
        assert (got[1][:, 5] == 0).all() if act == "relu" else np.isnan(got[1][:, 5]).all()
