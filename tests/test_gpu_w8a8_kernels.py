"""Which kernel of the layers with 8-bit weights runs, read from the kernel log; every tile with both of its rings of stages, and
the largest numbers of channels and tokens."""
import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce
from test_gpu_moe import check_experts, experts_case, run_experts
from test_gpu_w8a8 import FILL, blank, check, make, run, up

pytestmark = pytest.mark.gpu

# pin: rows and channels of a tile, its stages where a CU has one tile at most, and where it has more
RINGS = {3: (64, 64, 4, 3), 4: (64, 128, 3, 2), 5: (128, 128, 3, 2), 6: (128, 256, 3, 3), 7: (256, 256, 2, 2)}
# bytes of K: two stages of 128, three, four, five and nine, the last of 16 bytes each; rings have two to four
DEPTHS = [144, 272, 400, 528, 1040]


def ran(lh, pin, call):
    """call's result under the pin, and the names in the kernel log."""
    lh.set_kernel_override(lh.FAMILY_W8A8, pin)
    lh.kernel_log_clear()
    try:
        got = call()
        return got, [n for n in lh.kernel_log() if n.startswith("w8a8")]
    finally:
        lh.set_kernel_override(lh.FAMILY_W8A8, 0)


def names(pin, many):
    if pin == 1:
        return ["w8a8_generic_kernel"]
    if pin == 2:
        return ["w8a8_stream_kernel"]
    bm, bn, few, more = RINGS[pin]
    return [f"w8a8_tile_kernel<{bm},{bn}>", f"w8a8_tile_kernel<{bm},{bn},{more if many else few}>"]


# ---- the rings ---------------------------------------------------------------------------------

@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("K", DEPTHS)
@pytest.mark.parametrize("pin", list(RINGS))
def test_linear_on_every_ring(gpu, pin, K, many, gated):
    """6 tiles and 272, ragged in rows and channels: the generic kernel's bits, and rows of the first and last tiles in float64."""
    lh = gpu
    bm, bn = RINGS[pin][:2]
    tiles_m, tiles_n = (16, 17) if many else (2, 3)
    cols = tiles_n * (bn // 2 if gated else bn) - 9
    T, N, act = tiles_m * bm - 5, cols * (1 + gated), "silu" if gated else "gelu_tanh"
    announce(f"ring of pin {pin}, {T} x {N} x {K} gated={gated}")
    x, xs, w, ws, bias = make(np.random.default_rng(pin * 10000 + K), T, N, K)
    call = lambda: run(lh, x, xs, w, ws, bias, act, gated, "f32", (16, 0, 0))  # noqa: E731
    got, log = ran(lh, pin, call)
    assert log == names(pin, many)
    plain, log = ran(lh, 1, call)
    assert log == names(1, many)
    np.testing.assert_array_equal(got.view(np.uint32), plain.view(np.uint32))
    rows = [0, 1, bm // 2, bm - 1, T - bm, T - 1]
    check(got[rows], ref.layer(x[rows], xs[rows], w, ws, bias, act, gated, "f32"), "f32")


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("K", [272, 400, 1040])
@pytest.mark.parametrize("pin", list(RINGS))
def test_experts_on_every_ring(gpu, pin, K, many, back):
    """Five uneven experts; gated from the tokens' rows, or back from the plan's."""
    lh = gpu
    bm, bn = RINGS[pin][:2]
    T, gated = (4 * bm if many else bm // 2) + 3, not back
    N = 27 * bn if many else bn + 2
    announce(f"experts on a ring of pin {pin}, {T} tokens x {N} x {K} back={back}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(pin * 10000 + K + 1), T, 5, 2, N, K)
    ids[:T // 2, 0] = 3
    ids[:T // 2, 1] = 1
    if not back:
        x, xs = x[:T], xs[:T]
    args = (ids, x, xs, w, ws, bias, "silu" if gated else "none", gated, "f32", back, not back)
    got, log = ran(lh, pin, lambda: run_experts(lh, *args))
    assert log == names(pin, many)
    plain, log = ran(lh, 1, lambda: run_experts(lh, *args))
    assert log == names(1, many)
    np.testing.assert_array_equal(got.view(np.uint32), plain.view(np.uint32))
    if not many:
        check_experts(got, *args)


@pytest.mark.parametrize("pin", [3, 4, 5])
def test_a_decode_step_s_experts(gpu, pin):
    """32 tokens' 8 of 64 experts, gated: a few rows of each, more tiles than CUs."""
    lh = gpu
    announce(f"a decode step's experts, pin {pin}")
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(50), 32, 64, 8, 640, 400)
    args = (ids, x[:32], xs[:32], w, ws, bias, "silu", True, "f16", False, True)
    got, log = ran(lh, pin, lambda: run_experts(lh, *args))
    assert log == names(pin, True)
    check_experts(got, *args)


# ---- which kernel ------------------------------------------------------------------------------

@pytest.mark.parametrize("pin", range(1, 8))
def test_a_pin_is_the_kernel_that_runs(gpu, pin):
    lh = gpu
    announce(f"pin {pin}")
    x, xs, w, ws, bias = make(np.random.default_rng(51), 16, 32, 144)
    got, log = ran(lh, pin, lambda: run(lh, x, xs, w, ws, bias, "relu", False, "f32"))
    assert log == names(pin, False)
    check(got, ref.layer(x, xs, w, ws, bias, "relu", False, "f32"), "f32")


@pytest.mark.parametrize("pin", range(8))
@pytest.mark.parametrize("K,pad,offset", [(33, (0, 0, 0), 0), (144, (8, 0, 0), 0), (144, (0, 4, 0), 0), (144, (0, 0, 0), 8)])
def test_layouts_of_the_generic_kernel(gpu, pin, K, pad, offset):
    """K, rows or bases that are no multiples of 16 bytes."""
    lh = gpu
    announce(f"generic layouts K = {K} {pad} {offset}, pin {pin}")
    x, xs, w, ws, bias = make(np.random.default_rng(52), 16, 32, K)
    got, log = ran(lh, pin, lambda: run(lh, x, xs, w, ws, bias, "none", False, "f32", pad, offset))
    assert log == names(1, False)
    check(got, ref.layer(x, xs, w, ws, bias, "none", False, "f32"), "f32")


@pytest.mark.parametrize("T,pin,ld,want", [(5, 7, 2 ** 23 - 16, 7), (5, 7, 2 ** 23, 2), (40, 7, 2 ** 23, 3), (40, 2, 2 ** 25, 2), (40, 2, 2 ** 27, 1),
                                             (5, 3, 2 ** 25, 2), (40, 3, 2 ** 25, 1), (40, 6, 2 ** 25, 1)])
def test_channels_that_a_kernel_cannot_span(gpu, T, pin, ld, want):
    """Channels so far apart that a tile's would span 2 GiB: the pinned kernel is passed over for the one that runs without a pin."""
    lh = gpu
    announce(f"rows of weights {ld} bytes apart, {T} tokens, pin {pin}")
    rng = np.random.default_rng(53)
    x, w = rng.integers(-127, 128, (T, 128)).astype(np.int8), rng.integers(-127, 128, (2, 128)).astype(np.int8)
    W, X, one, Y = lh.HIPDeviceArray("i8", (ld + 128,)), up(lh, x), up(lh, np.ones(T, np.float32)), blank(lh, "f32", T, 2)
    for n in range(2):
        lh._lib.call("lava_hip_memcpy_h2d", W.ptr + n * ld, w[n].ctypes.data, 128)
    try:
        _, log = ran(lh, pin, lambda: lh.w8a8_raw(lh.w8_layer_raw(W.ptr, one.ptr, 2, 128, ld), X.ptr, one.ptr, T, 128, "f32", Y.ptr, 2))
        lh.synchronize()
        assert log == names(want, False)
        np.testing.assert_array_equal(Y.to_numpy().T, x.astype(np.float64) @ w.T.astype(np.float64))
    finally:
        W.close()


# rows, channels, K and the pin whose kernel the library takes by itself, more tiles than CUs or not
CHOSEN = [(1, 4096, 4096, 2, False), (16, 7168, 512, 2, False), (16, 7169, 512, 3, False), (17, 64, 512, 3, False),
          (16, 14336, 4096, 3, False), (40, 33000, 256, 3, True), (64, 28672, 4096, 4, False), (512, 4096, 2048, 4, False),
          (1024, 4096, 4096, 5, False), (600, 8192, 256, 5, True), (333, 14336, 4096, 6, False), (4096, 4096, 4096, 7, False),
          (8192, 4096, 4096, 7, True), (64, 64, 4095, 1, False)]


@pytest.mark.parametrize("T,N,K,pin,many", CHOSEN)
def test_the_kernel_that_is_chosen(gpu, T, N, K, pin, many):
    lh = gpu
    announce(f"the choice for {T} x {N} x {K}")
    X, W, one, Y = blank(lh, "i8", T, K), blank(lh, "i8", N, K), up(lh, np.ones(max(T, N), np.float32)), lh.HIPDeviceArray("f32", (N, T))
    _, log = ran(lh, 0, lambda: lh.w8a8_raw(lh.w8_layer_raw(W.ptr, one.ptr, N, K, K), X.ptr, one.ptr, T, K, "f32", Y.ptr, N))
    lh.synchronize()
    assert log == names(pin, many)
    assert (Y.to_numpy() == FILL * FILL * K).all()


# ---- the largest -------------------------------------------------------------------------------

MOST = 2 ** 31 - 256


def put(lh, at, a):
    lh._lib.call("lava_hip_memcpy_h2d", at, a.ctypes.data, a.nbytes)


@pytest.mark.parametrize("gated", [False, True])
def test_the_most_channels(gpu, gated):
    """One token, K = 16: more tiles of 64 x 64 than a launch holds, so a wider tile runs."""
    lh = gpu
    announce(f"{MOST} channels, gated={gated}")
    K, cols = 16, MOST // 2 if gated else MOST
    rng = np.random.default_rng(54)
    seen = np.array([0, 1, cols // 2, cols - 130, cols - 2, cols - 1])
    x, w = rng.integers(-127, 128, K).astype(np.int8), rng.integers(-127, 128, (seen.size, K)).astype(np.int8)
    W, S, Y = lh.HIPDeviceArray("i8", (MOST * K,)), lh.HIPDeviceArray("f32", (MOST,)), lh.HIPDeviceArray("f16", (cols,))
    X, one = up(lh, x), up(lh, np.float32([2.0 ** -6]))
    try:
        W.fill_bytes(0)
        S.fill_bytes(0x3c)
        Y.fill_bytes(FILL)
        s = float(np.array([0x3c3c3c3c], np.uint32).view(np.float32)[0])
        for n, row in zip(seen, w):
            put(lh, W.ptr + int(n) * K, row)
            if gated:
                put(lh, W.ptr + int(n + cols) * K, w[0])
        lh.synchronize()
        layer = lh.w8_layer_raw(W.ptr, S.ptr, MOST, K, K, gated=gated)
        _, log = ran(lh, 0, lambda: lh.w8a8_raw(layer, X.ptr, one.ptr, 1, K, "f16", Y.ptr, cols))
        lh.synchronize()
        assert log == names(4, True)
        got = Y.to_numpy()
    finally:
        for a in (W, S, Y):
            a.close()
    sums = w.astype(np.float64) @ x * 2.0 ** -6 * s
    want = sums * sums[0] if gated else sums
    assert (np.abs(got[seen] - want) <= np.abs(want) * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25).all()
    got[seen] = 0
    assert not got.any()


def test_the_most_tokens(gpu):
    """One channel: only tiles of 256 rows fit a launch."""
    lh = gpu
    announce(f"{MOST} tokens")
    K = 16
    rng = np.random.default_rng(55)
    seen = np.array([0, 1, MOST // 2, MOST - 257, MOST - 1])
    x, w = rng.integers(-127, 128, (seen.size, K)).astype(np.int8), rng.integers(-127, 128, (1, K)).astype(np.int8)
    X, S, Y = lh.HIPDeviceArray("i8", (MOST * K,)), lh.HIPDeviceArray("f32", (MOST,)), lh.HIPDeviceArray("f16", (MOST,))
    W, one = up(lh, w), up(lh, np.float32([0.5]))
    try:
        X.fill_bytes(0)
        S.fill_bytes(0x3c)
        Y.fill_bytes(FILL)
        s = float(np.array([0x3c3c3c3c], np.uint32).view(np.float32)[0])
        for t, row in zip(seen, x):
            put(lh, X.ptr + int(t) * K, row)
        lh.synchronize()
        layer = lh.w8_layer_raw(W.ptr, one.ptr, 1, K, K)
        _, log = ran(lh, 0, lambda: lh.w8a8_raw(layer, X.ptr, S.ptr, MOST, K, "f16", Y.ptr, 1))
        lh.synchronize()
        assert log == names(7, True)
        got = Y.to_numpy()
    finally:
        for a in (X, S, Y):
            a.close()
    want = x.astype(np.float64) @ w[0] * 0.5 * s
    assert (np.abs(got[seen] - want) <= np.abs(want) * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25).all()
    got[seen] = 0
    assert not got.any()
