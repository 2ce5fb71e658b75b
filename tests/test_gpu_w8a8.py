"""Tokens quantised to 8 bits and layers with 8-bit weights on them, against float64 and whole numbers."""
import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = ("f32", "f16", "bf16")
FILL = 0x5A


def up(lh, a, dtype=None):
    """A host array (rows first) as a device array of the same bytes, features fastest."""
    a = np.ascontiguousarray(a)
    dtype = dtype or {np.dtype(np.int8): "i8", np.dtype(np.int32): "i32", np.dtype(np.float32): "f32",
                      np.dtype(np.float16): "f16", np.dtype(np.uint16): "bf16"}[a.dtype]
    d = lh.HIPDeviceArray(dtype, a.shape[::-1])
    d.copy_from(a.T)
    return d


def blank(lh, dtype, rows, ld):
    """A device array (ld, rows) of the byte FILL."""
    d = lh.HIPDeviceArray(dtype, (ld, rows))
    d.fill_bytes(FILL)
    return d


def untouched(a):
    return (np.ascontiguousarray(a).view(np.uint8) == FILL).all()


@pytest.fixture(params=range(8))
def choice(gpu, request):
    """Every kernel of the family: one that cannot take a call leaves it to the automatic choice."""
    gpu.set_kernel_override(gpu.FAMILY_W8A8, request.param)
    yield request.param
    gpu.set_kernel_override(gpu.FAMILY_W8A8, 0)


# ---- quantisation ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,pad", [(1, 1, 0), (1, 64, 0), (3, 7, 1), (5, 15, 17), (2, 16, 0), (4, 63, 1), (3, 257, 7), (2, 1024, 8),
                                     (9, 1408, 0), (1, 4096, 0), (2, 5003, 13), (1, 8192, 0), (2, 14336, 16), (1, 20001, 0), (130, 96, 32)])
def test_quantize(gpu, rng, dtype, T, K, pad):
    lh = gpu
    announce(f"quantize {dtype} {T} x {K}, rows {pad} apart")
    x = rng.standard_normal((T, K)) * np.exp(rng.standard_normal((T, 1)))
    store = ref.to_store(x, dtype)
    padded = np.zeros((T, K + pad), store.dtype)
    padded[:, :K] = store
    X, Q, S = up(lh, padded), blank(lh, "i8", T, K + pad), blank(lh, "f32", T, 1)
    lh.quantize_i8_raw(dtype, X.ptr, Q.ptr, S.ptr, K, T, K + pad, K + pad)
    lh.synchronize()
    q, s = ref.quantize(ref.to_float(store, dtype))
    got = Q.to_numpy().T
    np.testing.assert_array_equal(got[:, :K], q)
    assert untouched(got[:, K:])
    np.testing.assert_array_equal(S.to_numpy().ravel(), s.astype(np.float32))   # a quotient, rounded once


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_at_the_borders_between_integers(gpu, dtype):
    """Quotients that are halves exactly and the nearest values to them, at sizes from the least to the largest."""
    lh = gpu
    announce(f"quantize borders {dtype}")
    eps = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[dtype]
    rows = []
    for scale in {"f32": (2.0 ** -149, 2.0 ** -130, 2.0 ** -100, 1.0, 2.0 ** 120), "bf16": (2.0 ** -133, 2.0 ** -100, 1.0, 2.0 ** 120),
                  "f16": (2.0 ** -24, 2.0 ** -14, 1.0, 2.0 ** 8)}[dtype]:
        half = np.arange(0.5, 64.0, 1.0)
        rows.append(np.concatenate(([254.0], half * 2, -half * 2)) * scale)      # top 254: halves are whole steps
        rows.append(np.concatenate(([127.0], half, -half)) * scale)
        if scale >= 2.0 ** -10:
            rows.append(np.concatenate(([127.0], half * (1 + eps), -half * (1 - eps / 2))) * scale)
            rows.append(np.concatenate(([129.0], half * 1.0157, -half * (1 - eps))) * scale)
    store = ref.to_store(np.array(rows), dtype)
    T, K = store.shape
    X, Q, S = up(lh, store), blank(lh, "i8", T, K), blank(lh, "f32", T, 1)
    lh.quantize_i8(Q, S, X)
    lh.synchronize()
    q, s = ref.quantize(ref.to_float(store, dtype))
    np.testing.assert_array_equal(Q.to_numpy().T, q)
    np.testing.assert_array_equal(S.to_numpy().ravel(), s.astype(np.float32))



@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [3, 64, 1500, 9000])
def test_quantize_rows_of_zeros_and_of_what_is_not_finite(gpu, rng, dtype, K):
    lh = gpu
    announce(f"quantize zeros, infinities and NaN, {dtype} K = {K}")
    x = rng.standard_normal((6, K))
    x[1] = 0.0
    x[2] = -0.0
    x[3, K - 1] = np.inf
    x[4, K // 2] = -np.inf
    x[5, 0] = np.nan
    store = ref.to_store(x, dtype)
    X, Q, S = up(lh, store), blank(lh, "i8", 6, K), blank(lh, "f32", 6, 1)
    lh.quantize_i8_raw(dtype, X.ptr, Q.ptr, S.ptr, K, 6, K, K)
    lh.synchronize()
    q, s = ref.quantize(ref.to_float(store, dtype))
    np.testing.assert_array_equal(Q.to_numpy().T, q)
    np.testing.assert_array_equal(S.to_numpy().ravel(), s.astype(np.float32))


def test_quantize_nothing(gpu):
    """k = 0: a scale of 0 a row."""
    lh = gpu
    S = blank(lh, "f32", 3, 1)
    lh.quantize_i8_raw("f16", 0, 0, S.ptr, 0, 3, 0, 0)
    lh.synchronize()
    assert (S.to_numpy() == 0).all()


# ---- the linear layer --------------------------------------------------------------------------

def make(rng, T, N, K, extremes=False):
    if extremes:
        x, w = rng.choice([-128, 127], (T, K)).astype(np.int8), rng.choice([-128, 127], (N, K)).astype(np.int8)
        x[0], w[0] = -128, -128
    else:
        x, w = rng.integers(-127, 128, (T, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    xs = (np.exp(rng.standard_normal(T)) * 0.02).astype(np.float32)
    ws = ((rng.random(N) + 0.5) / (70 * np.sqrt(K + 1.0))).astype(np.float32)
    return x, xs, w, ws, (rng.standard_normal(N) * 0.3).astype(np.float32)


def run(lh, x, xs, w, ws, bias, act, gated, dtype, pad=(0, 0, 0), offset=0):
    """The layer's Y, (T, columns), with rows `pad` (X, W, Y) longer than they need to be and X and W `offset` bytes off."""
    (T, K), N = x.shape, w.shape[0]
    cols = N // 2 if gated else N

    def flat(a, extra):
        rows = np.full((a.shape[0], K + extra), 77, np.int8)   # what lies between rows must not count
        rows[:, :K] = a
        return up(lh, np.concatenate((np.full(offset, 99, np.int8), rows.ravel(), np.full(32, 99, np.int8))))

    X, W, Y = flat(x, pad[0]), flat(w, pad[1]), blank(lh, dtype, T, cols + pad[2])
    XS, WS, B = up(lh, xs), up(lh, ws), up(lh, bias) if bias is not None else None
    layer = lh.w8_layer_raw(W.ptr + offset, WS.ptr, N, K, K + pad[1], bias=B.ptr if B is not None else 0, act=act, gated=gated)
    lh.w8a8_raw(layer, X.ptr + offset, XS.ptr, T, K + pad[0], dtype, Y.ptr, cols + pad[2])
    lh.synchronize()
    got = Y.to_numpy().T
    assert untouched(got[:, cols:])
    return got[:, :cols]


def check(got, want, dtype):
    y, err = want
    off = np.abs(ref.to_float(got, dtype) - y)
    bad = ~(off <= err) & ~((np.abs(y) > 6.5e4) & (dtype == "f16"))
    assert not bad.any(), f"{bad.sum()} of {bad.size} values off, the first at {np.argwhere(bad)[0]}: {ref.to_float(got, dtype)[bad][0]} for {y[bad][0]} +- {err[bad][0]}"


# rows around the kernels' tiles (16, 32, 64, 128, 256) and channels and K around theirs; every type, activation and gate
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 64, 128), (1, 4096, 256), (2, 48, 64), (3, 7, 5), (5, 30, 33), (15, 130, 80), (16, 32, 272),
          (17, 64, 1040), (31, 96, 64), (32, 100, 144), (33, 128, 512), (48, 66, 208), (63, 40, 96), (64, 256, 384), (65, 18, 1000),
          (100, 258, 128), (127, 128, 112), (128, 128, 640), (129, 272, 336), (130, 1000, 48), (255, 130, 160), (256, 256, 256),
          (257, 514, 400), (300, 384, 1168), (513, 770, 144)]
KINDS = [("none", False), ("relu", False), ("gelu_tanh", False), ("gelu_erf", False), ("silu", False), ("silu", True),
         ("gelu_tanh", True), ("none", True)]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear(gpu, choice, i):
    lh = gpu
    T, N, K = SHAPES[i]
    rng = np.random.default_rng(100 + i)
    x, xs, w, ws, bias = make(rng, T, N, K)
    for j in range(3):
        (act, gated), dtype = KINDS[(i + 3 * j) % len(KINDS)], DTYPES[(i + j) % 3]
        n = N // 2 * 2 if gated else N
        b = bias[:n] if (i + j) % 2 else None
        if n == 0:
            continue
        announce(f"linear {T} x {n} x {K} {act} gated={gated} {dtype} bias={b is not None} choice {choice}")
        got = run(lh, x, xs, w[:n], ws[:n], b, act, gated, dtype)
        check(got, ref.layer(x, xs, w[:n], ws[:n], b, act, gated, dtype), dtype)


@pytest.mark.parametrize("T,N,K", [(1, 64, 256), (20, 96, 192), (70, 130, 320), (300, 520, 256)])
@pytest.mark.parametrize("pad,offset", [((16, 32, 4), 0), ((16, 16, 3), 16), ((1, 0, 0), 0), ((0, 5, 1), 0), ((16, 0, 8), 1),
                                        ((8, 8, 2), 8)])
def test_linear_strides_and_alignment(gpu, choice, T, N, K, pad, offset):
    lh = gpu
    announce(f"linear {T} x {N} x {K}, rows {pad} longer, {offset} bytes off, choice {choice}")
    x, xs, w, ws, bias = make(np.random.default_rng(7), T, N, K)
    got = run(lh, x, xs, w, ws, bias, "none", False, "f32", pad, offset)
    check(got, ref.layer(x, xs, w, ws, bias, "none", False, "f32"), "f32")


@pytest.mark.parametrize("T,N,K", [(1, 16, 131071), (16, 32, 131056), (130, 140, 65536)])
def test_linear_of_the_largest_sums(gpu, choice, T, N, K):
    """-128 times -128 in every place of a row: the 32-bit sums' end."""
    lh = gpu
    announce(f"linear largest sums {T} x {N} x {K}, choice {choice}")
    x, xs, w, ws, _ = make(np.random.default_rng(8), T, N, K, extremes=True)
    got = run(lh, x, xs, w, ws, None, "none", False, "f32")
    check(got, ref.layer(x, xs, w, ws, None, "none", False, "f32"), "f32")


def test_linear_without_k(gpu, choice):
    """k = 0: the bias alone, through the activation."""
    lh = gpu
    announce(f"linear k = 0, choice {choice}")
    x, xs, w, ws, bias = make(np.random.default_rng(9), 5, 20, 0)
    B, XS, WS, Y = up(lh, bias), up(lh, xs), up(lh, ws), blank(lh, "f32", 5, 20)
    lh.w8a8_raw(lh.w8_layer_raw(0, WS.ptr, 20, 0, 0, bias=B.ptr, act="silu"), 0, XS.ptr, 5, 0, "f32", Y.ptr, 20)
    lh.synchronize()
    check(Y.to_numpy().T, ref.layer(x, xs, w, ws, bias, "silu", False, "f32"), "f32")


def test_linear_shows_scales_that_are_not_finite(gpu, choice):
    """A token whose scale is NaN (its row held one) gives NaN, through every activation; the others' results stand."""
    lh = gpu
    announce(f"linear NaN scales, choice {choice}")
    x, xs, w, ws, bias = make(np.random.default_rng(10), 40, 64, 128)
    bad = xs.copy()
    bad[[3, 39]] = np.nan
    for act, gated in KINDS:
        good, got = (run(lh, x, s, w, ws, bias, act, gated, "f32") for s in (xs, bad))
        assert np.isnan(got[[3, 39]]).all()
        keep = [t for t in range(40) if t not in (3, 39)]
        np.testing.assert_array_equal(got[keep], good[keep])


@pytest.mark.parametrize("T,N,K", [(2100, 2180, 97), (2180, 2100, 272), (40, 33000, 131), (2050, 2306, 15)])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_of_many_tiles(gpu, T, N, K, gated):
    """More tiles than CUs, on the kernel the library chooses and on the generic one."""
    lh = gpu
    x, xs, w, ws, bias = make(np.random.default_rng(13), T, N, K)
    want = ref.layer(x, xs, w, ws, bias, "relu", gated, "f16")
    got = {}
    for c in (0, 1):
        announce(f"linear {T} x {N} x {K} gated={gated}, choice {c}")
        lh.set_kernel_override(lh.FAMILY_W8A8, c)
        try:
            got[c] = run(lh, x, xs, w, ws, bias, "relu", gated, "f16", (K % 2, K % 3, 1))
        finally:
            lh.set_kernel_override(lh.FAMILY_W8A8, 0)
        check(got[c], want, "f16")
    np.testing.assert_array_equal(got[0].view(np.uint16), got[1].view(np.uint16))


@pytest.mark.parametrize("T,N,K,act,gated", [(1, 128, 512, "silu", True), (16, 256, 256, "none", False), (40, 96, 128, "gelu_erf", False),
                                             (200, 384, 640, "gelu_tanh", True), (600, 512, 256, "silu", False)])
def test_every_kernel_gives_the_same_bits(gpu, T, N, K, act, gated):
    lh = gpu
    x, xs, w, ws, bias = make(np.random.default_rng(11), T, N, K)
    got = {}
    for c in range(8):
        announce(f"linear {T} x {N} x {K} {act}, choice {c}")
        lh.set_kernel_override(lh.FAMILY_W8A8, c)
        try:
            got[c] = run(lh, x, xs, w, ws, bias, act, gated, "f32")
        finally:
            lh.set_kernel_override(lh.FAMILY_W8A8, 0)
    for c in got:
        np.testing.assert_array_equal(got[c].view(np.uint32), got[0].view(np.uint32), err_msg=f"choice {c}")


def test_quantised_tokens_through_a_layer(gpu, rng):
    """The arrays' form of both calls, one behind the other, on a stream of its own."""
    lh = gpu
    announce("quantize and linear through arrays")
    T, N, K = 70, 96, 256
    x, w = rng.standard_normal((T, K)), rng.integers(-127, 128, (N, K)).astype(np.int8)
    ws = ((rng.random(N) + 0.5) * 1e-4).astype(np.float32)
    store = ref.to_store(x, "bf16")
    X, W, WS = up(lh, store), up(lh, w), up(lh, ws)
    Q, S, Y = blank(lh, "i8", T, K), lh.HIPDeviceArray("f32", (T,)), blank(lh, "f16", T, N // 2)
    layer = lh.W8Layer(W, WS, act="silu", gated=True)
    lh.synchronize()
    st = lh.Stream()
    lh.quantize_i8(Q, S, X, stream=st.handle)
    lh.w8a8(Y, layer, Q, S, stream=st.handle)
    st.synchronize()
    q, s = ref.quantize(ref.to_float(store, "bf16"))
    check(Y.to_numpy().T, ref.layer(q, s.astype(np.float32), w, ws, None, "silu", True, "f16"), "f16")
    st.close()
    with pytest.raises(ValueError):
        lh.w8a8(Y, layer, X, S)
    with pytest.raises(ValueError):
        lh.quantize_i8(Q, WS, X)


def test_a_layer_whose_tokens_and_channels_pass_32_bits(gpu, choice):
    """Rows 65536 bytes apart: the last token and the last channel lie 2 GiB behind the first."""
    lh = gpu
    announce(f"linear past 2 GiB, choice {choice}")
    K, ld, far = 128, 65536, 32800
    rng = np.random.default_rng(12)
    a = lh.HIPDeviceArray("i8", (ld * far,))
    few, one = rng.integers(-127, 128, (40, K)).astype(np.int8), rng.integers(-127, 128, (3, K)).astype(np.int8)
    seen = [0, 32768, far - 1]
    a.fill_bytes(0)
    for n, row in zip(seen, one):
        lh._lib.call("lava_hip_memcpy_h2d", a.ptr + n * ld, row.ctypes.data, K)
    F, ones = up(lh, few), up(lh, np.ones(far, np.float32))
    try:
        for far_tokens in (False, True):
            T, N = (far, 40) if far_tokens else (40, far)
            Y = blank(lh, "f32", T, N)
            X, W = (a, F) if far_tokens else (F, a)
            layer = lh.w8_layer_raw(W.ptr, ones.ptr, N, K, K if far_tokens else ld)
            lh.w8a8_raw(layer, X.ptr, ones.ptr, T, ld if far_tokens else K, "f32", Y.ptr, N)
            lh.synchronize()
            got = Y.to_numpy() if far_tokens else Y.to_numpy().T      # (40, far)
            Y.close()
            want = np.zeros((40, far))
            want[:, seen] = few.astype(np.float64) @ one.T.astype(np.float64)
            np.testing.assert_array_equal(got, want)
    finally:
        a.close()


def test_quantize_around_2_32_threads(gpu):
    """Launches of 2^32 threads in one dimension (a wavefront a row), which HIP runs modulo 2^32, are refused by name."""
    lh = gpu
    T = 2 ** 26
    announce(f"quantize {T} rows of 1")
    X, Q, S = lh.HIPDeviceArray("f16", (T,)), lh.HIPDeviceArray("i8", (T,)), lh.HIPDeviceArray("f32", (T,))
    try:
        X.fill_bytes(0x3c)
        Q.fill_bytes(FILL)
        lh.synchronize()
        with pytest.raises(lh.Unsupported, match="quantize_rows_kernel"):
            lh.quantize_i8_raw("f16", X.ptr, Q.ptr, S.ptr, 1, T, 1, 1)
        lh.synchronize()
        assert untouched(Q.to_numpy())
        lh.quantize_i8_raw("f16", X.ptr, Q.ptr, S.ptr, 1, T - 4, 1, 1)
        lh.synchronize()
        q = Q.to_numpy()
        assert (q[:-4] == 127).all() and (q[-4:] == FILL).all()
    finally:
        for a in (X, Q, S):
            a.close()
