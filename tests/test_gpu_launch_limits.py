"""Launches of 2^32 threads and more in one dimension, which HIP runs modulo 2^32 without an error: refused by name, and the
largest below them right."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [65535, 65537])
def test_generic_w8a16_around_2_32_elements(gpu, rows):
    """A thread an element of Y (K = 4 is for no other kernel): rows x 65536 of them."""
    lh = gpu
    announce(f"generic W8A16, {rows} x 65536 elements")
    M, N, K = rows, 65536, 4
    rng = np.random.default_rng(3)
    x, w = rng.integers(-8, 9, (M, K)), rng.integers(-8, 9, (K, N))
    X = lh.HIPDeviceArray.from_numpy(x.astype(np.float16), "f16", "C")
    W = lh.HIPDeviceArray.from_numpy(w.astype(np.int8), "i8", "C")
    S = lh.HIPDeviceArray.from_numpy(np.ones(N, np.float16), "f16")
    Y = lh.HIPDeviceArray("f32", (M, N), order="C")
    Y.fill_bytes(0x5a)
    lh.synchronize()

    def row(m):
        out = np.empty(N, np.float32)
        lh._lib.call("lava_hip_memcpy_d2h", out.ctypes.data, Y.ptr + 4 * m * N, out.nbytes)
        return out

    seen = [0, 1, M // 2, M - 2, M - 1]
    try:
        if rows * N >= 2 ** 32:
            with pytest.raises(lh.Unsupported, match="w8a16_generic_kernel"):
                lh.w8a16(Y, X, W, S)
            lh.synchronize()
            assert all((row(m).view(np.uint32) == 0x5a5a5a5a).all() for m in seen)
        else:
            lh.w8a16(Y, X, W, S)
            lh.synchronize()
            for m in seen:
                np.testing.assert_array_equal(row(m), (x[m] @ w).astype(np.float32))
    finally:
        for a in (X, W, S, Y):
            a.close()
