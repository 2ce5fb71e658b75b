"""Launches of 2^32 threads and more: sums of experts' rows and rows of no values are refused by name, the largest below them right."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_w8a8 import FILL, untouched, up

pytestmark = pytest.mark.gpu

T = 2 ** 24


def test_combine_of_the_most_tokens(gpu):
    lh = gpu
    announce(f"combine {T} tokens of 1")
    Y, W, O = lh.HIPDeviceArray("f16", (T,)), lh.HIPDeviceArray("f32", (T,)), lh.HIPDeviceArray("f16", (T,))
    try:
        Y.fill_bytes(0x3c)
        W.fill_bytes(0x3f)
        O.fill_bytes(FILL)
        lh.synchronize()
        with pytest.raises(lh.Unsupported, match="moe_combine"):
            lh.moe_combine_raw("f16", Y.ptr, 1, 0, W.ptr, T, 1, 1, O.ptr, 1)
        lh.synchronize()
        assert untouched(O.to_numpy())
        lh.moe_combine_raw("f16", Y.ptr, 1, 0, W.ptr, T - 1, 1, 1, O.ptr, 1)
        lh.synchronize()
        got = O.to_numpy()
    finally:
        for a in (Y, W, O):
            a.close()
    y, w = np.array([0x3c3c], np.uint16).view(np.float16)[0], np.array([0x3f3f3f3f], np.uint32).view(np.float32)[0]
    assert (got[:-1] == np.float16(np.float64(y) * np.float64(w))).all() and untouched(got[-1:])


def test_quantize_the_most_rows_of_nothing(gpu):
    lh = gpu
    announce(f"quantize {T} rows of 0")
    S = lh.HIPDeviceArray("f32", (T,))
    try:
        S.fill_bytes(FILL)
        lh.synchronize()
        with pytest.raises(lh.Unsupported, match="quantize_kernel"):
            lh.quantize_i8_raw("f16", 0, 0, S.ptr, 0, T, 0, 0)
        lh.synchronize()
        assert untouched(S.to_numpy())
        lh.quantize_i8_raw("f16", 0, 0, S.ptr, 0, T - 1, 0, 0)
        lh.synchronize()
        got = S.to_numpy()
    finally:
        S.close()
    assert not got[:-1].any() and untouched(got[-1:])


def test_ids_past_the_experts_are_read_where_no_plan_knows_them(gpu):
    """A plan leaves out any id that is no expert; the sum, which does not know how many there are, only negative ones."""
    lh = gpu
    announce("ids past the experts")
    ids = np.array([[0, 9], [-1, 1]], np.int32)
    p, I = lh.MoePlan(2, 2, 2), up(lh, ids)
    lh.moe_sort(p, I)
    O, Y, W = lh.HIPDeviceArray("f32", (8, 2)), up(lh, np.arange(4, dtype=np.float32).repeat(8).reshape(4, 8) + 1), up(lh, np.ones((2, 2), np.float32))
    lh.moe_combine(O, Y, W, I)
    lh.synchronize()
    assert p.offsets.to_numpy().tolist() == [0, 1, 2] and p.order.to_numpy().tolist() == [0, 3, -1, -1]
    assert (O.to_numpy() == np.array([1 + 2, 4])).all()
