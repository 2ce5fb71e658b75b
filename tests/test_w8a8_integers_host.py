"""Integers that the descriptors and calls of the layers and of the paged cache would cut off, on the host."""
import pytest

import lava_hip as lh

A = 1 << 20


@pytest.mark.parametrize("n", [-1, 2 ** 64, -2 ** 63])
def test_workspaces_of_lengths_that_are_none(n):
    """-1 would be the largest size there is and pass for a workspace of any length."""
    with pytest.raises(ValueError, match="workspace_bytes"):
        lh.moe_plan_raw(5000, 8, 2, A, A, A, n)
    with pytest.raises(ValueError, match="workspace_bytes"):
        lh.paged_batch_raw(1, 1, A, A, A, 1, workspace=A, workspace_bytes=n)


def test_workspaces_up_to_the_largest_length():
    for n in (0, 5, 2 ** 63, 2 ** 64 - 1):
        assert lh.moe_plan_raw(5000, 8, 2, A, A, A, n).workspace_bytes == n
        assert lh.paged_batch_raw(1, 1, A, A, A, 1, workspace=A, workspace_bytes=n).workspace_bytes == n


CUT = 2 ** 64   # 0 in 64 bits: a call of no tokens, which has nothing to do and refuses nothing


@pytest.mark.parametrize("hides", [-1, -2 ** 63, 1])
def test_a_cut_off_integer_beside_a_negative_one(hides):
    """A negative integer's bits, put together with those that are cut off, look like a number that fits."""
    with pytest.raises(ValueError, match="tokens"):
        lh.quantize_i8_raw("f16", A, A, A, 64, CUT, hides, 64)
    with pytest.raises(ValueError, match="tokens"):
        lh.w8a8_raw(lh.w8_layer_raw(A, A, 64, 128, 128), A, A, CUT, hides, "f16", A, 64)
    with pytest.raises(ValueError, match="tokens"):
        lh.moe_route_raw(lh.moe_router_raw(8, 2), "f32", A, hides, CUT, A, A)
    with pytest.raises(ValueError, match="tokens"):
        lh.moe_combine_raw("f32", A, hides, A, A, CUT, 2, 64, A, 64)
    with pytest.raises(ValueError, match="top_k"):
        lh.moe_combine_raw("f32", A, hides, A, A, 0, 2 ** 32, 64, A, 64)
    with pytest.raises(ValueError, match="ldy"):
        lh.experts_w8a8_raw(lh.moe_plan_raw(0, 4, 2, 0, 0), lh.w8_layer_raw(0, 0, 0, 0, 0, experts=4), 0, 0, hides, "f16", 0, CUT)


@pytest.mark.parametrize("x", [-2 ** 63, 2 ** 63 - 1])
def test_integers_that_just_fit(x):
    """They reach the library, whose refusal names them."""
    lh.quantize_i8_raw("f16", A, A, A, 64, 0, x, x)
    with pytest.raises(lh.InvalidArgument if x < 0 else lh.Unsupported, match="tokens"):
        lh.w8a8_raw(lh.w8_layer_raw(A, A, 64, 128, 128), A, A, x, 128, "f16", A, 64)
