"""Integers that the descriptors of the layers and of the paged cache would cut off, on the host."""
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
