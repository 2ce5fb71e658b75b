"""Routing where scores saturate or tie."""
import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce
from test_gpu_moe import check_route, route
from test_gpu_w8a8 import up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2), (3, 2, 2)])
def test_route_by_logits_whose_scores_are_equal_in_64_bits(gpu, dtype, score, groups, top, best):
    """Sigmoids of 38 and more are 1 in 64 bits, and a softmax 800 below the highest is 0: without a bias single experts go by their
    logits, however groups are counted."""
    lh = gpu
    announce(f"route saturated {score} {dtype} {groups} {top} {best}")
    rng = np.random.default_rng(60)
    T, E, k = 90, 48, 10
    size = E // groups
    # whole numbers, all different in a row; groups differ by a logit near zero each (a sigmoid's best two, a softmax's top)
    x = np.argsort(rng.random((T, E)), axis=1) + 40.0
    if score == "softmax":
        x = -900.0 - 4 * x
        x[np.arange(T), rng.integers(0, E, T)] = 0.0
    if groups > 1:
        x = x.reshape(T, groups, size)
        if score == "sigmoid" and best == 2:
            # in all groups but two only one is high, so that the counts differ
            low = np.argsort(rng.random((T, groups)), axis=1)[:, :groups - 2]
            for t in range(T):
                for g in low[t]:
                    x[t, g, 1:] = -5.0 - np.arange(size - 1) - g * 0.125
        x = x.reshape(T, E)
    store = ref.to_store(x, dtype)
    r = lh.MoeRouter(E, k, score, None, groups, top, best)
    check_route(route(lh, store, dtype, r), store, dtype, k, score=score, groups=groups, top_groups=top, group_best=best)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", ["none", "zero", "random"])
@pytest.mark.parametrize("E,k,groups,top,best", [(256, 8, 8, 4, 2), (64, 8, 1, 1, 1), (96, 6, 4, 2, 2)])
def test_route_of_16_bit_logits(gpu, dtype, score, bias, E, k, groups, top, best):
    """Logits of 16 bits, many of them equal, on the paths that compare scores."""
    lh = gpu
    announce(f"route 16-bit logits {dtype} {score} bias {bias} {k} of {E}")
    rng = np.random.default_rng(61)
    store = ref.to_store(rng.standard_normal((200, E)) * 1.5, dtype)
    b = {"none": None, "zero": np.zeros(E, np.float32), "random": (rng.standard_normal(E) * 0.1).astype(np.float32)}[bias]
    r = lh.MoeRouter(E, k, score, up(lh, b) if b is not None else None, groups, top, best)
    check_route(route(lh, store, dtype, r), store, dtype, k, score=score, bias=b, groups=groups, top_groups=top, group_best=best)
