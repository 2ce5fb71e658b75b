"""Plans whose offsets are none: what an experts' layer writes, and that it writes nothing else."""
import numpy as np
import pytest

import w8a8_reference as ref
from conftest import announce
from test_gpu_moe import experts_case
from test_gpu_w8a8 import FILL, choice, untouched, up  # noqa: F401

pytestmark = pytest.mark.gpu

BAD_OFFSETS = {
    "far outside": [0, -5, 2 ** 31 - 1, 10, -2 ** 31, 3, 2 ** 31 - 1],
    "falling": [5, 20, 20, 15, 60, 60, 200],
    "all past the end": [2 ** 31 - 1] * 7,
    "all negative": [-1] * 7,
    "a gap in front": [30, 31, 31, 40, 77, 77, 79],
}


@pytest.mark.parametrize("name", list(BAD_OFFSETS))
@pytest.mark.parametrize("sorted_", [(False, True), (True, False)])
def test_experts_of_bad_offsets_write_their_rows_alone(gpu, choice, name, sorted_):  # noqa: F811
    """Y lies inside a larger array, its rows longer than they need to be.  Offsets are cut to the rows there are: rows in no run, the
    columns behind Y's and everything in front of and behind Y stay; a row in one run is that expert's, in two either's."""
    lh = gpu
    announce(f"experts of offsets {name} sorted={sorted_}, choice {choice}")
    T, E, k, N, K, pad, guard = 40, 6, 2, 64, 128, 5, 4096
    rows = T * k
    ids, x, xs, w, ws, bias = experts_case(np.random.default_rng(62), T, E, k, N, K, masked=0.0)
    _, order = ref.plan(ids, E)
    X, W, XS, WS, B = up(lh, x), up(lh, w), up(lh, xs), up(lh, ws), up(lh, bias)
    O, R = up(lh, np.array(BAD_OFFSETS[name], np.int32)), up(lh, order)
    ld = N + pad
    all_ = lh.HIPDeviceArray("f32", (2 * guard + rows * ld,))
    all_.fill_bytes(FILL)
    layer = lh.w8_layer_raw(W.ptr, WS.ptr, N, K, K, bias=B.ptr, experts=E, expert_stride=N * K)
    lh.experts_w8a8_raw(lh.moe_plan_raw(T, E, k, O.ptr, R.ptr), layer, X.ptr, XS.ptr, K, "f32", all_.ptr + 4 * guard, ld,
                        x_sorted=sorted_[0], y_sorted=sorted_[1])
    lh.synchronize()
    got = all_.to_numpy()
    assert untouched(got[:guard]) and untouched(got[guard + rows * ld:])
    got = got[guard:guard + rows * ld].reshape(rows, ld)
    assert untouched(got[:, N:])

    runs = [[] for _ in range(rows)]      # of each place of the plan, the experts whose run has it
    cut = np.clip(np.array(BAD_OFFSETS[name], np.int64), 0, rows)
    for e in range(E):
        for at in range(cut[e], max(cut[e + 1], cut[e])):
            runs[at].append(e)
    for at in range(rows):
        src, dst = at if sorted_[0] else order[at] // k, at if sorted_[1] else order[at]
        if not runs[at]:
            assert untouched(got[dst])
            continue
        fits = np.zeros(N, bool)
        for e in runs[at]:
            y, err = ref.layer(x[src:src + 1], xs[src:src + 1], w[e], ws[e], bias[e], "none", False, "f32")
            fits |= np.abs(got[dst, :N] - y[0]) <= err[0]
        assert fits.all(), f"place {at}, experts {runs[at]}"
