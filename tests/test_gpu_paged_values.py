"""Attention over the paged cache at unusual values: caps far above the scores, values that are not finite at keys of
little weight, negative numbers of leading keys."""
import numpy as np
import pytest

from conftest import announce
from paged_reference import TINY, U, Case, bad, to_bits, to_f64
from test_gpu_paged_attn import KERNELS, Device

pytestmark = pytest.mark.gpu


def run(lh, dev, kernel):
    lh.set_kernel_override(lh.FAMILY_PAGED, kernel)
    try:
        dev.clear()
        dev.launch()
        lh.synchronize()
    finally:
        lh.set_kernel_override(lh.FAMILY_PAGED, 0)
    return dev.result()


# ---- caps -------------------------------------------------------------------------------------------------------

def capped(case):
    """O of a causal capped case in 64 bits and its bound.  As paged_reference's, but a score's error from the cap goes by the
    score's size, 2^-20 of it: |z| <= 1/2, z = score / cap: the polynomial's fit 2^-23.8 and its roundings, 2^-21; beyond, cap
    (1 - 2 / (1 + e^2z)) from an exponential off by 2^-22.4, a reciprocal and a sum, 2^-20.5.  (A cap of at most 88 may have that form for
    small scores too: its exponential's and reciprocal's 2^-22.1 of a term of up to 2 cap, 2^-21 of the cap.)  To first order O
    moves by sum w (v - O) ds."""
    O, bound = np.full((case.T, case.Hq, case.D), np.nan), np.full((case.T, case.Hq, case.D), np.nan)
    u = U[case.dtype]
    kp, vp = to_f64(case.keys[-1], case.dtype), to_f64(case.values[-1], case.dtype)
    for b, (n, kv) in enumerate(case.lens):
        r = slice(int(case.q_start[b]), int(case.q_start[b]) + n)
        k = np.concatenate([kp, to_f64(case.keys[b], case.dtype)])
        v = np.concatenate([vp, to_f64(case.values[b], case.dtype)])
        keep = np.arange(len(k))[None] <= (len(k) - n + np.arange(n))[:, None]
        for h in range(case.Hq):
            kh, vh = k[:, h * case.Hkv // case.Hq], v[:, h * case.Hkv // case.Hq]
            q = to_f64(case.q[r, h], case.dtype)
            raw = (q @ kh.T) * case.scale
            s = case.cap * np.tanh(raw / case.cap)
            ds = (np.abs(q) @ np.abs(kh).T) * case.scale * (case.D + 2) * 2.0 ** -24 + np.abs(s) * 2.0 ** -20 + 2.0 ** -22
            ds = ds + (case.cap * 2.0 ** -21 if case.cap <= 88 else 0)
            s = np.where(keep, s, -np.inf)
            e = np.exp(s - s.max(axis=1, keepdims=True))
            w = e / e.sum(axis=1, keepdims=True)
            o, a = w @ vh, w @ np.abs(vh)
            moved = (w * ds) @ np.abs(vh) + (w * ds).sum(axis=1, keepdims=True) * np.abs(o)
            O[r, h] = o
            bound[r, h] = 1.01 * (2 * u * a + moved + (len(k) + 8) * 2.0 ** -24 * a + u * np.abs(o) + TINY[case.dtype]
                                  + (2.0 ** -24 * (keep.astype(float) @ np.abs(vh)) if case.dtype == "f16" else 0))
    return O, bound


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("cap", [50.0, 1e4, 1e6, 1e9, 1e20, 3e38])
def test_caps_far_above_the_scores(gpu, kernel, cap):
    """cap tanh(s / cap) is s there, to 32 bits: no cap may cost a score its last places."""
    announce(f"cap {cap} kernel={kernel}")
    case = Case(lens=((1, 300), (40, 200), (3, 20)), cap=cap, Hq=4, Hkv=2, D=64, q_size=2.0, seed=31, prefix=0)
    dev = Device(gpu, case)
    got, _, _ = run(gpu, dev, kernel)
    want, bound = capped(case)
    off = bad(got, want, bound)
    assert not off.any(), (np.argwhere(off)[:4], got[off][:4], want[off][:4], bound[off][:4])


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("prefix", [0, 90])
@pytest.mark.parametrize("cap", [3.0, 1e7])
def test_capped_scores_of_all_sizes_in_one_block(gpu, kernel, prefix, cap):
    """Every few keys one whose score is beyond half the cap among others far below it: of either sign, or (where only rows
    without a large positive score can show an error of the others) negative."""
    announce(f"capped scores of all sizes cap={cap} kernel={kernel} prefix={prefix}")
    case = Case(dtype="bf16", lens=((1, 300), (40, 200), (3, 20)), cap=cap, Hq=4, Hkv=2, D=64, seed=32, prefix=prefix)
    if cap > 100:
        case.q = to_bits(np.abs(to_f64(case.q, "bf16")), "bf16")
    for b in (0, 1, 2, -1):
        x = to_f64(case.keys[b], "bf16")
        if cap > 100:
            x[5::23] = -cap
        else:
            x[5::23] *= 2 * cap
        case.keys[b] = to_bits(x, "bf16")
        case.put(case.k, b, case.keys[b])
    dev = Device(gpu, case)
    got, _, _ = run(gpu, dev, kernel)
    want, bound = capped(case)
    off = bad(got, want, bound)
    assert not off.any(), (np.argwhere(off)[:4], got[off][:4], want[off][:4], bound[off][:4])


# ---- values that are not finite -----------------------------------------------------------------------------------

FAINT = {
    "decode": dict(lens=((3, 40), (5, 150)), Hq=4, Hkv=2, D=64),
    "prompt": dict(lens=((90, 200), (64, 70)), Hq=4, Hkv=2, D=128),
    "window": dict(lens=((90, 200), (5, 150)), Hq=4, Hkv=1, D=128, window=60),
    "bf16": dict(lens=((90, 200), (5, 150)), Hq=4, Hkv=2, D=64, dtype="bf16"),
    "d256": dict(lens=((40, 200), (5, 150)), Hq=2, Hkv=1, D=256),
    "shared": dict(lens=((3, 9), (4, 8), (90, 100)), prefix=150, window=120, Hq=4, Hkv=2, D=64),
}


@pytest.mark.parametrize("name", list(FAINT))
@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_values_that_are_not_finite_at_keys_of_little_weight(gpu, kernel, name):
    """A key whose weight is below the operands' smallest numbers, in a block that only some rows see whole: every row that sees
    it is not finite in the columns where its values are not, the others do not notice it."""
    announce(f"not finite values of little weight kernel={kernel} {name}")
    case = Case(seed=33, **FAINT[name])
    case.q = to_bits(np.abs(to_f64(case.q, case.dtype)) + 0.5, case.dtype)
    at = []
    for b, (n, kv) in enumerate(case.lens):
        j = kv - 1 - n // 2   # the later half of the new tokens sees it
        at.append(j)
        # a score 30 below the others in f16 (weight 2^-43), 110 in bf16 (2^-159)
        low = -{"f16": 30.0, "bf16": 110.0}[case.dtype] / (1.3 * case.D * case.scale)
        x = to_f64(case.keys[b], case.dtype) * 0.1
        x[j] = low
        case.keys[b] = to_bits(x, case.dtype)
        case.put(case.k, b, case.keys[b])
        case.values[b][j, :, 1:4] = 0
        bits = case.values[b].copy()
        bits[j, :, 1:4] = to_bits(np.array([np.inf, -np.inf, np.nan]), case.dtype)
        case.put(case.v, b, bits)
    got, _, _ = run(gpu, Device(gpu, case), kernel)
    want, _, bound, _ = case.reference()
    seen = np.zeros((case.T, 1), bool)
    for b, (n, kv) in enumerate(case.lens):
        pos = kv - n + np.arange(n)
        see = (at[b] <= pos) & ((at[b] > pos - case.window) if case.window else True)
        assert see.any() and not see.all()
        seen[case.q_start[b]:case.q_start[b] + n, 0] = see
    for d in (1, 2, 3):
        ok = np.where(seen, ~np.isfinite(got[:, :, d]), True)
        assert ok.all(), (d, np.argwhere(~ok)[:5])
    rest = np.ones(got.shape, bool)
    rest[:, :, 1:4] = ~seen[:, :, None]
    off = bad(got, want, bound) & rest
    assert not off.any(), (np.argwhere(off)[:5], got[off][:5], want[off][:5])


# ---- leading keys -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_negative_numbers_of_leading_keys(gpu, kernel):
    """No key lies below them, down to the least integer: the call is a causal one."""
    announce(f"negative leading keys kernel={kernel}")
    case = Case(lens=((70, 100), (40, 200), (3, 20), (1, 50)), bidir=[-2 ** 31, -1, -2 ** 31 + 1, -2 ** 31], Hq=4, Hkv=2, D=64, seed=34)
    got, lse, _ = run(gpu, Device(gpu, case), kernel)
    want, wlse, bound, lbound = case.reference()
    assert not bad(got, want, bound).any() and not bad(lse, wlse, lbound).any()
