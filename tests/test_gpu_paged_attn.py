"""Attention over the paged cache, by kernel, against softmax in 64 bits with derived bounds (paged_reference)."""
import numpy as np
import pytest

from conftest import announce
from paged_reference import Case, bad, to_f64

pytestmark = pytest.mark.gpu

KERNELS = {1: "paged_any_kernel", 2: "paged_rows_kernel", 3: "paged_tile_kernel", 4: "paged_tile_kernel"}


class Device:
    """A case's arrays on the GPU and its descriptors; `call` runs it and gives (O, lse, raw O)."""

    def __init__(self, lh, case, max_q=None, table=None, ppages=None):
        self.lh, self.case = lh, case
        d = {"f16": "f16", "bf16": "bf16"}[case.dtype]
        up = lambda a, t: lh.HIPDeviceArray.from_numpy(np.ascontiguousarray(a).ravel(), t)
        self.q, self.k, self.v = up(case.q, d), up(case.k, d), up(case.v, d)
        self.q_start, self.kv_len = up(case.q_start, "i32"), up(case.kv_len, "i32")
        self.table = up(case.table if table is None else table, "i32")
        pp = case.ppages if ppages is None else ppages
        self.ppages = up(pp if len(pp) else np.zeros(1, np.int32), "i32")
        self.slope = up(case.slope, "f32") if case.slope is not None else None
        self.bid = up(case.bid, "i32") if case.bid is not None else None
        self.o = lh.HIPDeviceArray(d, (max(1, case.T * case.Hq * case.D),))
        self.lse = lh.HIPDeviceArray("f32", (max(1, case.T * case.Hq),))
        self.cache = lh.paged_cache_raw(d, self.k.ptr, self.v.ptr, case.D, case.page, case.Hkv, case.pages,
                                        case.cache_strides)
        mq = max(n for n, _ in case.lens) if max_q is None else max_q
        self.batch = lh.paged_batch_raw(case.B, case.T, self.q_start.ptr, self.kv_len.ptr, self.table.ptr,
                                        case.max_pages, max_q=mq)
        self.score = lh.attn_score_raw(case.scale, case.causal, case.window, case.cap,
                                       self.slope.ptr if self.slope else 0, self.bid.ptr if self.bid else 0)
        self.packed = (1, case.D, case.Hq * case.D)

    def launch(self, stream=None, lse=True):
        c = self.case
        lp = self.lse.ptr if lse else 0
        if c.prefix:
            self.lh.shared_prefix_attn_raw(self.cache, self.batch, self.score, self.ppages.ptr, c.prefix, self.q.ptr,
                                           self.o.ptr, c.Hq, self.packed, self.packed, lp, stream)
        else:
            self.lh.paged_attn_raw(self.cache, self.batch, self.score, self.q.ptr, self.o.ptr, c.Hq, self.packed,
                                   self.packed, lp, stream)

    def result(self):
        c = self.case
        o = self.o.to_numpy().reshape(c.T, c.Hq, c.D)
        return to_f64(o, c.dtype), self.lse.to_numpy().reshape(c.T, c.Hq).astype(np.float64), o

    def clear(self):
        self.o.fill_bytes(0x5a)
        self.lse.fill_bytes(0x5a)


def check(lh, case, kernel, dead=(), **more):
    announce(f"paged attention kernel={kernel} {({k: v for k, v in case.__dict__.items() if k in ARGS})} {more}")
    dev = Device(lh, case, **more)
    lh.set_kernel_override(lh.FAMILY_PAGED, kernel)
    try:
        for _ in range(2):   # twice: a call leaves nothing behind that the next one trips over
            dev.clear()
            lh.kernel_log_clear()
            dev.launch()
            log = lh.kernel_log()
            lh.synchronize()
            got, lse, raw = dev.result()
    finally:
        lh.set_kernel_override(lh.FAMILY_PAGED, 0)
    if kernel:
        assert log[0] == (KERNELS[kernel] if kernel < 3 or case.D <= 128 else KERNELS[2]), log
    want, wlse, bound, lbound = case.reference(dead=dead)
    off = bad(got, want, bound)
    assert not off.any(), (np.argwhere(off)[:5], got[off][:5], want[off][:5], bound[off][:5])
    off = bad(lse, wlse, lbound)
    assert not off.any(), (np.argwhere(off)[:5], lse[off][:5], wlse[off][:5], lbound[off][:5])
    # rows of no sequence are as they were
    free = np.isnan(wlse)
    assert (raw.view(np.uint16)[free] == 0x5a5a).all()
    return got


ARGS = ("dtype", "Hq", "Hkv", "D", "page", "order", "lens", "causal", "window", "cap", "slopes", "bidir", "prefix",
        "gap", "tail")
RAGGED = ((1, 1), (1, 2), (0, 7), (1, 15), (1, 16), (1, 17), (1, 31), (1, 33), (1, 127), (1, 128), (1, 129), (1, 300))
CASES = {
    "one_token": dict(lens=((1, 1),)),
    "decode_ragged": dict(lens=RAGGED, Hq=8, Hkv=2, D=128),
    "decode_bf16": dict(lens=RAGGED, Hq=8, Hkv=2, D=128, dtype="bf16", order="lh"),
    "decode_d64": dict(lens=RAGGED, Hq=3, Hkv=3, D=64, page=32),
    "decode_d80": dict(lens=RAGGED, Hq=14, Hkv=2, D=80, page=24),
    "decode_d256": dict(lens=RAGGED, Hq=4, Hkv=1, D=256, page=16, dtype="bf16"),
    "decode_d8": dict(lens=RAGGED, Hq=4, Hkv=1, D=8, page=8),
    "wide_groups": dict(lens=((1, 90), (2, 70), (0, 0), (1, 0)), Hq=40, Hkv=2, D=64),
    "few_tokens": dict(lens=((4, 100), (3, 3), (1, 64), (4, 129)), Hq=8, Hkv=2, D=128, gap=3, tail=5),
    "no_keys": dict(lens=((1, 0), (2, 0), (0, 0), (1, 5))),
    "more_new_than_cached": dict(lens=((5, 3), (9, 0), (4, 4)), Hq=4, Hkv=4),
    "prompt": dict(lens=((150, 150), (33, 33), (64, 64), (65, 65)), Hq=4, Hkv=2, D=128),
    "prompt_bf16_d64": dict(lens=((150, 150), (257, 257)), Hq=2, Hkv=2, D=64, dtype="bf16", order="lh"),
    "chunk": dict(lens=((70, 300), (1, 200), (130, 131)), Hq=6, Hkv=2, D=64, page=64),
    "chunk_all_keys": dict(lens=((70, 300), (1, 200), (130, 131)), Hq=4, Hkv=2, D=128, causal=False),
    "window": dict(lens=((1, 300), (40, 200), (3, 20), (1, 33)), window=33, Hq=4, Hkv=2, D=128),
    "window_one": dict(lens=((1, 300), (40, 200), (3, 20)), window=1),
    "window_all_keys": dict(lens=((1, 300), (40, 200), (3, 20)), window=50, causal=False),
    "cap": dict(lens=((1, 300), (40, 200), (3, 20)), cap=2.0, Hq=8, Hkv=2, D=128, q_size=3.0),
    "cap_bf16": dict(lens=((1, 300), (40, 200), (3, 20)), cap=30.0, dtype="bf16", D=64, q_size=3.0),
    "slopes": dict(lens=((1, 300), (40, 200), (3, 20)), slopes=True, Hq=8, Hkv=2, D=64),
    "slopes_window_cap": dict(lens=((1, 300), (40, 200), (3, 20)), slopes=True, window=77, cap=5.0, Hq=8, Hkv=2, D=128,
                              dtype="bf16"),
    "bidirectional": dict(lens=((100, 100), (40, 200), (3, 20), (50, 50)), bidir=[40, 300, 0, 1], Hq=4, Hkv=2, D=64),
    "bidirectional_window": dict(lens=((100, 100), (40, 200), (3, 20)), bidir=[60, 190, 20], window=40, slopes=True),
    "negative_scale": dict(lens=((1, 200), (20, 40)), scale=-0.2),
    "zero_scale": dict(lens=((1, 200), (20, 40)), scale=0.0),
    "large_scores": dict(lens=((1, 200), (20, 40)), scale=3.0, q_size=8.0, dtype="bf16"),
    "shared": dict(lens=((1, 1), (1, 40), (2, 9), (0, 5), (1, 130)), prefix=100, Hq=8, Hkv=2, D=128),
    "shared_bf16": dict(lens=((1, 1), (1, 40), (4, 9), (1, 130)), prefix=256, Hq=4, Hkv=4, D=64, dtype="bf16", page=32),
    "shared_window": dict(lens=((1, 1), (1, 40), (4, 9), (1, 130)), prefix=200, window=60, slopes=True, cap=8.0, Hq=4,
                          Hkv=1, D=128),
    "shared_own_empty": dict(lens=((1, 0), (1, 1), (2, 0)), prefix=77, Hq=4, Hkv=2, D=64),
    "shared_long_rows": dict(lens=((90, 90), (1, 4), (17, 30)), prefix=133, Hq=4, Hkv=2, D=128, order="lh"),
    "shared_all_keys": dict(lens=((9, 12), (1, 4)), prefix=70, causal=False, D=256, Hq=2, Hkv=1),
    # more blocks of work than workgroups: parts of several blocks, sequences that share a workgroup and that are split
    "split_uneven": dict(lens=tuple((1, 1 + (i * 397) % 1900) for i in range(48)), Hq=16, Hkv=8, D=128),
    "split_uneven_d64": dict(lens=tuple((1 + i % 3, 4 + (i * 397) % 1900) for i in range(48)), Hq=32, Hkv=16, D=64,
                             dtype="bf16", page=40),
    "split_wide": dict(lens=tuple((9, 9 + (i * 397) % 1500) for i in range(24)), Hq=48, Hkv=8, D=128, window=700),
    "split_shared": dict(lens=tuple((1, 1 + (i * 97) % 300) for i in range(60)), prefix=1999, Hq=32, Hkv=8, D=128),
    "split_shared_window": dict(lens=tuple((1 + i % 2, 2 + (i * 97) % 300) for i in range(60)), prefix=1999, window=1200,
                                Hq=32, Hkv=8, D=64, dtype="bf16", slopes=True),
    # more keys than a wavefront finds the pages of at once (16 and 32 blocks), ends at and around them
    "long_keys": dict(lens=((1, 2047), (1, 2048), (1, 2049), (3, 4100), (70, 4200)), Hq=2, Hkv=1, D=64, page=8),
    "long_keys_one_head": dict(lens=((1, 200001),), Hq=1, Hkv=1, D=64, page=64),
    "long_prefix": dict(lens=((1, 30), (2, 2060), (40, 40)), prefix=6200, Hq=4, Hkv=2, D=64, page=24),
    "many": dict(lens=tuple((1 if i % 5 else 2, 2 + i % 37) for i in range(150)), Hq=2, Hkv=1, D=64),
}


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_attention(gpu, kernel, name):
    check(gpu, Case(seed=sum(map(ord, name)), **CASES[name]), kernel)
