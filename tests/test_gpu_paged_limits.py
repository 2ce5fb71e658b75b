"""Attention over the paged cache and appends to it at the limits of sizes: page tables far wider than the sequences are long,
more tokens than a launch has workgroups in one dimension, batches that grow step by step."""
import numpy as np
import pytest

from conftest import announce
from paged_reference import Case, bad, to_f64
from test_gpu_paged_attn import Device

pytestmark = pytest.mark.gpu


def pinned_run(lh, dev, kernel):
    lh.set_kernel_override(lh.FAMILY_PAGED, kernel)
    try:
        dev.clear()
        lh.kernel_log_clear()
        dev.launch()
        log = lh.kernel_log()
        lh.synchronize()
    finally:
        lh.set_kernel_override(lh.FAMILY_PAGED, 0)
    return dev.result(), log


def widen(lh, dev, page, width):
    """The same batch with pages of `page` tokens, of which only those in use have memory, and `width` of them a sequence, all
    but the first none."""
    c = dev.case
    assert max(kv for _, kv in c.lens) <= c.page and c.prefix <= c.page
    table = np.full((c.B, width), -1, np.int32)
    table[:, 0] = c.table[:, 0]
    dev.cache = lh.paged_cache_raw(c.dtype, dev.k.ptr, dev.v.ptr, c.D, page, c.Hkv, c.pages, c.cache_strides)
    dev.table = lh.HIPDeviceArray.from_numpy(table.ravel(), "i32")
    dev.batch = lh.paged_batch_raw(c.B, c.T, dev.q_start.ptr, dev.kv_len.ptr, dev.table.ptr, width,
                                   max_q=max(n for n, _ in c.lens))


WIDE = {   # (case, kernel pin, kernels that have to run)
    "rows": (dict(lens=tuple((1, 1 + i % 37) for i in range(70)), Hq=32, Hkv=32, D=64), 0, ["paged_rows_kernel"]),
    "rows_slopes": (dict(lens=tuple((1 + i % 3, 4 + i % 137) for i in range(70)), Hq=64, Hkv=32, D=64, slopes=True), 2,
                    ["paged_rows_kernel"]),
    "tiles": (dict(lens=tuple((40, 40 + i % 137) for i in range(70)), Hq=64, Hkv=32, D=64, dtype="bf16"), 0,
              ["paged_tile_kernel"]),
    "tiles_128": (dict(lens=tuple((40, 40 + i % 137) for i in range(70)), Hq=32, Hkv=32, D=64, cap=20.0), 4,
                  ["paged_tile_kernel", "paged_tile_kernel<32>"]),
    "shared": (dict(lens=tuple((1, 1 + i % 37) for i in range(70)), prefix=300, Hq=64, Hkv=32, D=64, slopes=True), 0,
               ["paged_tile_kernel", "paged_rows_kernel", "paged_join_kernel"]),
    # more blocks of rows than can be counted with one head: all on whole tiles
    "many_rows": (dict(lens=tuple((1, 1 + i % 37) for i in range(300)), Hq=6, Hkv=3, D=64), 0, ["paged_tile_kernel"]),
    "many_rows_shared": (dict(lens=tuple((1, 1 + i % 37) for i in range(300)), Hq=6, Hkv=3, D=128, prefix=300, window=200), 0,
                         ["paged_tile_kernel"]),
    "shared_rows": (dict(lens=tuple((1, 1 + i % 37) for i in range(70)), prefix=300, Hq=64, Hkv=32, D=64), 2,
                    ["paged_rows_kernel", "paged_join_kernel"]),
}


@pytest.mark.parametrize("name", list(WIDE))
def test_tables_as_wide_as_a_sequence_may_be(gpu, name):
    """2^30 tokens of table a sequence, some hundred in use: the MFMA kernels run, and give the bits of a narrow table."""
    kw, kernel, names = WIDE[name]
    announce(f"wide table {name}")
    case = Case(seed=41, page=512, **kw)
    dev = Device(gpu, case)
    (got, lse, raw), log = pinned_run(gpu, dev, kernel)
    want, wlse, bound, lbound = case.reference()
    assert not bad(got, want, bound).any() and not bad(lse, wlse, lbound).any()
    widen(gpu, dev, 1 << 15, 1 << 15)
    (got, lse, _), log = pinned_run(gpu, dev, kernel)
    assert "paged_any_kernel" not in log and all(k in log for k in names), log
    off = bad(got, want, bound)
    assert not off.any(), (np.argwhere(off)[:5], got[off][:5], want[off][:5])
    assert not bad(lse, wlse, lbound).any()


def test_append_more_tokens_than_a_launch_has_threads(gpu):
    """2^24 + 3 tokens, 256 threads each in the kernel: every query turned, the last keys stored."""
    lh = gpu
    announce("append 2^24 + 3 tokens")
    T, D, page = (1 << 24) + 3, 8, 64
    x = np.arange(T * D, dtype=np.uint32).reshape(T, D) % 1024
    x = (x.astype(np.float32) / 512 - 1).astype(np.float16)
    X = lh.HIPDeviceArray.from_numpy(x.ravel(), "f16")
    O = lh.HIPDeviceArray("f16", (T * D,))
    O.fill_bytes(0x5a)
    up = lambda a, t: lh.HIPDeviceArray.from_numpy(np.asarray(a, np.int32 if t == "i32" else np.float32), t)
    QS, KL, TB = up([0, T], "i32"), up([128], "i32"), up([1, 0], "i32")
    F = up([1.0, 0.1, 0.01, 0.001], "f32")
    for rot, kernel in ((8, "kv_append_kernel"), (6, "kv_append_any_kernel")):
        K, V = (lh.HIPDeviceArray("f16", (2 * page * D,)) for _ in range(2))
        K.fill_bytes(0x5a)
        V.fill_bytes(0x5a)
        cache = lh.paged_cache_raw("f16", K.ptr, V.ptr, D, page, 1, 2, (1, D, page * D, page * D))
        lh.kernel_log_clear()
        lh.kv_append_raw(cache, lh.paged_batch_raw(1, T, QS.ptr, KL.ptr, TB.ptr, 2), X.ptr, X.ptr, (1, D, D), Q=X.ptr,
                         Q_out=O.ptr, q_heads=1, q_strides=(1, D, D), qo_strides=(1, D, D),
                         rope=lh.rope_raw(F.ptr, rot, interleaved=True))
        assert lh.kernel_log() == [kernel]
        lh.synchronize()
        got = O.to_numpy().reshape(T, D)

        def turned(t):
            a = (128 - T + t)[:, None] * np.array([1.0, 0.1, 0.01, 0.001], np.float32).astype(np.float64)[None, :rot // 2]
            r = x[t].astype(np.float64)
            o = r.copy()
            o[:, 0:rot:2] = r[:, 0:rot:2] * np.cos(a) - r[:, 1:rot:2] * np.sin(a)
            o[:, 1:rot:2] = r[:, 1:rot:2] * np.cos(a) + r[:, 0:rot:2] * np.sin(a)
            return o
        # each off by half a step of its own size (below 1.5) and 2^-21 of the pair's
        t = np.concatenate([np.arange(0, T, 4099), np.arange(T - 200, T)])
        want = turned(t)
        assert (np.abs(got[t].astype(np.float64) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20 + 2.0 ** -25).all()
        bits = got.view(np.uint16).reshape(T, D)
        assert not (bits == 0x5a5a).all(axis=1).any()   # no row left out
        last = np.arange(T - 128, T)
        for cached, rows, exact in ((K, turned(last), False), (V, x[last].astype(np.float64), True)):
            c = cached.to_numpy().reshape(2, page, D)[[1, 0]].reshape(128, D).astype(np.float64)
            assert (np.abs(c - rows) <= (0 if exact else 2.0 ** -11 * np.abs(rows) + 2.0 ** -20 + 2.0 ** -25)).all()


def test_generic_attention_of_more_rows_than_a_launch_has_threads(gpu):
    """2^26 + 64 rows, a wavefront each: D = 1, 64 heads, three keys."""
    lh = gpu
    announce("generic attention of 2^26 + 64 rows")
    T, H = (1 << 20) + 1, 64
    rng = np.random.default_rng(42)
    q = (rng.integers(-8, 9, (T, H)) / 4).astype(np.float16)
    k, v = (rng.standard_normal(3).astype(np.float16) for _ in range(2))
    Q, K, V = (lh.HIPDeviceArray.from_numpy(a.ravel(), "f16") for a in (q, k, v))
    O = lh.HIPDeviceArray("f16", (T * H,))
    O.fill_bytes(0x5a)
    up = lambda a: lh.HIPDeviceArray.from_numpy(np.asarray(a, np.int32), "i32")
    QS, KL, TB = up([0, T]), up([3]), up([0])
    cache = lh.paged_cache_raw("f16", K.ptr, V.ptr, 1, 3, 1, 1, (1, 1, 3, 3))
    lh.kernel_log_clear()
    lh.paged_attn_raw(cache, lh.paged_batch_raw(1, T, QS.ptr, KL.ptr, TB.ptr, 1), lh.attn_score_raw(1.0, causal=False),
                      Q.ptr, O.ptr, H, (1, 1, H), (1, 1, H))
    assert lh.kernel_log() == ["paged_any_kernel"]
    lh.synchronize()
    got = O.to_numpy().reshape(T, H)
    x = np.arange(-8, 9) / 4   # the 17 queries there are
    e = np.exp(x[:, None] * k.astype(np.float64)[None])
    want = (e @ v.astype(np.float64)) / e.sum(1)
    size = (e @ np.abs(v.astype(np.float64))) / e.sum(1)
    i = (q * 4).astype(np.int32) + 8
    # scores are off by 2^-21 at most (|s| < 8), the result by half a step
    assert (np.abs(got - want[i]) <= 2.0 ** -11 * np.abs(want[i]) + 2.0 ** -19 * size[i] + 2.0 ** -25).all()


def test_tile_launches_of_more_workgroups_than_one_dimension_has(gpu):
    """2^28 tokens are announced, some hundred are there: tiles beyond them have no rows, and none runs twice."""
    announce("tile launch of 2^23 and more workgroups")
    case = Case(lens=((150, 150), (33, 133), (64, 64)), Hq=4, Hkv=1, D=64, seed=43)
    dev = Device(gpu, case)
    want, wlse, bound, lbound = case.reference()
    dev.batch = gpu.paged_batch_raw(case.B, 1 << 28, dev.q_start.ptr, dev.kv_len.ptr, dev.table.ptr, case.max_pages, max_q=150)
    (got, lse, _), log = pinned_run(gpu, dev, 4)
    assert log[0] == "paged_tile_kernel", log
    assert not bad(got, want, bound).any() and not bad(lse, wlse, lbound).any()


def test_a_growing_batch_allocates_few_workspaces(gpu):
    """A batch that grows by a token a step: the stream's workspace grows by factors, not with every step (each outgrown buffer
    is kept for work that is still queued)."""
    lh = gpu
    announce("a growing batch behind a shared prefix")
    n = 64
    case = Case(lens=tuple((1, 1 + i % 5) for i in range(n)), prefix=40, Hq=32, Hkv=8, D=128, seed=44, tail=0)
    dev = Device(lh, case)
    want, _, bound, _ = case.reference()
    s = lh.Stream()
    grown = []
    for b in range(1, n + 1):
        dev.batch = lh.paged_batch_raw(b, b, dev.q_start.ptr, dev.kv_len.ptr, dev.table.ptr, case.max_pages, max_q=1)
        lh.kernel_log_clear()
        dev.launch(stream=s.handle)
        grown.append(lh.kernel_log().count("fill_bytes_kernel"))   # a new workspace's counters cleared
    s.synchronize()
    need = [lh.paged_workspace_bytes(dev.cache, lh.paged_batch_raw(b, b, dev.q_start.ptr, dev.kv_len.ptr, dev.table.ptr,
                                                                   case.max_pages, max_q=1), case.Hq, case.prefix) for b in (1, n)]
    assert sum(grown) <= 2 + np.log(need[1] / need[0]) / np.log(1.5), (sum(grown), need)
    assert not bad(dev.result()[0], want, bound).any()
    s.close()


def test_a_captured_step_of_a_batch_with_its_own_workspace(gpu):
    """A decode step captured on a fresh stream, which has no workspace yet: replayed beside eager calls on that stream."""
    lh = gpu
    announce("a captured step with its own workspace")
    D, page, Hkv, Hq, B = 64, 16, 2, 8, 3
    rng = np.random.default_rng(45)
    lens = np.array([200, 17, 90], np.int32)
    cache = lh.PagedCache("f16", D, page, Hkv, 30)
    for a in (cache.k, cache.v):
        a.copy_from(rng.standard_normal(a.dims).astype(np.float16))
    table = np.full((14, B), -1, np.int32, order="F")
    table[:, 0] = rng.permutation(14)
    table[:6, 1:] = 14 + rng.permutation(12).reshape(6, 2)
    i32 = lambda a: lh.HIPDeviceArray.from_numpy(np.asarray(a, np.int32), "i32")
    batch = lh.PagedBatch(B, i32(np.arange(B + 1)), i32(lens), lh.HIPDeviceArray.from_numpy(table, "i32"), max_q=1)
    Q = lh.HIPDeviceArray.from_numpy(np.asfortranarray(rng.standard_normal((D, Hq, B)).astype(np.float16)), "f16")
    O, P = (lh.HIPDeviceArray("f16", (D, Hq, B)) for _ in range(2))
    lh.paged_attn(P, cache, batch, Q)
    lh.synchronize()
    want = P.to_numpy()
    s = lh.Stream()
    g = lh.Graph(s)
    assert batch.own_workspace(cache, Hq) is batch
    with g.capture():
        lh.paged_attn(O, cache, batch, Q, stream=s.handle)
    for _ in range(4):
        O.fill_bytes(0x5a)
        lh.synchronize()
        g.launch()
        s.synchronize()
        assert (O.to_numpy().view(np.uint16) == want.view(np.uint16)).all()
        lh.paged_attn(P, cache, batch, Q, stream=s.handle)
        s.synchronize()
        assert (P.to_numpy().view(np.uint16) == want.view(np.uint16)).all()
    g.close()
    s.close()
    cache.close()
