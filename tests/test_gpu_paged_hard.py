"""Attention over the paged cache where it is easily wrong: what masked places hold, tables and lengths that are
malformed, layouts, streams, workspaces and graphs, and the operators in the order a program runs them."""
import numpy as np
import pytest

from conftest import announce
from paged_reference import Case, bad, to_bits, to_f64
from test_gpu_paged_attn import KERNELS, Device, check

pytestmark = pytest.mark.gpu


def pinned(lh, kernel):
    lh.set_kernel_override(lh.FAMILY_PAGED, kernel)


# ---- infinities and NaN at positions that some rows see and others do not -------------------------------------

HIDDEN = {
    "causal": dict(lens=((90, 200), (3, 40), (64, 64)), Hq=4, Hkv=2, D=64),
    "causal_d128": dict(lens=((90, 200), (17, 40)), Hq=8, Hkv=2, D=128, dtype="bf16"),
    "window": dict(lens=((90, 200), (5, 150)), window=40, Hq=4, Hkv=1, D=128),
    "cap": dict(lens=((90, 200), (5, 150)), cap=9.0, Hq=4, Hkv=2, D=128),
    "d256": dict(lens=((40, 200), (5, 150)), Hq=2, Hkv=1, D=256),
    "split": dict(lens=((40, 5000), (8, 3000)), Hq=8, Hkv=2, D=128),
    "shared": dict(lens=((3, 9), (1, 1), (90, 100)), prefix=150, window=80, Hq=4, Hkv=2, D=64),
}


@pytest.mark.parametrize("name", list(HIDDEN))
@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_values_that_are_not_finite(gpu, kernel, name):
    """One key of each sequence has infinities, of either sign, and NaN among its values: the rows that see it have them
    in those columns, everything else is as if they were zero."""
    case = Case(seed=len(name), **HIDDEN[name])
    announce(f"not finite values kernel={kernel} {name}")
    at = []
    for b, (n, kv) in enumerate(case.lens):
        j = kv - max(1, n // 2)   # seen by the later half of the new tokens (a window's last ones apart)
        at.append(j)
        case.values[b][j, :, 1:4] = 0
        x = to_bits(np.array([np.inf, -np.inf, np.nan]), case.dtype)
        bits = case.values[b].copy()
        bits[j, :, 1:4] = x
        case.put(case.v, b, bits)
    dev = Device(gpu, case)
    pinned(gpu, kernel)
    try:
        dev.clear()
        dev.launch()
        gpu.synchronize()
    finally:
        pinned(gpu, 0)
    got, lse, _ = dev.result()
    want, wlse, bound, lbound = case.reference()
    seen = np.zeros((case.T, 1), bool)
    for b, (n, kv) in enumerate(case.lens):
        i = np.arange(n)
        pos = kv - n + i
        see = (at[b] <= pos) & ((at[b] > pos - case.window) if case.window else True)
        assert n == 1 or (see.any() and not see.all())
        seen[case.q_start[b]:case.q_start[b] + n, 0] = see
    for d, test in ((1, np.isposinf), (2, np.isneginf), (3, np.isnan)):
        ok = np.where(seen, test(got[:, :, d]), True)
        assert ok.all(), (d, np.argwhere(~ok)[:5])
    rest = np.ones(got.shape, bool)
    rest[:, :, 1:4] = ~seen[:, :, None]
    off = bad(got, want, bound) & rest
    assert not off.any(), (np.argwhere(off)[:5], got[off][:5], want[off][:5])
    assert not bad(lse, wlse, lbound).any()


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_hidden_keys_that_are_not_finite(gpu, kernel):
    """Keys of NaN and infinity that the first rows do not see change nothing for them; rows that see them are NaN."""
    case = Case(lens=((90, 200), (4, 40)), Hq=4, Hkv=2, D=64, seed=3)
    announce(f"not finite keys kernel={kernel}")
    for b, x in ((0, np.nan), (1, np.inf)):
        bits = case.keys[b].copy()
        bits[case.kv_len[b] - 2] = to_bits(np.full(64, x), "f16")   # infinities of q.k's terms cancel to NaN
        case.put(case.k, b, bits)
    dev = Device(gpu, case)
    pinned(gpu, kernel)
    try:
        dev.launch()
        gpu.synchronize()
    finally:
        pinned(gpu, 0)
    got, _, _ = dev.result()
    want, _, bound, _ = case.reference()
    off = bad(got, want, bound)
    for b in range(2):
        end = case.q_start[b + 1]
        assert not off[case.q_start[b]:end - 2].any()
        assert np.isnan(got[end - 2:end]).all()


# ---- tables and lengths ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("name", ["decode", "prompt"])
def test_pages_that_are_none(gpu, kernel, name):
    """Page numbers outside the cache, amid and at the end of a sequence: their keys are masked."""
    lens = ((1, 300), (1, 16), (2, 130)) if name == "decode" else ((100, 300), (40, 41))
    case = Case(lens=lens, Hq=4, Hkv=2, D=64, seed=5)
    table, dead = case.table.copy(), []
    for b, page, no in ((0, 0, -1), (0, 7, case.pages), (0, 18, -5), (1, 0, 2 ** 31 - 1)):
        table[b, page] = no
        dead += [(b, j) for j in range(page * 16, min(page * 16 + 16, case.lens[b][1]))]
    check(gpu, case, kernel, dead=dead, table=table)


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_prefix_pages_that_are_none(gpu, kernel):
    case = Case(lens=((1, 3), (2, 20)), prefix=100, Hq=4, Hkv=2, D=64, seed=6)
    pp = case.ppages.copy()
    pp[2] = -1
    check(gpu, case, kernel, dead=[(-1, j) for j in range(32, 48)], ppages=pp)


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("max_q", [0, 1, 7, 10 ** 9])
def test_wrong_most_new_tokens(gpu, kernel, max_q):
    """max_q is a hint: results are right whatever it says."""
    check(gpu, Case(lens=((1, 30), (70, 150), (9, 9)), Hq=4, Hkv=2, D=64, seed=7), kernel, max_q=max_q)


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("prefix", [0, 20])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 231])
def test_windows_wider_than_the_cache(gpu, kernel, prefix, window):
    """Also with more new tokens than the cache is said to hold, whose positions are negative."""
    check(gpu, Case(lens=((5, 3), (40, 200), (1, 0)), Hq=4, Hkv=2, D=64, seed=10, window=window, prefix=prefix), kernel)


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("prefix", [0, 40])
def test_lengths_past_the_buffers(gpu, kernel, prefix):
    """kv_len past the table is cut to it, row numbers to T, negative ones to 0; nothing else is written."""
    announce(f"lengths past the buffers kernel={kernel} prefix={prefix}")
    case = Case(lens=((1, 47), (2, 48), (0, 3)), Hq=4, Hkv=2, D=64, seed=8, prefix=prefix, tail=0)
    table = np.ascontiguousarray(case.table[:, :3])   # 48 tokens
    case.table, case.max_pages = table, 3
    dev = Device(gpu, case)
    dev.kv_len.copy_from(np.array([47, 2 ** 31 - 1, -7], np.int32))
    dev.q_start.copy_from(np.array([-3, 1, 3, 2 ** 31 - 1], np.int32))
    pinned(gpu, kernel)
    try:
        dev.clear()
        dev.launch()
        gpu.synchronize()
    finally:
        pinned(gpu, 0)
    got, lse, _ = dev.result()
    want, wlse, bound, lbound = case.reference()
    assert not bad(got, want, bound).any() and not bad(lse, wlse, lbound).any()


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("prefix", [0, 40])
def test_rows_that_fall(gpu, kernel, prefix):
    """A q_start that falls is no batch; the call ends and a right one behind it is right."""
    announce(f"q_start falls kernel={kernel} prefix={prefix}")
    case = Case(lens=((30, 47), (20, 48), (10, 30)), Hq=4, Hkv=2, D=64, seed=9, prefix=prefix)
    dev = Device(gpu, case)
    pinned(gpu, kernel)
    try:
        dev.q_start.copy_from(np.array([0, 50, 5, 60], np.int32))
        dev.launch()
        gpu.synchronize()
    finally:
        pinned(gpu, 0)
    check(gpu, case, kernel)


# ---- layouts -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["q_odd", "o_4", "o_odd", "token_major", "page_7", "d_20"])
@pytest.mark.parametrize("rows", [1, 60])
def test_layouts(gpu, kind, rows):
    """Strides and sizes that the MFMA kernels take only in part, or not at all (the generic kernel then runs)."""
    announce(f"layout {kind} rows={rows}")
    D, page = (20 if kind == "d_20" else 64), (7 if kind == "page_7" else 16)
    case = Case(lens=((rows, 100), (1, 30), (rows, rows)), Hq=4, Hkv=2, D=D, page=page, seed=11)
    dev = Device(gpu, case)
    qs, os_ = list(dev.packed), list(dev.packed)
    if kind == "token_major":   # heads outside tokens
        qs, os_ = [1, case.T * D, D], [1, case.T * D, D]
    if kind == "q_odd":
        qs = [1, D + 3, case.Hq * (D + 3) + 1]
    if kind in ("o_4", "o_odd"):
        x = 4 if kind == "o_4" else 1
        os_ = [1, D + x, case.Hq * (D + x)]

    def span(st):
        return (case.T - 1) * st[2] + (case.Hq - 1) * st[1] + D

    def index(st):
        t, h, d = np.ogrid[:case.T, :case.Hq, :D]
        return t * st[2] + h * st[1] + d

    q = np.zeros(span(qs), case.q.dtype)
    q[index(qs)] = case.q
    Q = gpu.HIPDeviceArray.from_numpy(q, "f16")
    O = gpu.HIPDeviceArray("f16", (span(os_),))
    O.fill_bytes(0x5a)
    gpu.kernel_log_clear()
    gpu.paged_attn_raw(dev.cache, dev.batch, dev.score, Q.ptr, O.ptr, case.Hq, qs, os_)   # no lse
    log = gpu.kernel_log()
    gpu.synchronize()
    generic = kind in ("q_odd", "o_odd", "page_7", "d_20")
    assert (log == ["paged_any_kernel"]) == generic, log
    flat = O.to_numpy()
    got = to_f64(flat[index(os_)], "f16")
    want, _, bound, _ = case.reference()
    assert not bad(got, want, bound).any()
    gaps = np.ones(flat.size, bool)
    gaps[index(os_).ravel()] = False
    assert (flat[gaps].view(np.uint16) == 0x5a5a).all()


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
def test_offsets_past_32_bits(gpu, kernel):
    """Pages a gigabyte apart: page 5 begins past 2^32 bytes and 2^31 elements."""
    announce(f"offsets past 32 bits kernel={kernel}")
    case = Case(lens=((3, 40), (40, 60)), Hq=4, Hkv=2, D=64, seed=12)
    step = 1 << 29   # elements
    order = np.argsort(np.concatenate([case.table[0, :3], case.table[1, :4]]))   # the seven pages in use
    used = np.concatenate([case.table[0, :3], case.table[1, :4]])
    place = {int(p): i for i, p in enumerate(used[order])}
    table = np.array([[place.get(int(p), -1) for p in row] for row in case.table], np.int32)
    n = case.Hkv * case.page * case.D
    dev = Device(gpu, case, table=table)
    big = [gpu.HIPDeviceArray("f16", (6 * step + n,)) for _ in range(2)]
    try:
        for a, src in zip(big, (case.k, case.v)):
            for p, i in place.items():
                h = np.ascontiguousarray(src[p]).ravel()
                gpu._lib.call("lava_hip_memcpy_h2d", a.ptr + 2 * i * step, h.ctypes.data, h.nbytes)
        cache = gpu.paged_cache_raw("f16", big[0].ptr, big[1].ptr, case.D, case.page, case.Hkv, 7,
                                    (1, case.D, case.page * case.D, step))
        dev.cache = cache
        pinned(gpu, kernel)
        dev.clear()
        dev.launch()
        gpu.synchronize()
        got, _, _ = dev.result()
    finally:
        pinned(gpu, 0)
        for a in big:
            a.close()
    want, _, bound, _ = case.reference()
    assert not bad(got, want, bound).any()


@pytest.mark.parametrize("kernel", [0] + list(KERNELS))
@pytest.mark.parametrize("shift", [2 ** 24, 2 ** 29])
def test_slopes_at_positions_past_24_bits(gpu, kernel, shift):
    """A window at the end of a long sequence, its earlier pages gone: distances are exact wherever they lie."""
    announce(f"slopes at positions past 24 bits kernel={kernel} shift={shift}")
    page = 2048
    case = Case(lens=((70, 400), (1, 300)), window=200, slopes=True, Hq=4, Hkv=2, D=64, page=page, seed=22)
    dev = Device(gpu, case)
    table = np.full((case.B, shift // page + case.max_pages), -1, np.int32)
    table[:, shift // page:] = case.table
    TB = gpu.HIPDeviceArray.from_numpy(table.ravel(), "i32")
    dev.kv_len.copy_from(case.kv_len + np.int32(shift))
    dev.batch = gpu.paged_batch_raw(case.B, case.T, dev.q_start.ptr, dev.kv_len.ptr, TB.ptr, table.shape[1], max_q=70)
    pinned(gpu, kernel)
    try:
        dev.clear()
        dev.launch()
        gpu.synchronize()
    finally:
        pinned(gpu, 0)
    got, lse, _ = dev.result()
    want, wlse, bound, lbound = case.reference()
    assert not bad(got, want, bound).any() and not bad(lse, wlse, lbound).any()


# ---- streams, workspaces, graphs --------------------------------------------------------------------------------

SERVED = {
    "decode": dict(lens=tuple((1, 1 + (i * 397) % 1900) for i in range(20)), Hq=16, Hkv=8, D=128),
    "chunks": dict(lens=((70, 900), (1, 200), (130, 131)), Hq=8, Hkv=2, D=64),
    "shared": dict(lens=tuple((1, 1 + i) for i in range(9)), prefix=1500, Hq=32, Hkv=8, D=128),
}


def own_workspace(lh, dev):
    c = dev.case
    n = lh.paged_workspace_bytes(dev.cache, dev.batch, c.Hq, c.prefix)
    ws = lh.HIPDeviceArray("u8", (max(n, 1),))
    ws.fill_bytes(0)
    dev.batch = lh.paged_batch_raw(c.B, c.T, dev.q_start.ptr, dev.kv_len.ptr, dev.table.ptr, c.max_pages,
                                   max_q=max(n for n, _ in c.lens), workspace=ws.ptr, workspace_bytes=n)
    return ws


@pytest.mark.parametrize("name", list(SERVED))
def test_streams_and_workspaces_give_the_same_bits(gpu, name):
    announce(f"streams and workspaces {name}")
    case = Case(seed=13, **SERVED[name])
    dev = Device(gpu, case)
    dev.clear()
    dev.launch()
    gpu.synchronize()
    _, _, first = dev.result()
    s = gpu.Stream()
    ws = None
    for own in (False, True):
        if own:
            ws = own_workspace(gpu, dev)
        for _ in range(3):
            dev.clear()
            gpu.synchronize()
            dev.launch(stream=s.handle)
            s.synchronize()
            _, _, raw = dev.result()
            assert (raw.view(np.uint16) == first.view(np.uint16)).all()
    ws.close()
    s.close()


@pytest.mark.parametrize("name", list(SERVED))
def test_graphs_with_their_own_workspaces(gpu, name):
    """Two graphs, captured from calls of different lengths, each with its workspace, replayed on two streams with
    eager calls between."""
    announce(f"graphs {name}")
    lens = SERVED[name]["lens"]
    cases = [Case(seed=14, **SERVED[name]), Case(seed=15, **dict(SERVED[name], lens=tuple((n, max(n, kv // 2)) for n, kv in lens)))]
    devs, eager, graphs, keep = [], [], [], []
    for case in cases:
        dev = Device(gpu, case)
        dev.clear()
        dev.launch()
        gpu.synchronize()
        eager.append(dev.result()[2].view(np.uint16).copy())
        keep.append(own_workspace(gpu, dev))
        s = gpu.Stream()
        g = gpu.Graph(s)
        with g.capture():
            dev.launch(stream=s.handle)
        devs.append(dev)
        graphs.append((s, g))
    for _ in range(4):
        for dev in devs:
            dev.clear()
        gpu.synchronize()
        for s, g in graphs:
            g.launch()
        for s, _ in graphs:
            s.synchronize()
        for dev, want in zip(devs, eager):
            assert (dev.result()[2].view(np.uint16) == want).all()
        devs[0].launch()   # an eager call between the replays
        gpu.synchronize()
    # new lengths in the arrays that the graph names
    case = cases[0]
    fewer = np.array([max(n, kv - 1) for n, kv in case.lens], np.int32)
    devs[0].kv_len.copy_from(fewer)
    devs[0].clear()
    gpu.synchronize()
    graphs[0][1].launch()
    graphs[0][0].synchronize()
    replayed = devs[0].result()[2].view(np.uint16).copy()
    devs[0].clear()
    devs[0].launch()
    gpu.synchronize()
    assert (devs[0].result()[2].view(np.uint16) == replayed).all()
    for s, g in graphs:
        g.close()
        s.close()


def test_capture_without_a_workspace_is_refused(gpu):
    """A capturing stream allocates nothing: without a workspace the call says so, and runs afterwards."""
    announce("capture without a workspace")
    case = Case(seed=16, **SERVED["decode"])
    dev = Device(gpu, case)
    s = gpu.Stream()
    g = gpu.Graph(s)
    with g.capture():
        with pytest.raises(gpu.LavaHIPError):
            dev.launch(stream=s.handle)
    dev.clear()
    gpu.synchronize()
    dev.launch(stream=s.handle)
    s.synchronize()
    want, _, bound, _ = case.reference()
    assert not bad(dev.result()[0], want, bound).any()
    g.close()
    s.close()


def test_small_and_misaligned_workspaces_are_refused(gpu):
    announce("workspace refusals")
    case = Case(seed=17, **SERVED["decode"])
    dev = Device(gpu, case)
    n = gpu.paged_workspace_bytes(dev.cache, dev.batch, case.Hq)
    ws = own_workspace(gpu, dev)
    for ptr, size in ((ws.ptr, n - 1), (ws.ptr + 8, n)):
        dev.batch.workspace, dev.batch.workspace_bytes = ptr, size
        with pytest.raises(gpu.InvalidArgument, match="workspace"):
            dev.launch()
    ws.close()


# ---- the operators together ---------------------------------------------------------------------------------------

def test_a_program_that_generates(gpu):
    """Prompts appended with rotary positions and attended, then decoded token by token, then continued by several samples
    behind the shared first prompt: every step's results against softmax over all the tokens so far in 64 bits."""
    lh = gpu
    announce("prompt, decode and shared prefix together")
    dtype, Hq, Hkv, D, page, B = "f16", 8, 2, 64, 16, 3
    rng = np.random.default_rng(21)
    prompts, steps = (50, 1, 33), 4
    cache = lh.PagedCache(dtype, D, page, Hkv, 40)
    cache.k.fill_bytes(0xff)
    cache.v.fill_bytes(0xff)   # NaN
    table = rng.permutation(40)[:24].reshape(B, 8).astype(np.int32)
    inv = (100.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    INV = lh.HIPDeviceArray.from_numpy(inv, "f32")
    held = [(np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))) for _ in range(B)]   # keys as the cache rounds them, values

    def turn(x, pos):   # (n, H, D) in 64 bits
        a = pos[:, None, None] * inv.astype(np.float64)
        x0, x1 = x[..., :D // 2], x[..., D // 2:]
        return np.concatenate([x0 * np.cos(a) - x1 * np.sin(a), x1 * np.cos(a) + x0 * np.sin(a)], -1)

    def step(new, lens, tables, past, prefix=0, prefix_pages=None):
        """new: tokens of each sequence; lens: what each holds behind `prefix`, without them; past: keys and values."""
        T = sum(new)
        q_start = np.cumsum([0] + list(new)).astype(np.int32)
        kv = np.array([l + n for l, n in zip(lens, new)], np.int32)
        q, k, v = (rng.standard_normal((T, H, D)).astype(np.float16) for H in (Hq, Hkv, Hkv))
        dev = lambda a: lh.HIPDeviceArray.from_numpy(np.asfortranarray(a.transpose(2, 1, 0)), dtype)
        batch = lh.PagedBatch(T, lh.HIPDeviceArray.from_numpy(q_start, "i32"), lh.HIPDeviceArray.from_numpy(kv, "i32"),
                              lh.HIPDeviceArray.from_numpy(np.asfortranarray(tables.T), "i32"), max(new))
        Q, K, V = dev(q), dev(k), dev(v)
        O = lh.HIPDeviceArray(dtype, (D, Hq, T))
        lse = lh.HIPDeviceArray("f32", (Hq, T))
        lh.kv_append(cache, batch, K, V, Q=Q, inv_freq=INV, offset=prefix)
        if prefix:
            lh.shared_prefix_attn(O, cache, batch, prefix_pages, prefix, Q, lse=lse)
        else:
            lh.paged_attn(O, cache, batch, Q, lse=lse)
        lh.synchronize()
        got, gl = O.to_numpy().transpose(2, 1, 0).astype(np.float64), lse.to_numpy().T
        out = []
        for b, n in enumerate(new):
            r = slice(q_start[b], q_start[b] + n)
            pos = prefix + lens[b] + np.arange(n)
            keys = np.concatenate([past[b][0], turn(k[r].astype(np.float64), pos)])
            vals = np.concatenate([past[b][1], v[r].astype(np.float64)])
            qt = turn(q[r].astype(np.float64), pos)
            out.append((keys, vals))
            for h in range(Hq):
                kh, vh = keys[:, h // (Hq // Hkv)], vals[:, h // (Hq // Hkv)]
                s = qt[:, h] @ kh.T / np.sqrt(D)
                # q and k are rounded to f16 when stored, half a step each, and a score to the sum's 32 bits
                ds = (np.abs(qt[:, h]) @ np.abs(kh).T / np.sqrt(D)) * (2 * 2.0 ** -11 + 2.0 ** -21 + (D + 2) * 2.0 ** -24) + 2.0 ** -21
                keep = np.arange(len(kh))[None] <= pos[:, None]
                s = np.where(keep, s, -np.inf)
                top = s.max(1, keepdims=True)
                e = np.exp(s - top)
                w = e / e.sum(1, keepdims=True)
                o, a = w @ vh, w @ np.abs(vh)
                near = np.where(keep, ds, 0).max(1, keepdims=True)
                bound = (2 * 2.0 ** -11 + 2 * near + 2.0 ** -24 * (len(kh) + 8)) * a + 2.0 ** -11 * np.abs(o) + 2.0 ** -24 * (
                    1 + keep.astype(float) @ np.abs(vh))
                off = np.abs(got[r, h] - o) > 1.02 * bound
                assert not off.any(), (b, h, np.argwhere(off)[:4])
                want = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
                assert (np.abs(gl[r, h] - want) <= 1.02 * (2.0 ** -11 + near[:, 0] + 2.0 ** -20)).all()
        return out

    held = step(list(prompts), [0] * B, table, held)
    lens = list(prompts)
    for _ in range(steps):
        held = step([1] * B, lens, table, held)
        lens = [n + 1 for n in lens]
    # five samples go on from the first prompt (48 of its tokens: three whole pages), each with pages of its own
    n, pre = 5, 48
    own = np.array([[p] for p in set(range(40)) - set(table.ravel().tolist())], np.int32)[:n]
    pages = lh.HIPDeviceArray.from_numpy(table[0, :3].copy(), "i32")
    samples = [(held[0][0][:pre], held[0][1][:pre])] * n
    for i in range(steps):
        samples = step([1] * n, [i] * n, own, samples, prefix=pre, prefix_pages=pages)
    cache.close()
