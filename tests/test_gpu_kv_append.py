"""Appending to the paged cache: every slot against the rotation in 64 bits, and everything else untouched.

Bound for a rotated element x cos - y sin: its own rounding (u of it, and f16's smallest step), and 2^-21 (|x| + |y|) for
the 32-bit sine and cosine (2^-22), their angle (2^-25 of a turn, 2^-22.3 radians) and the products."""
import numpy as np
import pytest

from conftest import announce
from paged_reference import TINY, U, to_bits, to_f64

pytestmark = pytest.mark.gpu


def run(lh, dtype="f16", Hq=4, Hkv=2, D=64, page=16, order="hl", lens=((1, 5),), rot=None, interleaved=False, positions=None,
        offset=0, fused=True, in_place=False, gap=0, tail=2, q=True, table_edit=None, kernel=None, seed=0, stream=None):
    rot = D if rot is None else rot
    announce(f"kv_append {dtype} Hq={Hq} Hkv={Hkv} D={D} page={page} {order} lens={lens} rot={rot} il={interleaved} "
             f"offset={offset} fused={fused} in_place={in_place} q={q}")
    rng = np.random.default_rng(seed)
    B = len(lens)
    q_start = np.cumsum([gap] + [n for n, _ in lens]).astype(np.int32)
    T = int(q_start[-1]) + tail
    need = [-(-kv // page) for _, kv in lens]
    pages, mp = sum(need) + 2, max(need + [1])
    perm, at = rng.permutation(pages).astype(np.int32), 0
    table = np.full((B, mp), -1, np.int32)
    for b, c in enumerate(need):
        table[b, :c] = perm[at:at + c]
        at += c
    if table_edit:
        table_edit(table, pages)
    heads = Hq + 2 * Hkv if fused else max(Hq, Hkv)
    x = to_bits(rng.standard_normal((3 if not fused else 1, T, heads, D)), dtype)
    shape = (pages, Hkv, page, D) if order == "hl" else (pages, page, Hkv, D)
    k0, v0 = to_bits(rng.standard_normal(shape), dtype), to_bits(rng.standard_normal(shape), dtype)
    up = lambda a, t: lh.HIPDeviceArray.from_numpy(np.ascontiguousarray(a).ravel(), t)
    X, K, V = up(x, dtype), up(k0, dtype), up(v0, dtype)
    QS, KL, TB = up(q_start, "i32"), up(np.array([kv for _, kv in lens], np.int32), "i32"), up(table, "i32")
    freq = (10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))).astype(np.float32)
    F = up(freq if len(freq) else np.zeros(1, np.float32), "f32")
    PO = up(np.asarray(positions, np.int32), "i32") if positions is not None else None
    out = lh.HIPDeviceArray(dtype, (T * Hq * D,))
    out.fill_bytes(0x5a)
    strides = (1, D, page * D, Hkv * page * D) if order == "hl" else (1, Hkv * D, D, page * Hkv * D)
    cache = lh.paged_cache_raw(dtype, K.ptr, V.ptr, D, page, Hkv, pages, strides)
    batch = lh.paged_batch_raw(B, T, QS.ptr, KL.ptr, TB.ptr, mp)
    rope = lh.rope_raw(F.ptr, rot, interleaved, PO.ptr if PO else 0, offset)
    plane, tok = T * heads * D, (1, D, heads * D)
    kp = X.ptr + 2 * (Hq * D if fused else plane)
    vp = X.ptr + 2 * ((Hq + Hkv) * D if fused else 2 * plane)
    qo, qos = (X.ptr, tok) if in_place else (out.ptr, (1, D, Hq * D))
    lh.kernel_log_clear()
    lh.kv_append_raw(cache, batch, kp, vp, tok, Q=X.ptr if q else 0, Q_out=qo if q else 0, q_heads=Hq if q else 0,
                     q_strides=tok if q else None, qo_strides=qos if q else None, rope=rope, stream=stream)
    if kernel:
        assert lh.kernel_log() == [kernel], lh.kernel_log()
    lh.synchronize()

    # the reference
    xin = to_f64(x, dtype)
    part = (lambda i, h0, n: xin[0][:, h0:h0 + n]) if fused else (lambda i, h0, n: xin[i][:, :n])
    xq, xk, xv = part(0, 0, Hq), part(1, Hq, Hkv), part(2, Hq + Hkv, Hkv)
    wk, wv, bk = to_f64(k0, dtype), to_f64(v0, dtype), np.zeros(shape)
    wq, bq = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    j = np.arange(rot // 2)
    e0, e1 = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)

    def turn(row, pos):
        a = pos * freq.astype(np.float64)
        o, bnd = row.copy(), np.zeros_like(row)
        o[:, e0] = row[:, e0] * np.cos(a) - row[:, e1] * np.sin(a)
        o[:, e1] = row[:, e1] * np.cos(a) + row[:, e0] * np.sin(a)
        for e in (e0, e1):
            bnd[:, e] = U[dtype] * np.abs(o[:, e]) + TINY[dtype] + 2.0 ** -21 * (np.abs(row[:, e0]) + np.abs(row[:, e1]))
        return o, bnd

    for b, (n, kv) in enumerate(lens):
        for i in range(n):
            t, slot = q_start[b] + i, kv - n + i
            pos = positions[t] if positions is not None else offset + slot
            if q:
                wq[t], bq[t] = turn(xq[t], pos)
            if slot < 0:
                continue
            p = table[b, slot // page]
            if p < 0 or p >= pages:
                continue
            at = (p, slice(None), slot % page) if order == "hl" else (p, slot % page)
            wk[at], bk[at] = turn(xk[t], pos)
            wv[at] = xv[t]
    gk, gv = to_f64(K.to_numpy().reshape(shape), dtype), to_f64(V.to_numpy().reshape(shape), dtype)
    np.testing.assert_array_equal(gv, wv)
    off = ~(np.abs(gk - wk) <= bk)
    assert not off.any(), (np.argwhere(off)[:5], gk[off][:5], wk[off][:5])
    after = to_f64(X.to_numpy().reshape(x.shape), dtype)
    if q and in_place:
        gq = after[0][:, :Hq]
        want = np.where(np.isnan(wq), xq, wq)
    elif q:
        raw = out.to_numpy().reshape(T, Hq, D)
        free = np.isnan(wq[:, 0, 0])
        assert (raw.view(np.uint16)[free] == 0x5a5a).all()
        gq, want = to_f64(raw, dtype)[~free], wq[~free]
        bq = bq[~free]
    if q:
        off = ~(np.abs(gq - want) <= bq)
        assert not off.any(), (np.argwhere(off)[:5], gq[off][:5], want[off][:5])
    if not in_place:
        np.testing.assert_array_equal(after, xin)


RAGGED = ((1, 1), (0, 9), (1, 16), (1, 17), (3, 3), (5, 40), (1, 33), (20, 31))
VEC, ANY = "kv_append_kernel", "kv_append_any_kernel"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(D=128, Hq=8, Hkv=2, kernel=VEC), dict(D=128, interleaved=True, order="lh", kernel=VEC),
    dict(D=128, rot=64, kernel=VEC), dict(D=128, rot=64, interleaved=True, kernel=VEC), dict(D=80, rot=16, kernel=VEC),
    dict(D=80, rot=80, kernel=VEC), dict(D=72, rot=72, interleaved=True, kernel=VEC), dict(D=256, page=24, kernel=VEC),
    dict(D=64, rot=0, kernel=VEC), dict(D=8, rot=8, interleaved=True, kernel=VEC), dict(D=64, rot=24, kernel=ANY),
    dict(D=77, rot=50, kernel=ANY), dict(D=77, rot=76, interleaved=True, page=5, kernel=ANY), dict(D=1, rot=0, kernel=ANY),
    dict(D=64, q=False, kernel=VEC), dict(D=64, in_place=True, kernel=VEC), dict(D=24, rot=20, in_place=True, kernel=ANY),
    dict(D=64, fused=False, kernel=VEC), dict(D=64, offset=4000000, kernel=VEC), dict(D=64, gap=3, tail=7, kernel=VEC),
])
def test_append(gpu, dtype, kw):
    run(gpu, dtype=dtype, lens=RAGGED, **kw)


def test_append_positions(gpu):
    T = sum(n for n, _ in RAGGED) + 2
    run(gpu, lens=RAGGED, positions=np.random.default_rng(1).integers(0, 1 << 21, T))


def test_append_more_new_than_cached(gpu):
    """Tokens in front of the cache's first slot are turned, not stored."""
    run(gpu, lens=((5, 3), (2, 0), (1, 1)))
    run(gpu, lens=((5, 3), (2, 0), (1, 1)), D=20, rot=20)


def test_append_pages_that_are_none(gpu):
    def edit(table, pages):
        table[5, 1], table[5, 2], table[6, 1] = -1, pages, 0x7fffffff
    run(gpu, lens=RAGGED, table_edit=edit)
    run(gpu, lens=RAGGED, table_edit=edit, D=20, rot=20)


def test_append_many_sequences(gpu):
    run(gpu, lens=tuple((i % 4, 4 + i % 31) for i in range(300)), D=64, kernel=VEC)


def test_append_empty(gpu):
    lh = gpu
    cache = lh.paged_cache_raw("f16", 0, 0, 64, 16, 2, 0, (1, 64, 1024, 2048))
    lh.kv_append_raw(cache, lh.paged_batch_raw(0, 0, 0, 0, 0, 0), 0, 0, None)
