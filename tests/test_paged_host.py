"""What the paged cache's entry points refuse, on the host: every call here fails, or has nothing to do, before
a device is touched."""
import ctypes as C

import pytest

import lava_hip as lh

A = 1 << 20   # a 16-byte aligned address that nothing reads


def cache(**kw):
    d = dict(dtype="f16", k=A, v=A, head_dim=64, page_size=16, heads=2, pages=9, strides=(1, 64, 1024, 2048))
    d.update(kw)
    return lh.paged_cache_raw(**d)


def batch(**kw):
    d = dict(sequences=3, tokens=5, q_start=A, kv_len=A, table=A, max_pages=4)
    d.update(kw)
    return lh.paged_batch_raw(**d)


def score(**kw):
    d = dict(scale=0.125)
    d.update(kw)
    return lh.attn_score_raw(**d)


def attn(c=None, b=None, s=None, Q=A, O=A, heads=4, qs=(1, 64, 256), os=(1, 64, 256), lse=0):
    lh.paged_attn_raw(c or cache(), b or batch(), s or score(), Q, O, heads, qs, os, lse)


def shared(s=None, pages=A, prefix=32, **kw):
    lh.shared_prefix_attn_raw(kw.get("c") or cache(), kw.get("b") or batch(), s or score(), pages, prefix, A, A, 4,
                              (1, 64, 256), (1, 64, 256))


def append(c=None, b=None, K=A, V=A, ks=(1, 64, 128), rope=None, **kw):
    lh.kv_append_raw(c or cache(), b or batch(), K, V, ks, rope=rope, **kw)


BAD_CACHES = {
    "head_dim 0": (dict(head_dim=0), "head_dim"),
    "page_size 0": (dict(page_size=0), "page_size"),
    "heads 0": (dict(heads=0), "heads"),
    "heads 65536": (dict(heads=65536), "heads"),
    "pages -1": (dict(pages=-1), "pages"),
    "pages 2^31": (dict(pages=2 ** 31), "pages"),
    "strided elements": (dict(strides=(2, 128, 2048, 4096)), "contiguous"),
    "negative stride": (dict(strides=(1, 64, -1024, 2048)), "stride"),
    "tokens overlap": (dict(strides=(1, 63, 1024, 2048)), "stride 1"),
    "heads overlap": (dict(strides=(1, 64, 32, 2048)), "stride 2"),
    "pages overlap": (dict(strides=(1, 64, 1024, 1)), "stride 3"),
    "no keys": (dict(k=0), "null"),
    "no values": (dict(v=0), "null"),
    "odd address": (dict(k=A + 1), "misaligned"),
}
UNSUPPORTED_CACHES = {
    "dtype": (dict(dtype="f32"), "dtype"),
    "head_dim 257": (dict(head_dim=257, strides=(1, 257, 257 * 16, 257 * 32)), "head_dim"),
    "a page of 2^31 bytes": (dict(strides=(1, 1 << 28, 64, 1 << 33)), "2\\^31"),
}
BAD_BATCHES = {
    "sequences": (dict(sequences=-1), "negative"),
    "tokens": (dict(tokens=-1), "negative"),
    "max_pages": (dict(max_pages=-1), "negative"),
    "max_q": (dict(max_q=-1), "negative"),
    "2^31 tokens": (dict(tokens=2 ** 31), "too large"),
    "no q_start": (dict(q_start=0), "null"),
    "no kv_len": (dict(kv_len=0), "null"),
    "no table": (dict(table=0), "null"),
    "odd table": (dict(table=A + 2), "misaligned"),
}
ENTRIES = {"attn": attn, "shared": shared, "append": append}


@pytest.mark.parametrize("entry", list(ENTRIES))
@pytest.mark.parametrize("name", list(BAD_CACHES))
def test_caches_that_are_refused(entry, name):
    change, words = BAD_CACHES[name]
    with pytest.raises(lh.InvalidArgument, match=words):
        ENTRIES[entry](c=cache(**change))


@pytest.mark.parametrize("entry", list(ENTRIES))
@pytest.mark.parametrize("name", list(UNSUPPORTED_CACHES))
def test_caches_that_are_not_supported(entry, name):
    change, words = UNSUPPORTED_CACHES[name]
    with pytest.raises(lh.Unsupported, match=words):
        ENTRIES[entry](c=cache(**change))


@pytest.mark.parametrize("entry", list(ENTRIES))
@pytest.mark.parametrize("name", list(BAD_BATCHES))
def test_batches_that_are_refused(entry, name):
    change, words = BAD_BATCHES[name]
    with pytest.raises(lh.InvalidArgument, match=words):
        ENTRIES[entry](b=batch(**change))


def test_sequences_of_more_than_2_30_tokens_are_not_supported():
    for entry in ENTRIES.values():
        with pytest.raises(lh.Unsupported, match="2\\^30"):
            entry(b=batch(max_pages=(1 << 26) + 1))


@pytest.mark.parametrize("change,words", [
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(cap=float("nan")), "finite"),
    (dict(cap=-1.0), "cap"), (dict(window=-1), "window"), (dict(slopes=A + 1), "misaligned"),
    (dict(bidirectional=A, causal=False), "causal"), (dict(scale=1e30, cap=1e-30), "overflows")])
def test_scores_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        attn(s=score(**change))
    if "bidirectional" not in change:
        with pytest.raises(lh.InvalidArgument, match=words):
            shared(s=score(**change))


@pytest.mark.parametrize("change,words", [
    (dict(heads=3), "multiple"), (dict(heads=-2), "q_heads"), (dict(heads=65536), "q_heads"), (dict(Q=0), "null"),
    (dict(O=0), "null"), (dict(qs=None), "null"), (dict(os=None), "null"), (dict(Q=A + 1), "misaligned"),
    (dict(O=A + 1), "misaligned"), (dict(lse=A + 2), "misaligned"), (dict(qs=(2, 128, 512)), "contiguous"),
    (dict(qs=(1, 32, 256)), "q_strides"), (dict(os=(1, 64, 8)), "o_strides"), (dict(os=(1, -64, 256)), "o_strides")])
def test_attention_arguments_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        attn(**change)


def test_null_descriptors_are_refused():
    st = (C.c_int64 * 3)(1, 64, 256)
    c, b, s = cache(), batch(), score()
    for args in ((None, C.byref(b), C.byref(s)), (C.byref(c), None, C.byref(s)), (C.byref(c), C.byref(b), None)):
        with pytest.raises(lh.InvalidArgument, match="null"):
            lh._lib.call("lava_hip_paged_attn", *args, A, A, 4, st, st, None, None)
    with pytest.raises(lh.InvalidArgument, match="null"):
        lh._lib.call("lava_hip_paged_workspace_bytes", C.byref(c), C.byref(b), 4, 0, None)


def test_shared_prefixes_that_are_refused():
    with pytest.raises(lh.InvalidArgument, match="prefix_len"):
        shared(prefix=-1)
    with pytest.raises(lh.InvalidArgument, match="null"):
        shared(pages=0)
    with pytest.raises(lh.InvalidArgument, match="misaligned"):
        shared(pages=A + 2)
    with pytest.raises(lh.Unsupported, match="prefix_len"):
        shared(prefix=1 << 30)
    with pytest.raises(lh.Unsupported, match="bidirectional"):
        shared(s=score(bidirectional=A))
    with pytest.raises(lh.InvalidArgument, match="prefix_len"):
        lh.paged_workspace_bytes(cache(), batch(), 4, -1)


@pytest.mark.parametrize("rope,words", [
    (dict(rot_dim=7), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=-2), "rot_dim"),
    (dict(inv_freq=0), "inv_freq"), (dict(inv_freq=A + 2), "misaligned"), (dict(positions=A + 2), "misaligned"),
    (dict(offset=-1), "offset"), (dict(offset=2 ** 30 + 1), "offset")])
def test_rotations_that_are_refused(rope, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        append(rope=lh.rope_raw(**dict(dict(inv_freq=A, rot_dim=64), **rope)))


@pytest.mark.parametrize("change,words", [
    (dict(K=0), "null"), (dict(V=0), "null"), (dict(ks=None), "null"), (dict(K=A + 1), "misaligned"),
    (dict(ks=(1, 8, 128)), "kv_strides"), (dict(Q=A, q_heads=4, q_strides=(1, 64, 256)), "go together"),
    (dict(Q_out=A, q_heads=4), "go together"), (dict(Q=A, Q_out=A, q_heads=4), "null"),
    (dict(Q=A, Q_out=2 * A, q_heads=4, q_strides=(1, 64, 256), qo_strides=(1, 6, 256)), "qo_strides"),
    (dict(Q=A, Q_out=A, q_heads=4, q_strides=(1, 64, 256), qo_strides=(1, 64, 512)), "in place"),
    (dict(Q=A, Q_out=A, q_heads=-1, q_strides=(1, 64, 256), qo_strides=(1, 64, 256)), "q_heads")])
def test_append_arguments_that_are_refused(change, words):
    with pytest.raises(lh.InvalidArgument, match=words):
        append(**change)


def test_calls_with_nothing_to_do():
    """No tokens, no sequences, no query heads: nothing is read, pointers may be null."""
    for b in (batch(tokens=0, q_start=0, kv_len=0, table=0), batch(sequences=0, q_start=0, kv_len=0, table=0)):
        attn(b=b, Q=0, O=0, qs=None, os=None)
        append(b=b, K=0, V=0, ks=None)
        assert lh.paged_workspace_bytes(cache(), b, 4) == 0
    attn(heads=0, Q=0, O=0)


def test_workspace_bytes():
    """Grows with the batch, and is none where the generic kernel runs."""
    assert 0 < lh.paged_workspace_bytes(cache(), batch(), 4) <= lh.paged_workspace_bytes(cache(), batch(), 4, 4096)
    assert lh.paged_workspace_bytes(cache(page_size=7), batch(), 4) == 0
    many = lh.paged_workspace_bytes(cache(), batch(tokens=4096, sequences=64, max_pages=2048), 16, 4096)
    assert many > lh.paged_workspace_bytes(cache(), batch(), 16, 4096)


def test_descriptors_have_the_header_s_layout():
    L = lh._lib
    assert C.sizeof(L.KVCacheDesc) == 72 and L.KVCacheDesc.strides.offset == 40
    assert C.sizeof(L.KVBatchDesc) == 64 and L.KVBatchDesc.q_start.offset == 24 and L.KVBatchDesc.workspace.offset == 48
    assert C.sizeof(L.RopeDesc) == 32 and L.RopeDesc.positions.offset == 16
    assert C.sizeof(L.AttnScoreDesc) == 32 and L.AttnScoreDesc.slopes.offset == 16
