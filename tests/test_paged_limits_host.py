"""Limits of the paged cache's entry points that the host checks or plans by: no call here touches a device."""
import pytest

import lava_hip as lh
from test_paged_host import append, attn, batch, cache, shared


def test_attention_takes_at_most_2_30_tokens():
    """Beyond them positions in front of the cache, less a window's or a key's, would leave 32 bits."""
    for entry in (attn, shared):
        with pytest.raises(lh.Unsupported, match="2\\^30"):
            entry(b=batch(tokens=2 ** 30 + 1))
    with pytest.raises(lh.Unsupported, match="2\\^30"):
        lh.paged_workspace_bytes(cache(), batch(tokens=2 ** 30 + 1), 4)
    with pytest.raises(lh.InvalidArgument, match="null"):   # an append goes on to its other checks
        append(b=batch(tokens=2 ** 31 - 1), K=0)


def needs(sequences, tokens, heads, keys, D=128, width=2 ** 16, page=16, max_q=0, prefix=0):
    """Bytes of workspace: none where the generic kernel would run."""
    c = cache(head_dim=D, page_size=page, heads=keys, strides=(1, D, page * D, keys * page * D))
    return lh.paged_workspace_bytes(c, batch(sequences=sequences, tokens=tokens, max_pages=width, max_q=max_q), heads, prefix)


@pytest.mark.parametrize("call", [
    dict(sequences=1, tokens=262144, heads=32, keys=8, width=262144 // 16),   # a prompt
    dict(sequences=1, tokens=196608, heads=64, keys=8, width=196608 // 16),
    dict(sequences=1, tokens=1 << 20, heads=64, keys=8, width=(1 << 20) // 16),
    dict(sequences=16, tokens=65536, heads=32, keys=8),                          # chunks before a table of 2^20 tokens
    dict(sequences=8, tokens=32768, heads=64, keys=8),
    dict(sequences=512, tokens=512, heads=32, keys=32, width=1 << 20, max_q=1),  # decode steps, tables of 2^24 and 2^30 tokens
    dict(sequences=64, tokens=64, heads=64, keys=8, width=1 << 26, max_q=1),
    dict(sequences=64, tokens=64, heads=64, keys=8, width=1 << 20, max_q=1, prefix=1 << 24),
    dict(sequences=4, tokens=1 << 20, heads=8, keys=8, D=256),
])
def test_wide_tables_and_long_prompts_keep_the_mfma_kernels(call):
    assert needs(**call) > 0


def test_where_the_generic_kernel_takes_over():
    """Rows on the row kernel: a head's tiles of 16 rows (one at most partly filled a sequence) times 2^23 blocks of 128 keys stay below
    2^31 up to 240 sequences of one row; whole tiles of 256 rows need no count of blocks, but hold heads of up to 128."""
    wide = dict(heads=3, keys=3, width=2 ** 26, max_q=1)
    assert needs(240, 240, D=256, **wide) > 0
    assert needs(241, 241, D=256, **wide) == 0
    assert needs(241, 241, D=128, **wide) > 0
    assert needs(100000, 100000, D=64, **wide) > 0


@pytest.mark.parametrize("make", [
    lambda x: cache(head_dim=x + 64), lambda x: cache(page_size=x + 16), lambda x: cache(heads=x + 2),
    lambda x: batch(sequences=x + 3), lambda x: batch(max_pages=x + 4), lambda x: lh.rope_raw(1 << 20, x + 64),
    lambda x: lh.rope_raw(1 << 20, 64, offset=x), lambda x: lh.attn_score_raw(1.0, window=x + 7)])
def test_integers_that_a_descriptor_would_cut_off_are_refused(make):
    for x in (2 ** 32, -2 ** 32):
        with pytest.raises(ValueError, match="32 bits"):
            make(x)
    make(0)


@pytest.mark.parametrize("make", [lambda x: cache(pages=x), lambda x: cache(strides=(1, 64, x, 2048)), lambda x: batch(tokens=x),
                                  lambda x: batch(max_q=x)])
def test_long_integers_that_a_descriptor_would_cut_off_are_refused(make):
    with pytest.raises(ValueError, match="64 bits"):
        make(2 ** 64 + 5)
    make(5)
