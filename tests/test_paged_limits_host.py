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
