"""Eviction's scratch, by the C entry points' answers (no GPU)."""
import ctypes

import pytest


@pytest.mark.parametrize("apart", [0, 1])
@pytest.mark.parametrize("keep", [1, 300, 2048, 2049, 1 << 20, 2 ** 31 - 1])
def test_scratch_goes_by_the_tokens_there_are(te, keep, apart):
    """Two lists of at most the kept tokens for each row and head, whatever `keep` allows beyond them."""
    rows, heads, length, size = 16, 8, 2048, ctypes.c_size_t(0)
    cache = te._capi.TrellisKVCache(k=256, v=256, scores=256, pos=256, table=256, lens=512, page_stride=8 * 16 * 64, head_stride=16 * 64,
                                    slot_stride=64, table_stride=128, pages=9, heads=heads, page_size=16, head_dim=64, dtype=1,
                                    rows=rows, width=128, max_len=length)
    assert te.library().trellis_evict_workspace_bytes(cache, keep, apart, size) == 0
    assert size.value <= rows * heads * 4 * (1 + 2 * min(keep, length)) + 3 * 256
    assert apart or keep < length or size.value == 0      # nothing can move
