"""Sizes of the paged cache's calls that no device has memory for: refused on the host before anything is multiplied past 64 bits. Runs without a GPU."""
import ctypes as C

import pytest

from test_paged_refusals import CTX, LIMIT, attention, cache, evict


@pytest.mark.parametrize("count,kv_heads,keep", [(65535, 65535, 1 << 30), (65535, 65535, 536887298), (46341, 46341, 1 << 30), (32768, 32768, 1 << 29)])
def test_evictions(pkg, count, kv_heads, keep):
    """Two words of scratch for every place: from 2^61 places on their bytes do not fit 64 bits."""
    c = cache(kv_heads=kv_heads, page_tokens=4096, max_pages=1 << 18)
    call = evict(count=count, keep=keep, ld=1 << 30)
    assert pkg.native.lib().m40llm_paged_evict_async(CTX, C.byref(c), C.byref(call)) == LIMIT


@pytest.mark.parametrize("dim", [64, 128, 509])
@pytest.mark.parametrize("rows,heads", [(65535, 65535), (65535, 32768)])
def test_scores(pkg, dim, rows, heads):
    c = cache(kv_heads=1, head_dim=dim, page_tokens=4096, max_pages=1 << 18)
    call = attention(rows=rows, q_heads=heads, ld_weights=1 << 30)
    assert pkg.native.lib().m40llm_attention_paged_async(CTX, C.byref(c), C.byref(call)) == LIMIT
