"""What the entry points of the paged cache and of the log probabilities refuse: all of it is found on the host, before the device is touched,
so it is tested without one (the context is a block of zeros that no refused call looks into)."""
import ctypes as C

import pytest

from helpers import load_package

load_package()
from m40_llm_b200 import native as N  # noqa: E402

LIMIT = N.ERR_LIMIT
CTX = C.create_string_buffer(4096)
P = 4096  # an aligned address that is never followed


def cache(**change):
    c = dict(k=P, v=P, table=P, pages=9, page_tokens=16, slots=4, max_pages=2, kv_heads=2, head_dim=64, elem_dtype=N.DT_F16)
    return N.PagedCache(**(c | change))


def append(**change):
    c = dict(q=P, k=P, v=P, q_out=P, turns=P, row_slot=P, row_entry=P, row_pos=P, entry_pos=P, weights=P, rows=3, ld=0, q_heads=8, pairs=32,
             rope_layout=0, ld_entry=32)
    return N.PagedAppend(**(c | change))


def attention(**change):
    c = dict(q=P, out=P, row_slot=P, row_len=P, row_begin=P, weights_in=P, weights_out=P, rows=3, q_heads=8, ld_weights=32, max_len=0, scale=0.1)
    return N.PagedAttention(**(c | change))


def evict(**change):
    c = dict(to=None, seq=P, len=P, weights=P, weights_out=P, entry_pos=P, entry_pos_out=P, origin=P, new_len=P, count=2, keep=9, first=2,
             recent=3, ld=32, max_len=0)
    return N.PagedEvict(**(c | change))


def logprobs(**change):
    c = dict(logits=P, tokens=P, logprob=P, rank=P, entropy=P, lse=P, top_ids=P, top_logprobs=P, rows=2, n=100, ld=0, top=5)
    return N.Logprobs(**(c | change))


CACHES = [(dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(pages=0), -2), (dict(slots=0), -2), (dict(max_pages=0), -2),
          (dict(kv_heads=0), -2), (dict(head_dim=0), -2), (dict(page_tokens=0), -2), (dict(page_tokens=24), -2), (dict(page_tokens=8192), LIMIT),
          (dict(head_dim=513), LIMIT), (dict(max_pages=1 << 27), LIMIT), (dict(elem_dtype=N.DT_BF16), -4), (dict(elem_dtype=9), -4),
          (dict(k=P + 1), -2), (dict(v=P + 2, elem_dtype=N.DT_F32), -2)]


@pytest.mark.parametrize("change,code", CACHES)
def test_cache(pkg, change, code):
    L, c = pkg.native.lib(), cache(**change)
    for f, call in ((L.m40llm_paged_append_async, append()), (L.m40llm_attention_paged_async, attention()), (L.m40llm_paged_evict_async, evict())):
        assert f(CTX, C.byref(c), C.byref(call)) == code
    to = cache(**change)
    assert L.m40llm_paged_evict_async(CTX, C.byref(cache()), C.byref(evict(to=C.addressof(to)))) == code


@pytest.mark.parametrize("change,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(row_slot=None), -1), (dict(row_entry=None), -1), (dict(q=None), -1), (dict(q_out=None), -1),
    (dict(turns=None), -1), (dict(row_pos=None), -1), (dict(row_pos=None, pairs=0), -1), (dict(rows=0), -2), (dict(pairs=33), -2),
    (dict(pairs=0x80000001), -2), (dict(rope_layout=2), -2), (dict(ld=511), -2), (dict(ld=127, q_heads=0), -2), (dict(ld_entry=31), -2),
    (dict(ld_entry=31, weights=None), -2), (dict(q_heads=1 << 30), -2)])
def test_append(pkg, change, code):
    assert pkg.native.lib().m40llm_paged_append_async(CTX, C.byref(cache()), C.byref(append(**change))) == code


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(row_slot=None), -1), (dict(row_len=None), -1), (dict(rows=0), -2), (dict(q_heads=0), -2),
    (dict(q_heads=7), -2), (dict(max_len=33), -2), (dict(ld_weights=31), -2), (dict(rows=65536), LIMIT), (dict(q_heads=65536), LIMIT)])
def test_attention(pkg, change, code):
    assert pkg.native.lib().m40llm_attention_paged_async(CTX, C.byref(cache()), C.byref(attention(**change))) == code


@pytest.mark.parametrize("change,code", [
    (dict(seq=None), -1), (dict(len=None), -1), (dict(weights=None), -1), (dict(new_len=None), -1), (dict(count=0), -2), (dict(keep=0), -2),
    (dict(keep=33), -2), (dict(first=5, recent=5), -2), (dict(first=0xffffffff, recent=10), -2), (dict(ld=31), -2), (dict(max_len=33), -2),
    (dict(count=65536), LIMIT)])
def test_evict(pkg, change, code):
    assert pkg.native.lib().m40llm_paged_evict_async(CTX, C.byref(cache()), C.byref(evict(**change))) == code


@pytest.mark.parametrize("change,code", [(dict(kv_heads=1), -2), (dict(head_dim=32), -2), (dict(slots=3), -2), (dict(max_pages=1, page_tokens=8), -2),
                                         (dict(elem_dtype=N.DT_F32), -4)])
def test_evict_to(pkg, change, code):
    to = cache(**change)
    assert pkg.native.lib().m40llm_paged_evict_async(CTX, C.byref(cache()), C.byref(evict(to=C.addressof(to)))) == code


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), -1), (dict(tokens=None), -1), (dict(tokens=None, logprob=None), -1), (dict(tokens=None, rank=None), -1), (dict(rows=0), -2),
    (dict(n=0), -2), (dict(ld=99), -2), (dict(top=65), LIMIT)])
def test_logprobs(pkg, change, code):
    assert pkg.native.lib().m40llm_logprobs_f32_async(CTX, C.byref(logprobs(**change))) == code


def test_null_handles(pkg):
    L = pkg.native.lib()
    assert L.m40llm_paged_append_async(None, C.byref(cache()), C.byref(append())) == -1
    assert L.m40llm_paged_append_async(CTX, None, C.byref(append())) == -1
    assert L.m40llm_attention_paged_async(CTX, C.byref(cache()), None) == -1
    assert L.m40llm_paged_evict_async(CTX, None, None) == -1
    assert L.m40llm_logprobs_f32_async(None, C.byref(logprobs())) == -1
    assert L.m40llm_logprobs_f32_async(CTX, None) == -1


def test_queries_in_place_of_a_packed_projection(pkg):
    """The turned queries are packed rows, so they may take the place of their input only where that is packed too."""
    L = pkg.native.lib()
    assert L.m40llm_paged_append_async(CTX, C.byref(cache()), C.byref(append(ld=8 * 64 + 4, q_out=P))) == -2


@pytest.mark.parametrize("change", [dict(page_tokens=32), dict(max_pages=1), dict(v=2 * P)])
def test_eviction_into_another_view_of_the_same_pages(pkg, change):
    L, to = pkg.native.lib(), cache(**change)
    assert L.m40llm_paged_evict_async(CTX, C.byref(cache()), C.byref(evict(to=C.addressof(to)))) == -2
