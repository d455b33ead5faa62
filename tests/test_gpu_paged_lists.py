"""Attention over a paged cache where its list of tiles is long: rows that every resident CTA has a part of, and rows over several batches of the list."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as T
from paged_cases import N

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


@pytest.mark.parametrize("kind,dim,heads", [("f16", 64, 2), ("f16", 64, 16), ("f16", 128, 4), ("f32", 64, 4), ("f32", 384, 2)])
@pytest.mark.parametrize("length", [33001, 61000])
def test_one_row_of_all_ctas(nat, kind, dim, heads, length):
    """One kv head and one row with a tile or more for every CTA: parts of all warps meet in one join, and in the weights."""
    rng = np.random.default_rng(dim + heads)
    c = T.Cache(nat, rng, 1, length + 100, 1, dim, 64, kind)
    q = (2 * rng.standard_normal((1, heads, dim))).astype(np.float32)
    got, _ = T.attend(nat, c, q, [0], [length])
    T.check_attention(c, q, [0], [length], got)
    w = rng.random((1, 1, c.capacity)).astype(np.float32)
    got, gw = T.attend(nat, c, q, [0], [length], weights=w, ld=c.capacity, in_place=True)
    T.check_attention(c, q, [0], [length], got, weights=w, got_w=gw, before=w)
    assert T.status(nat) == 0


@pytest.mark.parametrize("kind,dim,heads,kv_heads,page", [("f32", 384, 2, 1, 16), ("f16", 64, 8, 2, 16), ("f16", 96, 6, 2, 1)])
@pytest.mark.parametrize("rows", [31, 32, 33, 64, 97, 256, 300])
def test_rows_of_several_batches(nat, kind, dim, heads, kv_heads, page, rows):
    """The tiles before a row are added up 32 rows at a time: rows at the ends of these batches, beside empty ones."""
    rng = np.random.default_rng(rows + dim)
    c = T.Cache(nat, rng, 7, 3000, kv_heads, dim, page, kind)
    slot = np.arange(rows) % 7
    length = rng.integers(0, 400, rows)
    length[31::32], length[0::32], length[5] = 700, 0, 2999
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    got, _ = T.attend(nat, c, q, slot, length, max_len=3000)
    some = np.unique(np.r_[5, np.arange(31, rows, 32), np.arange(30, rows, 32), np.arange(0, rows, 32), np.arange(1, rows, 32), rows - 1])
    T.check_attention(c, q[some], slot[some], length[some], got[some])
    assert T.status(nat) == 0


def test_more_work_than_can_be_counted_is_refused(nat):
    """256 rows of 60 heads that may have 2^30 entries each: refused where nothing says that they are shorter."""
    rng = np.random.default_rng(1)
    c = T.Cache(nat, rng, 1, 16, 60, 260, 16, "f32")
    table = np.full(1 << 26, 0xffffffff, np.uint32)  # the first page is there, the others are outside the pool
    table[0] = c.table[0, 0]
    q = rng.standard_normal((256, 60, 260)).astype(np.float32)
    desc, call, out, _ = T.attention_call(nat, c, q, np.zeros(256), np.full(256, 3))
    desc.table, desc.max_pages = nat.buf(table).ptr, len(table)
    call.max_len = 16
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    T.check_attention(c, q[:2], [0, 0], [3, 3], out.download(np.float32, q.shape)[:2])
    call.max_len = 0
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == N.ERR_LIMIT
    call.rows = 128
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    assert T.status(nat) == 0
