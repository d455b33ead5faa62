"""The paged cache through the C ABI against the float64 statements of oracle/paged_oracle.py: append, attention of single tokens with
accumulated weights, eviction by weight, and a run of the three together."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as T
from paged_cases import N, P

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -11


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


# ------------------------------------------------------------------------------------------------------------------ append
def run_append(nat, c, rng, slot, entry, pos, q_heads, pairs, layout, packed, entry_arrays=True, pad=3):
    rows, kvw, qw = len(slot), c.kv_heads * c.dim, q_heads * c.dim
    q, k, v = (rng.standard_normal((rows, w)).astype(np.float32) for w in (qw, kvw, kvw))
    turns = 10000.0 ** (-np.arange(pairs) / max(1, pairs)) / (2 * np.pi)
    if packed:
        whole = T.f32(nat, np.concatenate([q, k, v, np.full((rows, pad), 9.0, np.float32)], 1))
        ptrs, ld = (whole.ptr, whole.ptr + 4 * qw, whole.ptr + 4 * (qw + kvw)), qw + 2 * kvw + pad
        q_out = T.f32(nat, np.zeros((rows, max(qw, 1))))
    else:
        dq = T.f32(nat, q)
        ptrs, ld, q_out = (dq.ptr, T.f32(nat, k).ptr, T.f32(nat, v).ptr), 0, dq  # in place
    ep = T.u32(nat, np.full((c.slots, c.kv_heads, c.capacity), 77)) if entry_arrays else None
    w = T.f32(nat, np.full((c.slots, c.kv_heads, c.capacity), 3.0)) if entry_arrays else None
    call = N.PagedAppend(ptrs[0] if q_heads else None, ptrs[1], ptrs[2], q_out.ptr if q_heads else None, nat.buf(turns).ptr if pairs else None,
                         T.u32(nat, slot).ptr, T.u32(nat, entry).ptr, T.u32(nat, pos).ptr, ep.ptr if ep else None, w.ptr if w else None, rows, ld,
                         q_heads, pairs, layout, c.capacity if ep else 0)
    desc = c.desc()
    assert nat.lib.m40llm_paged_append_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    return q, k, v, turns, q_out, ep, w


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,pairs,page", [(8, 2, 64, 32, 16), (4, 1, 33, 7, 1), (0, 3, 1, 0, 4), (32, 8, 128, 64, 64),
                                                              (5, 5, 80, 13, 2), (2, 1, 512, 256, 8)])
@pytest.mark.parametrize("layout,packed", [(0, True), (1, True), (1, False), (0, False)])
def test_append(nat, kind, q_heads, kv_heads, dim, pairs, page, layout, packed):
    check_append(nat, kind, q_heads, kv_heads, dim, pairs, page, layout, packed, 3, 0 if packed else 3)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,pairs,page", [(8, 2, 64, 32, 16), (16, 2, 128, 32, 16), (4, 1, 128, 20, 1), (0, 3, 8, 4, 4), (2, 2, 72, 0, 8),
                                                              (32, 8, 128, 64, 64), (3, 1, 512, 256, 2)])
@pytest.mark.parametrize("layout,packed", [(0, True), (1, True), (1, False), (0, False)])
def test_append_eights(nat, kind, q_heads, kv_heads, dim, pairs, page, layout, packed):
    """Rows on 16 bytes, heads of eights, pairs of fours."""
    check_append(nat, kind, q_heads, kv_heads, dim, pairs, page, layout, packed, 4, 0)


def check_append(nat, kind, q_heads, kv_heads, dim, pairs, page, layout, packed, pad, offset):
    rng = np.random.default_rng(dim + pairs + layout)
    c = T.Cache(nat, rng, 3, 37, kv_heads, dim, page, kind, offset=offset)
    slot, entry = np.array([2, 0, 2, 1, 0, 2]), np.array([0, 36, 17, 5, 16, c.capacity - 1])
    pos = np.array([0, 36, 123456, 5, 4000000000, 2])
    q, k, v, turns, q_out, ep, w = run_append(nat, c, rng, slot, entry, pos, q_heads, pairs, layout, packed, pad=pad)
    # an angle is the product of a position and a double, whole turns dropped in double: 2^-53 of the product; sine, cosine, two products and a sum
    def bound(x):
        angle = 2 * np.pi * 2.0 ** -52 * pos[:, None, None] * (turns.max() if pairs else 0.0)
        other = np.abs(x).max(-1, keepdims=True)
        return (8 * U32 + angle) * (np.abs(x) + other)
    heads = lambda a: a.reshape(len(slot), -1, dim)  # noqa: E731
    if q_heads:
        got = heads(q_out.download(np.float32, (len(slot), q_heads * dim)))
        assert (np.abs(got - P.turned(heads(q), pos, turns, layout)) <= bound(heads(q))).all()
    want_k, err_k, want_v = P.turned(heads(k), pos, turns, layout), bound(heads(k)), heads(v)
    gk, gv = c.download()
    half = U16 if kind == "f16" else U32
    for r in range(len(slot)):
        page_, at = c.table[slot[r], entry[r] // page], entry[r] % page
        assert (np.abs(gk[page_, :, at] - want_k[r]) <= err_k[r] + half * np.abs(want_k[r]) + 2.0 ** -25).all()
        assert np.array_equal(gv[page_, :, at], want_v[r].astype(c.dtype))
        gk[page_, :, at], gv[page_, :, at] = c.k[page_, :, at], c.v[page_, :, at]
    assert np.array_equal(gk, c.k) and np.array_equal(gv, c.v), "other entries changed"
    want_p, want_w = np.full((3, kv_heads, c.capacity), 77), np.full((3, kv_heads, c.capacity), 3.0)
    for r in range(len(slot)):
        want_p[slot[r], :, entry[r]], want_w[slot[r], :, entry[r]] = pos[r], 0
    assert np.array_equal(ep.download(np.uint32, want_p.shape), want_p) and np.array_equal(w.download(np.float32, want_w.shape), want_w)
    assert T.status(nat) == 0


def test_append_outside(nat):
    """Rows outside the cache and pages outside the pool are left out, the others are done."""
    rng = np.random.default_rng(5)
    c = T.Cache(nat, rng, 3, 40, 2, 64, 8)
    c.table[1, 2] = c.pages  # one too high
    c.upload()
    slot, entry = np.array([3, 0, 1, 0xffffffff, 2, 1]), np.array([0, c.capacity, 17, 1, 3, 1])
    q, k, v, *_ = run_append(nat, c, rng, slot, entry, slot * 0, 4, 0, 0, True)
    gk, gv = c.download()
    for r in (4, 5):
        at = (c.table[slot[r], entry[r] // 8], slice(None), entry[r] % 8)
        c.k[at], c.v[at] = k[r].reshape(2, 64), v[r].reshape(2, 64)
    assert np.array_equal(gk, c.k) and np.array_equal(gv, c.v)
    assert T.status(nat) == 2


# --------------------------------------------------------------------------------------------------------------- attention
LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 200]
SHAPES = [(8, 2, 64, 16), (4, 4, 128, 32), (7, 1, 128, 1), (10, 2, 64, 2), (9, 1, 64, 64), (16, 1, 128, 128), (17, 1, 64, 16), (40, 2, 128, 16),
          (3, 3, 256, 16), (12, 2, 96, 8), (5, 1, 80, 4), (6, 2, 33, 16), (2, 2, 1, 8), (8, 1, 512, 16), (2, 1, 384, 32), (6, 1, 4, 16)]


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("entries", [200, 300])
def test_attention_shapes(nat, kind, q_heads, kv_heads, dim, page, entries):
    rng = np.random.default_rng(q_heads * 1000 + dim + page)
    c = T.Cache(nat, rng, len(LENS), entries, kv_heads, dim, page, kind)
    q = (2 * rng.standard_normal((len(LENS), q_heads, dim))).astype(np.float32)
    slot = rng.permutation(len(LENS))
    got, _ = T.attend(nat, c, q, slot, LENS)
    T.check_attention(c, q, slot, LENS, got)
    assert not got[0].any() and T.status(nat) == 0


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f16", 64), ("f32", 128), ("f16", 96)])
@pytest.mark.parametrize("max_len", [0, 3001])
def test_attention_many_chunks(nat, kind, dim, max_len):
    rng = np.random.default_rng(dim)
    c = T.Cache(nat, rng, 2, 5000, 2, dim, 16, kind)
    q = (2 * rng.standard_normal((2, 8, dim))).astype(np.float32)
    got, _ = T.attend(nat, c, q, [1, 0], [3001, 777], max_len=max_len)
    T.check_attention(c, q, [1, 0], [3001, 777], got)


@pytest.mark.parametrize("kind,dim,heads", [("f16", 128, 8), ("f16", 64, 24), ("f32", 64, 8), ("f16", 80, 8)])
def test_attention_window(nat, kind, dim, heads):
    rng = np.random.default_rng(dim + heads)
    c = T.Cache(nat, rng, 5, 700, 2, dim, 32, kind)
    q = (2 * rng.standard_normal((7, heads, dim))).astype(np.float32)
    slot, length, begin = [0, 1, 2, 3, 4, 0, 1], [700, 700, 65, 300, 1, 128, 0], [0, 63, 64, 300, 5, 1, 0xffffffff]
    got, _ = T.attend(nat, c, q, slot, length, begin=begin, max_len=700)
    T.check_attention(c, q, slot, length, got, begin=[min(b, n) for b, n in zip(begin, length)])
    assert not got[3].any() and not got[4].any() and not got[6].any() and T.status(nat) == 0


@pytest.mark.parametrize("kind,dim,offset", [("f16", 128, 0), ("f16", 64, 0), ("f16", 64, 1), ("f32", 64, 0), ("f32", 64, 1), ("f16", 36, 0), ("f16", 96, 0)])
@pytest.mark.parametrize("entries,max_len", [(300, 0), (300, 200), (5000, 0)])
def test_attention_ignores_what_is_masked(nat, kind, dim, offset, entries, max_len):
    """Infinities and NaN behind a row's entries, before its window, on its last page and on other pages do not reach the output."""
    rng = np.random.default_rng(dim + offset)
    c = T.Cache(nat, rng, 4, entries, 2, dim, 16, kind, offset=offset)
    length, begin = [1, 130, 200, 64], [0, 3, 70, 0]
    q = (2 * rng.standard_normal((4, 8, dim))).astype(np.float32)
    seen = np.zeros((c.pages, 16), bool)
    for s in range(4):
        for e in range(begin[s], length[s]):
            seen[c.table[s, e // 16], e % 16] = True
    bad = np.array([np.inf, -np.inf, np.nan, np.finfo(c.dtype).min], c.dtype)
    for pool in (c.k, c.v):
        pool.transpose(0, 2, 1, 3)[~seen] = rng.choice(bad, pool.transpose(0, 2, 1, 3)[~seen].shape)
    c.upload()
    got, _ = T.attend(nat, c, q, [0, 1, 2, 3], length, begin=begin, max_len=max_len)
    T.check_attention(c, q, [0, 1, 2, 3], length, got, begin=begin)


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f32", 128)])
@pytest.mark.parametrize("n", [300, 230, 5000])
def test_attention_values_that_are_not_finite(nat, kind, dim, n):
    """What a row does see reaches its output as the formula says; the rows beside it keep theirs."""
    rng = np.random.default_rng(1)
    c = T.Cache(nat, rng, 3, n, 1, dim, 16, kind)
    at = lambda s, e: (c.table[s, e // 16], 0, e % 16)  # noqa: E731
    c.v[at(0, 5)][3] = np.inf
    c.k[at(1, 200)][0] = np.nan
    c.upload()
    q = rng.standard_normal((3, 4, dim)).astype(np.float32)
    got, _ = T.attend(nat, c, q, [0, 1, 2], [n, n, n])
    assert (got[0][:, 3] == np.inf).all() and np.isfinite(np.delete(got[0], 3, 1)).all()
    assert np.isnan(got[1]).all()
    T.check_attention(c, q[2:], [2], [n], got[2:])


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f16", 64), ("f32", 40)])
def test_attention_large_and_small_scores(nat, kind, dim):
    """Scores of a few hundred and weights that differ by many powers of ten."""
    rng = np.random.default_rng(2)
    c = T.Cache(nat, rng, 2, 600, 1, dim, 16, kind)
    q = (np.array([30.0, 1e-6])[:, None, None] * rng.standard_normal((2, 3, dim))).astype(np.float32)
    got, _ = T.attend(nat, c, q, [0, 1], [600, 600])
    T.check_attention(c, q, [0, 1], [600, 600], got)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 32, 4), (128, 16, 2), (128, 16, 1), (64, 9, 1), (128, 3, 3)])
@pytest.mark.parametrize("rows", [1, 2, 5, 24, 150])
@pytest.mark.parametrize("entries", [70, 250, 1000, 2000])
def test_attention_clusters(nat, dim, heads, kv_heads, rows, entries):
    """Few rows and many, bounds on both sides of the sizes that clusters take; rows shorter than the cluster's shares, empty ones, windows, and their weights."""
    rng = np.random.default_rng(rows + entries + dim)
    slots = min(rows, 6)
    c = T.Cache(nat, rng, slots, entries, kv_heads, dim, 16)
    slot = np.arange(rows) % slots
    length = rng.integers(0, entries + 1, rows)
    length[0] = entries
    if rows > 3:
        length[1:4] = 0, 1, 65
    begin = np.where(rng.random(rows) < 0.3, length // 2, 0)
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    some = np.unique(np.r_[0, rng.integers(0, rows, 6), np.minimum(rows - 1, [1, 2, 3])])
    got, _ = T.attend(nat, c, q, slot, length, begin=begin, max_len=entries)
    T.check_attention(c, q[some], slot[some], length[some], got[some], begin=begin[some])
    again, _ = T.attend(nat, c, q, slot, length, begin=begin, max_len=entries)
    assert np.array_equal(got, again) and T.status(nat) == 0
    if rows <= 5:
        w = rng.random((slots, kv_heads, c.capacity)).astype(np.float32)
        got, gw = T.attend(nat, c, q, slot, length, begin=begin, max_len=entries, weights=w, ld=c.capacity, in_place=True)
        T.check_attention(c, q, slot, length, got, begin=begin, weights=w, got_w=gw, before=w)


@pytest.mark.parametrize("kind,dim,heads,kv_heads,page", [("f16", 64, 32, 4, 16), ("f16", 128, 16, 2, 1), ("f16", 128, 40, 2, 128), ("f16", 64, 17, 1, 2),
                                                          ("f16", 128, 4, 4, 64), ("f32", 128, 8, 1, 16), ("f16", 96, 6, 2, 4), ("f16", 33, 4, 2, 16)])
@pytest.mark.parametrize("rows", [9, 270])
def test_attention_long_bounds(nat, kind, dim, heads, kv_heads, page, rows):
    """A bound of 20000 entries for rows of any length: the smallest, empty ones, windows, a page outside the pool, rows outside the cache, and weights."""
    rng = np.random.default_rng(rows + page + dim)
    c = T.Cache(nat, rng, 9, 20000, kv_heads, dim, page, kind)
    slot = np.arange(rows) % 9
    length = rng.choice(LENS, rows)
    length[:9] = 3000, 1, 0, 77, 64, 5000, 16, 2, 400
    begin = np.where(rng.random(rows) < 0.3, length // 2, 0)
    begin[:9] = 0, 0, 0, 5, 64, 1003, 0, 0, 0
    c.table[8, 130 // page] = c.pages  # entry 130 of slot 8
    c.upload()
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    some = np.unique(np.r_[np.arange(9), rng.integers(0, rows, 20)])
    got, _ = T.attend(nat, c, q, slot, length, begin=begin)
    T.check_attention(c, q[some], slot[some], length[some], got[some], begin=begin[some])
    assert T.status(nat) == 1 and not got[length <= begin].any()
    w = rng.random((9, kv_heads, c.capacity)).astype(np.float32)
    got, gw = T.attend(nat, c, q[:9], slot[:9], length[:9], begin=begin[:9], weights=w, ld=c.capacity, in_place=True)
    T.check_attention(c, q[:9], slot[:9], length[:9], got, begin=begin[:9], weights=w, got_w=gw, before=w)
    outside = length.copy()
    outside[3], slot[4] = c.capacity + 1, 9
    got2, _ = T.attend(nat, c, q, slot, outside, begin=begin)
    assert not got2[3:5].any() and np.array_equal(got2[5:9], T.attend(nat, c, q, slot, outside, begin=begin)[0][5:9]) and T.status(nat) == 1
    T.check_attention(c, q[5:9], slot[5:9], length[5:9], got2[5:9], begin=begin[5:9])


@pytest.mark.parametrize("kind,dim,heads", [("f16", 128, 8), ("f16", 64, 12), ("f32", 64, 8), ("f16", 40, 8)])
@pytest.mark.parametrize("queries,keys", [(1e-5, 4096.0), (1e-12, 8192.0), (1e6, 1e-3)])
@pytest.mark.parametrize("entries", [600, 5000])
def test_attention_sizes_of_queries_and_keys(nat, kind, dim, heads, queries, keys, entries):
    """Queries far from 1 keep their bits: the scores are what they are for queries and keys that share the size."""
    rng = np.random.default_rng(3)
    c = T.Cache(nat, rng, 2, entries, 1, dim, 16, kind)
    c.k = (c.k.astype(np.float32) * np.float32(keys)).astype(c.dtype)
    c.upload()
    q = (queries * rng.standard_normal((2, heads, dim))).astype(np.float32)
    got, _ = T.attend(nat, c, q, [0, 1], [600, 130])
    T.check_attention(c, q, [0, 1], [600, 130], got)


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f32", 64), ("f16", 20)])
@pytest.mark.parametrize("n", [100, 700, 5000])
def test_attention_weights_where_nothing_is_seen(nat, kind, dim, n):
    """Rows whose pages are all outside the pool, and rows whose scores are all -inf: zeros, and the weights stay."""
    rng = np.random.default_rng(4)
    c = T.Cache(nat, rng, 3, n, 1, dim, 16, kind)
    c.table[1] = 0xffffffff
    for page in c.table[2]:
        c.k[page] = -np.inf
    c.upload()
    w = rng.random((3, 1, c.capacity)).astype(np.float32)
    q = np.abs(rng.standard_normal((3, 2, dim))).astype(np.float32) + np.float32(0.1)
    got, gw = T.attend(nat, c, q, [0, 1, 2], [n, n, n], weights=w, ld=c.capacity)
    assert not got[1].any() and not got[2].any() and np.array_equal(gw[1:, :, :n], w[1:, :, :n]) and T.status(nat) == 1
    T.check_attention(c, q[:1], [0], [n], got[:1])


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f16", 64), ("f32", 64), ("f16", 20)])
def test_attention_outside(nat, kind, dim):
    """Rows outside the cache give zeros and status bit 1; entries on a page outside the pool are masked."""
    rng = np.random.default_rng(3)
    c = T.Cache(nat, rng, 3, 400, 2, dim, 16, kind)
    q = rng.standard_normal((5, 4, dim)).astype(np.float32)
    slot, length = [3, 0, 1, 0xffffffff, 2], [10, c.capacity + 1, 200, 1, 400]
    got, _ = T.attend(nat, c, q, slot, length)
    assert not got[[0, 1, 3]].any() and T.status(nat) == 1
    T.check_attention(c, q[[2, 4]], [1, 2], [200, 400], got[[2, 4]])
    got, _ = T.attend(nat, c, q, [0, 0, 1, 1, 2], [100, 101, 100, 0, 100], max_len=100)
    assert not got[[1, 3]].any() and T.status(nat) == 1
    c.table[2, 3], c.table[1, 0] = 0xffffffff, c.pages
    c.upload()
    got, _ = T.attend(nat, c, q[:3], [0, 1, 2], [399, 16, 400])
    T.check_attention(c, q[:3], [0, 1, 2], [399, 16, 400], got)
    assert not got[1].any() and T.status(nat) == 1


def test_attention_rows_share_slots_and_pages(nat):
    rng = np.random.default_rng(4)
    c = T.Cache(nat, rng, 2, 300, 2, 64, 16)
    c.table[1, :5] = c.table[0, :5]  # a common beginning
    c.upload()
    q = rng.standard_normal((4, 8, 64)).astype(np.float32)
    got, _ = T.attend(nat, c, q, [0, 1, 1, 0], [200, 201, 202, 80])
    T.check_attention(c, q, [0, 1, 1, 0], [200, 201, 202, 80], got)


@pytest.mark.parametrize("kind,dim,heads,kv_heads", [("f16", 128, 8, 2), ("f16", 64, 32, 2), ("f32", 64, 4, 4), ("f16", 72, 6, 2), ("f16", 64, 20, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_attention_weights_of_short_rows(nat, kind, dim, heads, kv_heads, in_place):
    rng = np.random.default_rng(dim + heads)
    c = T.Cache(nat, rng, 5, 240, kv_heads, dim, 16, kind)
    w = rng.random((5, kv_heads, c.capacity)).astype(np.float32)
    slot, length, begin = [3, 1, 3, 0, 3, 4], [200, 130, 201, 0, 100, 1], [0, 10, 0, 0, 64, 0]
    q = (2 * rng.standard_normal((6, heads, dim))).astype(np.float32)
    got, gw = T.attend(nat, c, q, slot, length, begin=begin, weights=w, ld=c.capacity, in_place=in_place)
    T.check_attention(c, q, slot, length, got, begin=begin, weights=w, got_w=gw, before=w if in_place else np.full(w.shape, -5.0, np.float32))


@pytest.mark.parametrize("kind,dim,heads,kv_heads", [("f16", 128, 8, 2), ("f16", 64, 32, 2), ("f32", 64, 4, 4), ("f16", 72, 6, 2), ("f16", 64, 20, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_attention_weights(nat, kind, dim, heads, kv_heads, in_place):
    """Accumulated weights: several rows of a slot, rows in any order, a window, an empty row, slots without rows."""
    rng = np.random.default_rng(dim + heads)
    c = T.Cache(nat, rng, 5, 900, kv_heads, dim, 32, kind)
    ld = c.capacity + 5
    w = rng.random((5, kv_heads, ld)).astype(np.float32)
    slot, length, begin = [3, 1, 3, 0, 3, 4], [850, 300, 851, 0, 100, 1], [0, 10, 0, 0, 64, 0]
    q = (2 * rng.standard_normal((6, heads, dim))).astype(np.float32)
    got, gw = T.attend(nat, c, q, slot, length, begin=begin, weights=w, ld=ld, in_place=in_place)
    T.check_attention(c, q, slot, length, got, begin=begin, weights=w, got_w=gw, before=w if in_place else np.full(w.shape, -5.0, np.float32))
    again, gw2 = T.attend(nat, c, q, slot, length, begin=begin, weights=w, ld=ld, in_place=in_place)
    assert np.array_equal(got, again) and np.array_equal(gw, gw2), "the same call twice"


def test_attention_weights_with_rows_outside(nat):
    """A slot with a row outside the cache keeps its weights; the others get theirs."""
    rng = np.random.default_rng(6)
    c = T.Cache(nat, rng, 3, 200, 2, 64, 16)
    w = rng.random((3, 2, c.capacity)).astype(np.float32)
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    slot, length = [0, 1, 0, 9], [100, 150, c.capacity + 1, 5]
    got, gw = T.attend(nat, c, q, slot, length, weights=w, ld=c.capacity, in_place=True)
    assert np.array_equal(gw[0], w[0]) and np.array_equal(gw[2], w[2]) and T.status(nat) == 1
    T.check_attention(c, q[1:2], [1], [150], got[1:2], weights=w, got_w=gw, before=w)


def test_attention_without_weights_before(nat):
    """weights_in null counts as zeros."""
    rng = np.random.default_rng(7)
    c = T.Cache(nat, rng, 1, 200, 2, 64, 16)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    zeros = np.zeros((1, 2, c.capacity), np.float32)
    desc, call, out, w_out = T.attention_call(nat, c, q, [0], [150], weights=zeros, ld=c.capacity)
    call.weights_in = None
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    T.check_attention(c, q, [0], [150], out.download(np.float32, q.shape), weights=zeros, got_w=w_out.download(np.float32, zeros.shape),
                      before=np.full(zeros.shape, -5.0, np.float32))


@pytest.mark.parametrize("dim", [128, 40])
def test_attention_beyond_32_bits(nat, dim):
    """The last pages of a pool of more than 2^32 elements."""
    rng = np.random.default_rng(8)
    pages = (1 << 32) // (8 * 64 * dim) + 5
    small = T.Cache(nat, rng, 1, 512, 8, dim, 64, spare=0)
    per = 8 * 64 * dim * 2
    big = [nat.buf(pages * per) for _ in range(2)]
    for b, a in zip(big, (small.k, small.v)):
        assert nat.lib.m40llm_memcpy_h2d(nat.ctx, b.ptr + (pages - 8) * per, a.ctypes.data_as(C.c_void_p), a.nbytes) == 0
    q = rng.standard_normal((1, 8, dim)).astype(np.float32)
    desc, call, out, _ = T.attention_call(nat, small, q, [0], [500])
    desc.k, desc.v, desc.pages, desc.table = big[0].ptr, big[1].ptr, pages, T.u32(nat, small.table + pages - 8).ptr
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    T.check_attention(small, q, [0], [500], out.download(np.float32, q.shape))
    assert T.status(nat) == 0


@pytest.mark.parametrize("entries", [2000, 9000])
def test_attention_captured(nat, entries):
    """A captured step is replayed while lengths and tables change; a second graph, captured later and larger, leaves the first one right."""
    rng = np.random.default_rng(9)
    c = T.Cache(nat, rng, 3, entries, 2, 128, 16)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    w = np.zeros((3, 2, c.capacity), np.float32)
    L = nat.lib

    def capture(weights):
        length = T.u32(nat, [5, 6, 7])
        desc, call, out, w_out = T.attention_call(nat, c, q, [0, 1, 2], [5, 6, 7], weights=w if weights else None, ld=c.capacity)
        call.row_len = length.ptr
        assert L.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
        nat.sync(1)
        graph = C.c_void_p()
        assert L.m40llm_cuda_graph_begin_capture(nat.ctx, 1) == 0
        assert L.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
        assert L.m40llm_cuda_graph_end_capture(nat.ctx, 1, C.byref(graph)) == 0
        return graph, length, out, w_out

    first, second = capture(False), capture(True)
    for length in ([1999, 1, 500], [0, 2000, 64]):
        for graph, d_len, out, w_out in (first, second, first):
            d_len.upload(np.array(length, np.uint32))
            assert L.m40llm_cuda_graph_launch(nat.ctx, graph, 1) == 0
            nat.sync(1)
            T.check_attention(c, q, [0, 1, 2], length, out.download(np.float32, q.shape))
    for graph, *_ in (first, second):
        L.m40llm_cuda_graph_destroy(graph)


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("f16", 64), ("f32", 64), ("f16", 96)])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_attention_queries_anywhere(nat, kind, dim, shift):
    """Queries that lie on 4, 8 and 12 bytes behind a 16-byte boundary."""
    rng = np.random.default_rng(shift)
    c = T.Cache(nat, rng, 2, 200, 2, dim, 16, kind)
    q = rng.standard_normal((2, 6, dim)).astype(np.float32)
    desc, call, out, _ = T.attention_call(nat, c, q, [1, 0], [200, 33])
    call.q = T.f32(nat, np.concatenate([np.zeros(shift), q.ravel()])).ptr + 4 * shift
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    T.check_attention(c, q, [1, 0], [200, 33], out.download(np.float32, q.shape))


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("f32", 32)])
def test_attention_many_rows(nat, kind, dim):
    """More rows than a launch takes, several of a slot, with their weights."""
    rng = np.random.default_rng(21)
    c = T.Cache(nat, rng, 40, 150, 1, dim, 16, kind)
    rows = 600
    q = rng.standard_normal((rows, 2, dim)).astype(np.float32)
    slot, length = rng.integers(0, 40, rows), rng.integers(0, 151, rows)
    w = rng.random((40, 1, c.capacity)).astype(np.float32)
    got, gw = T.attend(nat, c, q, slot, length, weights=w, ld=c.capacity, in_place=True)
    T.check_attention(c, q, slot, length, got, weights=w, got_w=gw, before=w)
    assert T.status(nat) == 0


# ---------------------------------------------------------------------------------------------------------------- eviction
def run_evict(nat, c, seq, length, keep, first, recent, weights, pos, to=None, in_place=True, max_len=0, origin=True):
    ld = weights.shape[2]
    w, p = T.f32(nat, weights), None if pos is None else T.u32(nat, pos)
    w_out = w if in_place else T.f32(nat, np.full(weights.shape, -5.0))
    p_out = p if in_place else T.u32(nat, np.full(weights.shape, 4242))
    org = T.u32(nat, np.full((len(seq), c.kv_heads, keep), 99)) if origin else None
    new = T.u32(nat, np.full(len(seq), 99))
    desc, dto = c.desc(), None if to is None else to.desc()
    call = N.PagedEvict(None if to is None else C.addressof(dto), T.u32(nat, seq).ptr, T.u32(nat, length).ptr, w.ptr, w_out.ptr,
                        None if p is None else p.ptr, None if p_out is None else p_out.ptr, org.ptr if org else None, new.ptr, len(seq), keep, first, recent,
                        ld, max_len)
    assert nat.lib.m40llm_paged_evict_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    return (org.download(np.uint32, (len(seq), c.kv_heads, keep)) if org else None, new.download(np.uint32, len(seq)),
            w_out.download(np.float32, weights.shape), None if p_out is None else p_out.download(np.uint32, weights.shape))


def check_evict(c, seq, length, keep, first, recent, weights, pos, got, to=None, in_place=True, before=None):
    """before: the target's pools as they were."""
    origin, new_len, w_out, p_out = got
    target = to or c
    gk, gv = target.download()
    wk, wv = (a.copy() for a in before)
    want_w = weights.copy() if in_place else np.full(weights.shape, -5.0, np.float32)
    index = np.broadcast_to(np.arange(weights.shape[2], dtype=np.uint32), weights.shape)
    places = index if pos is None else pos
    want_p = places.copy() if in_place else np.full(weights.shape, 4242, np.uint32)
    for i, s in enumerate(seq):
        left = min(length[i], keep)
        assert new_len[i] == left
        for h in range(c.kv_heads):
            if left == 0:
                continue
            org = P.evict(weights[s, h], places[s, h], first, recent, keep, length[i])
            if origin is not None:
                assert np.array_equal(origin[i, h, :left], org) and (origin[i, h, left:] == P.NONE).all()
            want_w[s, h, :left], want_p[s, h, :left] = weights[s, h, org], places[s, h, org]
            for e, o in enumerate(org):
                src, dst = (c.table[s, o // c.page], h, o % c.page), (target.table[s, e // target.page], h, e % target.page)
                wk[dst], wv[dst] = c.k[src], c.v[src]
    assert np.array_equal(gk, wk) and np.array_equal(gv, wv)
    assert np.array_equal(w_out, want_w, equal_nan=True)
    if p_out is not None:
        assert np.array_equal(p_out, want_p)


def heavy_tailed(rng, shape):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    w[rng.random(shape) < 0.2] = 0
    return w


@pytest.mark.parametrize("kind,dim,page", [("f16", 128, 16), ("f16", 64, 1), ("f32", 64, 32), ("f16", 33, 8), ("f32", 3, 4)])
@pytest.mark.parametrize("where", ["in place", "other arrays", "other pages"])
@pytest.mark.parametrize("keep,first,recent", [(100, 0, 0), (64, 4, 20), (1, 0, 1), (300, 10, 290), (399, 399, 0)])
def test_evict(nat, kind, dim, page, where, keep, first, recent):
    rng = np.random.default_rng(keep + dim)
    c = T.Cache(nat, rng, 5, 400, 2, dim, page, kind)
    to = T.Cache(nat, rng, 6, keep, 2, dim, 16, kind) if where == "other pages" else None
    seq, length = [4, 0, 2, 3], [400, keep, min(keep + 1, 400), 0]
    w = heavy_tailed(rng, (5, 2, c.capacity + 3))
    pos = np.argsort(rng.random((5, 2, c.capacity + 3)), -1).astype(np.uint32)
    in_place, target = where == "in place", to or c
    got = run_evict(nat, c, seq, length, keep, first, recent, w, pos, to, in_place)
    check_evict(c, seq, length, keep, first, recent, w, pos, got, to, in_place, (target.k, target.v))
    assert T.status(nat) == 0


@pytest.mark.parametrize("name", ["ties", "zeros", "nan", "infinite", "signed", "equal positions", "close"])
@pytest.mark.parametrize("positions", [True, False])
def test_evict_order(nat, name, positions):
    """Ties go to the lower entry; NaN is the least; -0 and 0 are equal; neighbours that differ in the last bit are told apart."""
    rng = np.random.default_rng(len(name))
    c = T.Cache(nat, rng, 1, 3000, 1, 8, 64)
    n, keep = 2900, 1100
    w = heavy_tailed(rng, (1, 1, c.capacity))
    if name == "ties":
        w = np.floor(w)
    elif name == "zeros":
        w[:] = 0
    elif name == "nan":
        w[rng.random(w.shape) < 0.8] = np.nan
    elif name == "infinite":
        w[rng.random(w.shape) < 0.3] = np.inf
        w[rng.random(w.shape) < 0.5] = -np.inf
    elif name == "signed":
        w = np.where(rng.random(w.shape) < 0.5, np.float32(-0.0), np.float32(0.0)) + np.where(rng.random(w.shape) < 0.3, -w, 0).astype(np.float32)
    elif name == "close":
        w = (np.float32(1.0).view(np.uint32) + rng.integers(0, 700, w.shape).astype(np.uint32)).view(np.float32)
    pos = np.argsort(rng.random(w.shape), -1).astype(np.uint32) if positions else None
    if positions and name == "equal positions":
        pos[:] = 5  # all of them among the newest: the lowest entries stay
    got = run_evict(nat, c, [0], [n], keep, 7, 13, w, pos, in_place=False)
    check_evict(c, [0], [n], keep, 7, 13, w, pos, got, None, False, (c.k, c.v))


@pytest.mark.parametrize("n,keep,heads", [(30000, 4097, 3), (70000, 69999, 1), (70001, 33, 2), (1025, 1024, 1), (400001, 5000, 1)])
def test_evict_long(nat, n, keep, heads):
    rng = np.random.default_rng(n)
    c = T.Cache(nat, rng, 2, n, heads, 8, 128, spare=1)
    w = heavy_tailed(rng, (2, heads, c.capacity))
    got = run_evict(nat, c, [1], [n], keep, 4, 16, w, None, in_place=False, max_len=n)
    check_evict(c, [1], [n], keep, 4, 16, w, None, got, None, False, (c.k, c.v))


def test_evict_without_origins_in_place_twice(nat):
    """origin may be null; a second eviction to the same length changes nothing."""
    rng = np.random.default_rng(11)
    c = T.Cache(nat, rng, 2, 300, 2, 16, 16)
    w = heavy_tailed(rng, (2, 2, c.capacity))
    got = run_evict(nat, c, [1], [300], 50, 2, 10, w, None, in_place=True, origin=False)
    check_evict(c, [1], [300], 50, 2, 10, w, None, got, None, True, (c.k, c.v))
    c.k, c.v = c.download()
    got2 = run_evict(nat, c, [1], [50], 50, 2, 10, got[2], None, in_place=True, origin=False)
    assert np.array_equal(got2[2], got[2]) and all(np.array_equal(a, b) for a, b in zip(c.download(), (c.k, c.v)))


@pytest.mark.parametrize("n", [5000, 300])
def test_evict_lengths_in_place(nat, n):
    """new_len may be the array of the lengths."""
    rng = np.random.default_rng(12)
    c = T.Cache(nat, rng, 3, n, 2, 64, 16)
    keep, length = 200, [n, 150, n - 7]
    w = rng.random((3, 2, c.capacity)).astype(np.float32)
    d_len, d_w = T.u32(nat, length), T.f32(nat, w)
    origin = T.u32(nat, np.zeros((3, 2, keep)))
    call = N.PagedEvict(seq=T.u32(nat, [0, 1, 2]).ptr, len=d_len.ptr, weights=d_w.ptr, weights_out=d_w.ptr, origin=origin.ptr, new_len=d_len.ptr, count=3,
                        keep=keep, ld=c.capacity)
    desc = c.desc()
    assert nat.lib.m40llm_paged_evict_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    assert d_len.download(np.uint32, 3).tolist() == [200, 150, 200] and T.status(nat) == 0
    got = origin.download(np.uint32, (3, 2, keep))
    for i in range(3):
        m = min(length[i], keep)
        for h in range(2):
            best = np.argsort(-w[i, h, :length[i]], kind="stable")[:m]
            assert np.array_equal(np.sort(got[i, h, :m]), np.sort(best)) and (got[i, h, m:] == 0xffffffff).all()


def test_evict_outside(nat):
    """Slots outside the cache, lengths beyond the bound and a slot named twice keep nothing and touch nothing; the others are done. Entries on pages outside the
    pool are not copied."""
    rng = np.random.default_rng(12)
    c = T.Cache(nat, rng, 4, 200, 2, 16, 16)
    w = heavy_tailed(rng, (4, 2, c.capacity))
    seq, length = [4, 1, 0xffffffff, 1, 2, 3], [100, 150, 5, 160, 181, 0]
    origin, new_len, w_out, p_out = run_evict(nat, c, seq, length, 40, 2, 8, w, None, in_place=True, max_len=180)
    assert list(new_len) == [0, 40, 0, 0, 0, 0] and (origin[[0, 2, 3, 4, 5]] == P.NONE).all()
    check_evict(c, [1], [150], 40, 2, 8, w, None, (origin[1:2], new_len[1:2], w_out, None), None, True, (c.k, c.v))
    assert T.status(nat) == 1
    c.k, c.v = c.download()
    c.table[0, 9] = c.pages
    c.upload()
    origin, new_len, *_ = run_evict(nat, c, [0], [160], 40, 0, 10, w, None, in_place=True)
    late = origin[0] >= 144
    assert new_len[0] == 40 and late.any() and T.status(nat) == 1
    gk, _ = c.download()
    for h in range(2):
        for e, o in enumerate(origin[0, h]):
            dst = (c.table[0, e // 16], h, e % 16)
            src = dst if o >= 144 else (c.table[0, o // 16], h, o % 16)
            assert np.array_equal(gk[dst], c.k[src])


def test_evict_captured(nat):
    """A captured eviction is replayed on other weights and lengths."""
    rng = np.random.default_rng(31)
    c = T.Cache(nat, rng, 3, 2500, 2, 16, 16)
    keep, L = 700, nat.lib
    w = heavy_tailed(rng, (3, 2, c.capacity))
    d_w, d_len, d_seq = T.f32(nat, w), T.u32(nat, [9, 9, 9]), T.u32(nat, [2, 0, 1])
    w_out, origin, new = T.f32(nat, w), T.u32(nat, np.zeros((3, 2, keep))), T.u32(nat, np.zeros(3))
    to = T.Cache(nat, rng, 3, keep, 2, 16, 64)
    desc, dto = c.desc(), to.desc()
    call = N.PagedEvict(C.addressof(dto), d_seq.ptr, d_len.ptr, d_w.ptr, w_out.ptr, None, None, origin.ptr, new.ptr, 3, keep, 3, 50, c.capacity, 0)
    run = lambda: L.m40llm_paged_evict_async(nat.ctx, C.byref(desc), C.byref(call))  # noqa: E731
    assert run() == 0
    nat.sync(1)
    graph = C.c_void_p()
    assert L.m40llm_cuda_graph_begin_capture(nat.ctx, 1) == 0
    assert run() == 0
    assert L.m40llm_cuda_graph_end_capture(nat.ctx, 1, C.byref(graph)) == 0
    for lens in ([2500, 700, 1], [0, 701, 1999]):
        w = heavy_tailed(rng, w.shape)
        d_w.upload(w)
        d_len.upload(np.array(lens, np.uint32))
        w_out.upload(np.full(w.shape, -5.0, np.float32))
        before = to.download()
        assert L.m40llm_cuda_graph_launch(nat.ctx, graph, 1) == 0
        nat.sync(1)
        got = origin.download(np.uint32, (3, 2, keep)), new.download(np.uint32, 3), w_out.download(np.float32, w.shape), None
        check_evict(c, [2, 0, 1], lens, keep, 3, 50, w, None, got, to, False, before)
    L.m40llm_cuda_graph_destroy(graph)


# ------------------------------------------------------------------------------------------------------------- all together
def test_a_run_of_appends_attention_and_evictions(nat):
    """Tokens go in one by one, the weights grow, and the cache is cut back whenever it has 96 entries; every output equals what the same
    run gives in float64, from the entries that the float64 run kept."""
    rng = np.random.default_rng(13)
    slots, kv_heads, q_heads, dim, page, keep, most = 2, 2, 8, 64, 16, 64, 96
    c = T.Cache(nat, rng, slots, most, kv_heads, dim, page)
    c.k[:], c.v[:] = 0, 0
    c.upload()
    ld, pairs = c.capacity, 32
    turns = 10000.0 ** (-np.arange(pairs) / pairs) / (2 * np.pi)
    d_turns, ep, w = nat.buf(turns), T.u32(nat, np.zeros((slots, kv_heads, ld))), T.f32(nat, np.zeros((slots, kv_heads, ld)))
    d_slot, d_entry, d_pos, d_len, d_new = (T.u32(nat, np.zeros(slots)) for _ in range(5))
    d_slot.upload(np.arange(slots, dtype=np.uint32))
    width = (q_heads + 2 * kv_heads) * dim
    packed, q_out, out = (nat.buf(4 * slots * n) for n in (width, q_heads * dim, q_heads * dim))
    append = N.PagedAppend(packed.ptr, packed.ptr + 4 * q_heads * dim, packed.ptr + 4 * (q_heads + kv_heads) * dim, q_out.ptr, d_turns.ptr, d_slot.ptr,
                           d_entry.ptr, d_pos.ptr, ep.ptr, w.ptr, slots, width, q_heads, pairs, 1, ld)
    attention = N.PagedAttention(q_out.ptr, out.ptr, d_slot.ptr, d_len.ptr, None, w.ptr, w.ptr, slots, q_heads, ld, most, 1 / np.sqrt(dim))
    evict = N.PagedEvict(None, d_slot.ptr, d_len.ptr, w.ptr, w.ptr, ep.ptr, ep.ptr, None, d_new.ptr, slots, keep, 4, 24, ld, most)
    desc, L = c.desc(), nat.lib
    K = np.zeros((slots, kv_heads, most, dim))
    V, W, EP = np.zeros_like(K), np.zeros((slots, kv_heads, most)), np.zeros((slots, kv_heads, most), np.int64)
    n = 0
    for t in range(200):
        x = rng.standard_normal((slots, width)).astype(np.float32)
        packed.upload(x)
        d_entry.upload(np.full(slots, n, np.uint32))
        d_pos.upload(np.full(slots, t, np.uint32))
        d_len.upload(np.full(slots, n + 1, np.uint32))
        assert L.m40llm_paged_append_async(nat.ctx, C.byref(desc), C.byref(append)) == 0
        assert L.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(attention)) == 0
        z = x.reshape(slots, -1, dim)
        zq, zk = (P.turned(z[:, a:b], np.full(slots, t), turns, 1) for a, b in ((0, q_heads), (q_heads, q_heads + kv_heads)))
        # the cache holds f16: what rounds differently there differs by one step, so the float64 run takes the device's own rows
        nat.sync(1)
        gk, gv = c.download()
        for s in range(slots):
            at = (c.table[s, n // page], slice(None), n % page)
            assert (np.abs(gk[at] - zk[s]) <= 2 * U16 * np.abs(zk[s]) + 1e-6).all()
            K[s, :, n], V[s, :, n] = gk[at], gv[at]
        EP[:, :, n], W[:, :, n] = t, 0
        n += 1
        got = out.download(np.float32, (slots, q_heads, dim))
        for s in range(slots):
            for h in range(kv_heads):
                for g in range(4):
                    q = zq[s, 4 * h + g]
                    sc = K[s, h, :n] @ q / np.sqrt(dim)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    W[s, h, :n] += p
                    err = P.out_error(q, K[s, h, :n], V[s, h, :n], p, 1 / np.sqrt(dim), p @ V[s, h, :n])
                    # q itself comes from the rotation: 8 u of a pair's size, which moves a score by as much of sum |k|
                    moved = 2 * 16 * U32 * np.abs(q).max() * np.abs(K[s, h, :n]).sum(-1).max() / np.sqrt(dim)
                    assert (np.abs(got[s, 4 * h + g] - p @ V[s, h, :n]) <= err + moved * (p @ np.abs(V[s, h, :n]))).all(), t
        gw = w.download(np.float32, (slots, kv_heads, ld))[:, :, :n]
        assert np.abs(gw - W[:, :, :n]).max() <= 1e-4 * max(1.0, W.max())
        if n == most:
            # the order is the device's weights': they may differ from the float64 run's in the last digits
            assert L.m40llm_paged_evict_async(nat.ctx, C.byref(desc), C.byref(evict)) == 0
            for s in range(slots):
                for h in range(kv_heads):
                    org = P.evict(gw[s, h], EP[s, h].astype(np.uint32), 4, 24, keep, n)
                    for a in (K, V, W, EP):
                        a[s, h, :keep] = a[s, h, org]
            n = keep
            nat.sync(1)
            assert (d_new.download(np.uint32, slots) == keep).all()
            assert np.array_equal(ep.download(np.uint32, (slots, kv_heads, ld))[:, :, :keep], EP[:, :, :keep])
    assert T.status(nat) == 0
