"""Paged cache: groups of more q heads than the weights' kernel of the joins takes, and evictions under a bound far above the lengths."""
import numpy as np
import pytest

import paged_cases as T
from test_gpu_paged import check_evict, heavy_tailed, run_evict

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


@pytest.mark.parametrize("kind,dim,heads,kv_heads", [("f16", 64, 130, 2), ("f16", 128, 65, 1), ("f32", 64, 65, 1), ("f16", 96, 66, 1), ("f16", 33, 70, 1), ("f16", 64, 64, 1)])
@pytest.mark.parametrize("entries", [240, 5000])
@pytest.mark.parametrize("in_place", [False, True])
def test_weights_of_wide_groups(nat, kind, dim, heads, kv_heads, entries, in_place):
    """64 q heads of a kv head and more: several rows of a slot, a window, an empty row, slots without rows."""
    rng = np.random.default_rng(dim + heads)
    c = T.Cache(nat, rng, 4, entries, kv_heads, dim, 16, kind)
    w = rng.random((4, kv_heads, c.capacity)).astype(np.float32)
    slot, length, begin = [3, 1, 3, 0, 3], [240, 130, 201, 0, 100], [0, 10, 0, 0, 64]
    q = (2 * rng.standard_normal((5, heads, dim))).astype(np.float32)
    got, gw = T.attend(nat, c, q, slot, length, begin=begin, weights=w, ld=c.capacity, in_place=in_place)
    T.check_attention(c, q, slot, length, got, begin=begin, weights=w, got_w=gw, before=w if in_place else np.full(w.shape, -5.0, np.float32))
    assert not got[3].any() and T.status(nat) == 0


@pytest.mark.parametrize("capacity,max_len", [(32768, 0), (32768, 30000), (16384, 0), (32768, 1100)])
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_evictions_under_a_loose_bound(nat, capacity, max_len, positions, in_place):
    """128 short lists of slots that could hold far more: one CTA a list, whose keys the bound alone would not let into shared memory."""
    rng = np.random.default_rng(capacity)
    c = T.Cache(nat, rng, 16, capacity, 8, 8, 64, spare=0)
    w = heavy_tailed(rng, (16, 8, c.capacity))
    pos = np.argsort(rng.random(w.shape), -1).astype(np.uint32) if positions else None
    seq, length = rng.permutation(16), rng.integers(1025, 1101, 16)
    length[:4] = 1100, 1024, 0, 7
    got = run_evict(nat, c, seq, length, 1024, 4, 64, w, pos, None, in_place, max_len)
    check_evict(c, seq, length, 1024, 4, 64, w, pos, got, None, in_place, (c.k, c.v))
    assert T.status(nat) == 0
