"""How much the paged attention loses in all: its outputs and the weights that it adds up, as vectors, against the float64 statement. test_paged_precision.py shows that the
bound tells f16 from two f16 parts."""
import numpy as np
import pytest

import paged_cases as T
from paged_cases import P

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


@pytest.mark.parametrize("kind,dim,heads", [("f16", 64, 8), ("f16", 128, 8), ("f16", 64, 24), ("f16", 128, 32), ("f32", 64, 8), ("f32", 128, 16), ("f16", 96, 8),
                                            ("f16", 33, 4)])
@pytest.mark.parametrize("n,queries,keys", [(200, 2.0, 1.0), (777, 2.0, 1.0), (3001, 2.0, 1.0), (600, 2e-5, 1024.0)])
@pytest.mark.parametrize("max_len", [0, 3001])
def test_outputs_and_weights(nat, kind, dim, heads, n, queries, keys, max_len):
    rng = np.random.default_rng(dim + n)
    c = T.Cache(nat, rng, 2, 3001, 2, dim, 16, kind)
    c.k = (c.k.astype(np.float32) * np.float32(keys)).astype(c.dtype)
    c.upload()
    q = (queries * rng.standard_normal((2, heads, dim))).astype(np.float32)
    length, scale = [n, n - 71], float(np.float32(1 / np.sqrt(dim)))
    got, gw = T.attend(nat, c, q, [1, 0], length, weights=np.zeros((2, 2, c.capacity), np.float32), ld=c.capacity, max_len=max_len or n)
    for r, s in enumerate((1, 0)):
        m = length[r]
        for h in range(2):
            K, V = (np.stack(P.rows_of(pool, c.table, s, h, range(m))) for pool in (c.k, c.v))
            weights, allowed = np.zeros(m), 0.0
            for g in range(h * heads // 2, (h + 1) * heads // 2):
                scores = K @ q[r, g].astype(np.float64) * scale
                p = np.exp(scores - scores.max())
                p /= p.sum()
                bound = P.typical_error(q[r, g], K, scale)
                assert np.linalg.norm(got[r, g] - p @ V) <= bound * np.linalg.norm(p @ V), (r, g)
                weights += p
                allowed += bound * np.linalg.norm(p) + heads * P.U32 * np.linalg.norm(weights)  # of the head, and of its addition
            assert np.linalg.norm(gw[s, h, :m] - weights) <= allowed, (r, h)
