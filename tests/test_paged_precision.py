"""Whether the tests of the paged attention's precision would notice a lost half: the kernel's arithmetic in numpy, whole and with one step of it left out, against the
float64 statement and the bound that test_gpu_paged_precision.py holds the kernel to. Runs without a GPU."""
import numpy as np
import pytest

from oracle import paged_oracle as P

F16, F32 = np.float16, np.float32
# head size, entries, size of the queries, size of the keys
CASES = [(dim, n, 2.0, 1.0) for dim in (64, 128) for n in (200, 777, 3001)] + [(64, 600, 2e-5, 1024.0), (128, 600, 2e-5, 1024.0)]


def halves(x, keep_low):
    hi = x.astype(F16).astype(F32)
    return hi + (x - hi).astype(F16).astype(F32) if keep_low else hi


def head(q, K, V, leave_out=""):
    """One head as paged_tiles_kernel computes it: (output, weights)."""
    scale = F32(1 / np.sqrt(len(q)))
    y = q * F32(scale * F32(np.log2(np.e)))
    up = F32(2.0 ** (9 - np.floor(np.log2(np.abs(y).max())))) if leave_out != "power of two" else F32(1)
    s = (halves(y * up, leave_out != "queries") @ K.astype(F32).T) / up
    p = np.exp2(s - (s.max() - F32(15)))
    total = p.sum(dtype=F32)
    out = (halves(p, leave_out != "weights") @ V.astype(F32)) / total
    kept = p / total
    return out, kept.astype(F16).astype(F32) if leave_out == "weights" else kept


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def drawn(dim, n, queries, keys, seed):
    rng = np.random.default_rng(seed)
    K, V = ((x * rng.standard_normal((n, dim))).astype(F16) for x in (keys, 1.0))
    return (queries * rng.standard_normal(dim)).astype(F32), K, V


def stated(q, K, V):
    scale = float(F32(1 / np.sqrt(len(q))))
    s = K.astype(np.float64) @ q.astype(np.float64) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ V.astype(np.float64), p, P.typical_error(q, K, scale)


@pytest.mark.parametrize("case", CASES)
def test_the_whole_arithmetic_is_within_the_bound(case):
    for seed in range(20):
        q, K, V = drawn(*case, seed)
        out, p, bound = stated(q, K, V)
        got, w = head(q, K, V)
        assert off(got, out) <= bound and off(w, p) <= bound, seed


# queries of 2 keep their bits without a power of two; scores of 0.02 lose nothing by the queries' lower half
@pytest.mark.parametrize("case,leave_out", [(c, x) for c in CASES for x in ("weights", "queries" if c[2] >= 1 else "power of two")])
def test_a_lost_half_is_beyond_it(case, leave_out):
    """Most heads of every size show it, and a tested row has eight of them."""
    out_beyond = weights_beyond = 0
    for seed in range(20):
        q, K, V = drawn(*case, seed)
        out, p, bound = stated(q, K, V)
        got, w = head(q, K, V, leave_out)
        out_beyond += off(got, out) > bound
        weights_beyond += off(w, p) > bound
    assert out_beyond >= 10 and weights_beyond >= 10, (out_beyond, weights_beyond)
