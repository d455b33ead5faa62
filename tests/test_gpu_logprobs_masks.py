"""Log probabilities under masks that leave runs of neighbouring tokens: few of a block's warps then hold all that is left."""
import numpy as np
import pytest

import paged_cases as T
from test_gpu_logprobs import check, run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


@pytest.mark.parametrize("left,where", [(1000, 4000), (600, 0), (2000, 30001), (513, 777), (512, 777), (64, 9001), (20, 5), (1000, -1000)])
@pytest.mark.parametrize("n,rows,top", [(32000, 2, 20), (131077, 2, 20), (32000, 150, 64), (50257, 2, 1)])
def test_runs_of_neighbours(nat, left, where, n, rows, top):
    rng = np.random.default_rng(left + n)
    x = np.full((2, n), -np.inf, np.float32)
    at = where % n
    kept = slice(at, min(n, at + left))
    x[:, kept] = 3 * rng.standard_normal(x[:, kept].shape)
    tokens = np.array([at, 1])
    x, tokens = np.tile(x, (rows // 2, 1)), np.tile(tokens, rows // 2)
    got = run(nat, x, tokens, top)
    check(x[:2], tokens[:2], top, {k: v[:2] for k, v in got.items()})
    check(x[-2:], tokens[-2:], top, {k: v[-2:] for k, v in got.items()})
    assert T.status(nat) == 0
