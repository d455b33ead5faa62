"""m40llm_logprobs_f32_async against the float64 statement of oracle/paged_oracle.py."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as T
from paged_cases import N, P

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def clean(nat):
    yield
    nat.free_all()
    T.status(nat)


def run(nat, x, tokens, top, ld=0, drop=()):
    rows, n = x.shape
    host = x if not ld else np.concatenate([x, np.full((rows, ld - n), 1e9, np.float32)], 1)
    bufs = {name: T.f32(nat, np.full(rows, 123.0)) for name in ("logprob", "entropy", "lse")}
    bufs |= {"rank": T.u32(nat, np.full(rows, 99)), "top_ids": T.u32(nat, np.full((rows, max(1, top)), 99)),
             "top_logprobs": T.f32(nat, np.full((rows, max(1, top)), 123.0))}
    call = N.Logprobs(logits=T.f32(nat, host).ptr, tokens=None if tokens is None else T.u32(nat, tokens).ptr, rows=rows, n=n, ld=ld, top=top,
                      **{k: b.ptr for k, b in bufs.items() if k not in drop})
    assert nat.lib.m40llm_logprobs_f32_async(nat.ctx, C.byref(call)) == 0
    nat.sync(1)
    return {k: b.download(np.uint32 if k in ("rank", "top_ids") else np.float32, (rows, top) if k.startswith("top") else rows)
            for k, b in bufs.items() if not (k.startswith("top") and top == 0)}


def bounds(x, lp, entropy, lse):
    """How far values may be off in 32 bits: exp of an argument d errs by (|d| + 4) u of itself; a sum of n of them in any order by at most n u, taken here as the depth
    of sums in threads and trees (n / 64 + 64) u; the log adds an ulp, and the subtractions u of their operands."""
    n = len(x)
    f = x[np.isfinite(x)]
    span = f.max() - f.min() if len(f) else 0.0
    total = (min(span, 110) + 4 + n / 64 + 64) * U32
    size = np.abs(f).max() if len(f) else 0.0
    return total + 4 * U32 * (size + 20), 2 * total * (20 + np.log(n)) + 8 * U32 * (size + 20)


def check(x, tokens, top, got):
    for r in range(len(x)):
        lp, rank, entropy, lse, ids, tops = P.logprobs(x[r], None if tokens is None else int(tokens[r]), top)
        b, be = bounds(x[r].astype(np.float64), lp, entropy, lse)
        for name, want in (("logprob", lp), ("lse", lse), ("top_logprobs", tops)):
            if name not in got or (tokens is None and name == "logprob"):
                continue
            g, want = np.atleast_1d(got[name][r]).astype(np.float64), np.atleast_1d(want)
            want = np.where(want < -np.finfo(np.float32).max, -np.inf, want)  # a difference of two f32 values may lie beyond f32: -inf is its rounding
            fine = np.isfinite(want)
            assert np.array_equal(g[~fine], want[~fine]) and (np.abs(g[fine] - want[fine]) <= b + 2 * U32 * np.abs(want[fine])).all(), (name, r, g, want)
        assert abs(got["entropy"][r] - entropy) <= be, (r, got["entropy"][r], entropy)
        if tokens is not None:
            assert got["rank"][r] == rank, r
        if top:
            assert np.array_equal(got["top_ids"][r], ids), r


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 1000, 1023, 1025, 4096, 32000, 50257, 131077, 300001])
@pytest.mark.parametrize("rows,top", [(1, 20), (3, 1), (2, 64)])
def test_sizes(nat, n, rows, top):
    rng = np.random.default_rng(n + rows)
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    tokens = rng.integers(0, n, rows)
    tokens[0] = x[0].argmax()
    got = run(nat, x, tokens, top)
    check(x, tokens, top, got)
    assert got["rank"][0] == 1 and T.status(nat) == 0


@pytest.mark.parametrize("rows,n,ld", [(7, 2003, 0), (64, 2003, 0), (149, 2003, 0), (400, 2003, 0), (445, 2003, 0), (1000, 2003, 0), (900, 1, 0), (700, 6, 0),
                                       (500, 4095, 4101), (500, 4096, 0), (460, 9001, 0), (889, 1000, 1001)])
def test_many_rows(nat, rows, n, ld):
    rng = np.random.default_rng(rows)
    x = (4 * rng.standard_normal((rows, n))).astype(np.float32)
    tokens = rng.integers(0, n, rows)
    check(x, tokens, 7, run(nat, x, tokens, 7, ld=ld))
    assert T.status(nat) == 0


@pytest.mark.parametrize("ld", [0, 5003, 5004, 5120])
def test_pitch(nat, ld):
    rng = np.random.default_rng(ld)
    x = rng.standard_normal((5, 5003)).astype(np.float32)
    tokens = rng.integers(0, 5003, 5)
    check(x, tokens, 9, run(nat, x, tokens, 9, ld=ld))


@pytest.mark.parametrize("name", ["equal", "few values", "ascending", "descending", "one large", "close", "masked", "nan", "infinite", "all masked", "all nan",
                                  "few left", "one thread's", "far apart", "huge"])
@pytest.mark.parametrize("n,times", [(600, 1), (33000, 1), (9001, 150)])
def test_rows_of_every_kind(nat, name, n, times):
    rng = np.random.default_rng(len(name))
    x = (3 * rng.standard_normal((3, n))).astype(np.float32)
    if name == "equal":
        x[:] = -1.5
    elif name == "few values":
        x = np.floor(x)
    elif name == "ascending":
        x.sort(-1)
    elif name == "descending":
        x = -np.sort(-x, -1)
    elif name == "one large":
        x[:, n // 2] = 200
    elif name == "close":
        x = (np.float32(1.0).view(np.uint32) + rng.integers(0, 50, x.shape).astype(np.uint32)).view(np.float32)
    elif name == "masked":
        x[rng.random(x.shape) < 0.95] = -np.inf
    elif name == "nan":
        x[rng.random(x.shape) < 0.3] = np.nan
    elif name == "infinite":
        x[0, 5], x[1, [3, n - 1]] = np.inf, np.inf
        x[2, 7] = -np.inf
    elif name == "all masked":
        x[:2] = -np.inf
    elif name == "all nan":
        x[1] = np.nan
    elif name == "few left":
        keep = x[:, [17, 400, 599]].copy()
        x[:] = -np.inf
        x[:, [17, 400, 599]] = keep
    elif name == "one thread's":
        for step in (256, 512, 1024):  # the largest values where one thread of a block would meet them all
            x[:, 3::step] += 50
    elif name == "far apart":
        x *= 1e4
    elif name == "huge":
        x = (np.finfo(np.float32).max * rng.uniform(-1, 1, x.shape)).astype(np.float32)
    tokens = np.array([5, n - 1, 7])
    if times == 1:
        check(x, tokens, 20, run(nat, x, tokens, 20))
        return
    got = run(nat, np.tile(x, (times, 1)), np.tile(tokens, times), 20)  # a long batch of the three rows
    for at in range(0, 12, 3):
        check(x, tokens, 20, {k: v[at:at + 3] for k, v in got.items()})
    for k, v in got.items():  # a row's place within 16 bytes decides which thread adds which value: it comes back after 12 rows, and with it every bit
        assert all(np.array_equal(v[i - 12], v[i]) for i in range(12, 3 * times)), k


def test_outputs_may_be_left_out(nat):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 999)).astype(np.float32)
    tokens = rng.integers(0, 999, 4)
    whole = run(nat, x, tokens, 6)
    for drop in (("logprob",), ("rank", "entropy"), ("lse", "top_ids"), ("top_logprobs",), ("top_ids", "top_logprobs")):
        got = run(nat, x, tokens, 6, drop=drop)
        for k in whole:
            if k in drop:
                assert (got[k] == (99 if whole[k].dtype == np.uint32 else 123.0)).all()
            else:
                assert np.array_equal(got[k], whole[k])
    got = run(nat, x, None, 6, drop=("logprob", "rank"))
    assert np.array_equal(got["top_ids"], whole["top_ids"]) and np.array_equal(got["entropy"], whole["entropy"])
    got = run(nat, x, tokens, 0)
    assert np.array_equal(got["logprob"], whole["logprob"]) and T.status(nat) == 0


def test_tokens_outside(nat):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 100)).astype(np.float32)
    got = run(nat, x, [100, 99, 0xffffffff], 2)
    check(x, np.array([100, 99, 0xffffffff]), 2, got)
    assert got["rank"][0] == 0 and got["logprob"][0] == -np.inf and T.status(nat) == 8


def test_with_the_greedy_choice_in_a_graph(nat):
    """The greedy token's own log probability, captured: the two entry points agree on which value comes first."""
    rng = np.random.default_rng(3)
    rows, n = 5, 7001
    d_x, d_tok = T.f32(nat, np.zeros((rows, n))), T.u32(nat, np.zeros(rows))
    out = {k: nat.buf(4 * rows) for k in ("logprob", "rank", "top_ids", "top_logprobs")}
    call = N.Logprobs(logits=d_x.ptr, tokens=d_tok.ptr, rows=rows, n=n, top=1, **{k: b.ptr for k, b in out.items()})
    L, graph = nat.lib, C.c_void_p()

    def both():
        assert L.m40llm_argmax_f32_async(nat.ctx, d_x.ptr, rows, n, d_tok.ptr) == 0
        assert L.m40llm_logprobs_f32_async(nat.ctx, C.byref(call)) == 0
    both()
    nat.sync(1)
    assert L.m40llm_cuda_graph_begin_capture(nat.ctx, 1) == 0
    both()
    assert L.m40llm_cuda_graph_end_capture(nat.ctx, 1, C.byref(graph)) == 0
    for _ in range(3):
        d_x.upload(np.floor(4 * rng.standard_normal((rows, n))).astype(np.float32))
        assert L.m40llm_cuda_graph_launch(nat.ctx, graph, 1) == 0
        nat.sync(1)
        got = {k: b.download(np.uint32 if k in ("rank", "top_ids") else np.float32, rows) for k, b in out.items()}
        assert (got["rank"] == 1).all() and np.array_equal(got["top_ids"], d_tok.download(np.uint32, rows))
        assert np.array_equal(got["logprob"], got["top_logprobs"])
    L.m40llm_cuda_graph_destroy(graph)
