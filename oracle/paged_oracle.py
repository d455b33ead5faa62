"""Plain float64 statements of the paged cache's operators and of the log probabilities, one function per mechanism.
Test infrastructure: the product library has no CPU path."""
from __future__ import annotations

import numpy as np

NONE = 0xFFFFFFFF


def turned(x, pos, turns, layout):
    """Heads x [rows, heads, dim]: pair m turns by pos * turns[m] full turns; (m, m + pairs) for layout 1, (2 m, 2 m + 1) for 0."""
    x = np.array(x, np.float64)
    m = len(turns)
    if m == 0:
        return x
    first = np.arange(m) if layout == 1 else 2 * np.arange(m)
    second = first + (m if layout == 1 else 1)
    t = np.asarray(pos, np.float64)[:, None] * np.asarray(turns, np.float64)
    a = 2 * np.pi * (t - np.rint(t))
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    u, v = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = u * c - v * s, u * s + v * c
    return x


def rows_of(pool, table, slot, head, entries):
    """Rows [len(entries), dim] of one kv head; entries on pages outside the pool are None."""
    pages, _, page_tokens, _ = pool.shape
    out = []
    for e in entries:
        page = int(table[slot, e // page_tokens])
        out.append(pool[page, head, e % page_tokens].astype(np.float64) if page < pages else None)
    return out


def attend(q, k_pool, v_pool, table, slot, begin, end, scale):
    """One row: q [q_heads, dim] -> (out [q_heads, dim], weights [kv_heads, end], a bound of the f32 error of out)."""
    kv_heads, dim = k_pool.shape[1], k_pool.shape[3]
    group = q.shape[0] // kv_heads
    out, w = np.zeros(q.shape), np.zeros((kv_heads, max(end, 0)))
    err = np.zeros(q.shape)
    entries = range(begin, end)
    for h in range(kv_heads):
        pairs = [(e, k, v) for e, k, v in zip(entries, rows_of(k_pool, table, slot, h, entries), rows_of(v_pool, table, slot, h, entries))
                 if k is not None]
        if not pairs:
            continue
        at = np.array([p[0] for p in pairs])
        K, V = np.stack([p[1] for p in pairs]), np.stack([p[2] for p in pairs])
        for g in range(h * group, (h + 1) * group):
            x = q[g].astype(np.float64)
            s = K @ x * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[g] = p @ V
            w[h, at] += p
            err[g] = out_error(x, K, V, p, scale, out[g])
    return out, w, err


U32 = 2.0 ** -24


def out_error(x, K, V, p, scale, out):
    """How far an output may be off in 32 bits. A score: x * scale * log2(e) rounds three times, is cut into two f16 parts that leave 2^-22
    of it, and its products are summed over the head (dim roundings, doubled for sums of the tensor cores that are cut off instead of rounded),
    together (2 dim + 8 + 4) u of sum |x| |k| scale. exp2: two ulp, and u of its argument. A weight thus errs by that much of itself, twice
    (numerator and sum); the sums run over at most 1024 entries of a chunk and 256 chunks, again doubled."""
    dim = len(x)
    score = (2 * dim + 12) * U32 * (np.abs(K) @ np.abs(x)).max() * abs(scale)
    weight = 2 * (score + 4 * U32) + 2 * (min(len(p), 1024) + 256) * U32
    return weight * (p @ np.abs(V)) + 2 * U32 * np.abs(out)


def evict_order(weights, pos, first, recent, n):
    """Entries 0 .. n - 1, best first: held ones by entry, then the others by weight (NaN last), the lower entry first."""
    newest = pos[:n].astype(np.int64).max()
    held = (pos[:n].astype(np.int64) < first) | (newest - pos[:n].astype(np.int64) < recent)
    w = np.array(weights[:n], np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    # NaN after -inf
    return np.lexsort((np.arange(n), np.isnan(weights[:n]) & ~held, np.where(held, 0.0, -w), ~held))


def evict(weights, pos, first, recent, keep, n):
    """Origins [min(n, keep)] of the entries of one kv head after an eviction."""
    left = min(n, keep)
    if n <= keep:
        return np.arange(n)
    chosen = set(evict_order(weights, pos, first, recent, n)[:left].tolist())
    late = iter(sorted(e for e in chosen if e >= left))
    return np.array([e if e in chosen else next(late) for e in range(left)])


def logprobs(x, token, top):
    """One row -> (logprob, rank, entropy, lse, top ids, top log probabilities)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    n, most = len(x), x.max()
    if most == -np.inf:
        lp = np.full(n, -np.inf)
        lse, entropy = -np.inf, 0.0
    else:
        with np.errstate(invalid="ignore"):
            d = np.where(x == most, 0.0, x - most)
        rest = np.log(np.exp(d).sum())
        lp, lse = d - rest, most + rest
        p = np.exp(lp)
        entropy = -(p[p > 0] * lp[p > 0]).sum()
    order = np.lexsort((np.arange(n), -x))
    listed = [i for i in order[:top] if x[i] > -np.inf]
    ids = np.array(listed + [NONE] * (top - len(listed)), np.uint32)
    tops = np.array([lp[i] for i in listed] + [-np.inf] * (top - len(listed)))
    if token is None or token >= n:
        return -np.inf, 0, entropy, lse, ids, tops
    rank = 1 + int(((x > x[token]) | ((x == x[token]) & (np.arange(n) < token))).sum())
    return lp[token], rank, entropy, lse, ids, tops


def typical_error(x, K, scale):
    """What the kernels' 32-bit arithmetic may leave of a head's outputs and weights as a vector, relative to its norm (out_error is for single values, where every rounding
    points the same way). A score: 8 u of it from x * scale * log2(e), the cut into two f16 parts (2^-22), the factor out of base 2 and the argument of exp2; per
    step of 16 dimensions the sum so far is cut off at 2 u of it, at its largest here. exp2: 6 u of a weight. Sums: 2 u per 64 entries, 64 u for warps, CTAs and their
    join. Twice, for outputs (or weights) and the sum that they are divided by."""
    dim, n = len(x), len(K)
    steps = np.add.reduceat(K.astype(np.float64) * np.asarray(x, np.float64) * scale, np.arange(0, dim, 16), axis=1)
    most = np.abs(np.cumsum(steps, axis=1)).max()
    return 2 * ((2 * -(-dim // 16) + 8) * most + 6 + 2 * n / 64 + 64) * U32
