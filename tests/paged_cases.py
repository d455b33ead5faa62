"""A paged cache with its contents on the host and on the device, and the calls over it, for the tests."""
import ctypes as C

import numpy as np

from helpers import load_package

load_package()
from m40_llm_b200 import native as N  # noqa: E402
from oracle import paged_oracle as P  # noqa: E402

KIND = {"f16": (np.float16, N.DT_F16), "f32": (np.float32, N.DT_F32)}


class Cache:
    """Pools with random contents; every slot has `entries` places, pages in any order, `spare` pages that belong to nobody."""

    def __init__(self, nat, rng, slots, entries, kv_heads, dim, page, kind="f16", spare=2, offset=0):
        self.nat, self.page, self.kind = nat, page, kind
        dtype, code = KIND[kind]
        per = -(-entries // page)
        self.pages = slots * per + spare
        shape = (self.pages, kv_heads, page, dim)
        self.k, self.v = (rng.standard_normal(shape).astype(dtype) for _ in range(2))
        self.table = rng.permutation(self.pages)[: slots * per].reshape(slots, per).astype(np.uint32)
        self.slots, self.kv_heads, self.dim, self.capacity, self.code, self.dtype = slots, kv_heads, dim, per * page, code, dtype
        self.offset = offset  # elements before the pools: other alignments
        self.upload()

    def upload(self):
        pad = np.zeros(self.offset, self.dtype)
        self.dk, self.dv = (self.nat.buf(np.concatenate([pad, a.ravel()])) for a in (self.k, self.v))
        self.dt = self.nat.buf(self.table)

    def desc(self):
        at = self.offset * self.k.itemsize
        return N.PagedCache(self.dk.ptr + at, self.dv.ptr + at, self.dt.ptr, self.pages, self.page, self.slots, self.table.shape[1],
                            self.kv_heads, self.dim, self.code)

    def download(self):
        n = self.k.size + self.offset
        return tuple(b.download(self.dtype, n)[self.offset:].reshape(self.k.shape) for b in (self.dk, self.dv))


def u32(nat, values):
    return nat.buf(np.ascontiguousarray(values, np.uint32))


def f32(nat, values):
    return nat.buf(np.ascontiguousarray(values, np.float32))


def status(nat):
    st = np.zeros(1, np.uint32)
    assert nat.lib.m40llm_context_take_device_status(nat.ctx, st.ctypes.data) == 0
    return int(st[0])


def attention_call(nat, cache, q, slot, length, begin=None, weights=None, ld=0, max_len=0, scale=None, in_place=False):
    """(descriptor, call, output buffers): weights None (none wanted), or a host array [slots, kv_heads, ld]."""
    rows, heads = q.shape[:2]
    out = f32(nat, np.full(q.shape, 7.0))
    w_in = w_out = None
    if weights is not None:
        w_in = f32(nat, weights)
        w_out = w_in if in_place else f32(nat, np.full(weights.shape, -5.0))
    call = N.PagedAttention(f32(nat, q).ptr, out.ptr, u32(nat, slot).ptr, u32(nat, length).ptr, None if begin is None else u32(nat, begin).ptr,
                            None if w_in is None else w_in.ptr, None if w_out is None else w_out.ptr, rows, heads, ld, max_len,
                            scale if scale is not None else 1.0 / np.sqrt(cache.dim))
    return cache.desc(), call, out, w_out


def attend(nat, cache, q, slot, length, **more):
    desc, call, out, w_out = attention_call(nat, cache, q, slot, length, **more)
    assert nat.lib.m40llm_attention_paged_async(nat.ctx, C.byref(desc), C.byref(call)) == 0
    nat.sync(1)
    weights = more.get("weights")
    return out.download(np.float32, q.shape), None if w_out is None else w_out.download(np.float32, weights.shape)


def check_attention(cache, q, slot, length, got, begin=None, weights=None, got_w=None, scale=None, before=None):
    """Outputs (and weights) against the plain statement, within the bound that the oracle derives from the values."""
    scale = float(np.float32(scale if scale is not None else 1.0 / np.sqrt(cache.dim)))
    sums, most = {}, {}
    for r in range(len(q)):
        b = 0 if begin is None else int(begin[r])
        out, w, err = P.attend(q[r], cache.k, cache.v, cache.table, int(slot[r]), b, int(length[r]), scale)
        off = np.abs(got[r] - out)
        assert np.isfinite(got[r]).all() and (off <= err + 1e-30).all(), (r, (off / np.maximum(err, 1e-30)).max())
        s = int(slot[r])
        sums.setdefault(s, np.zeros((cache.kv_heads, cache.capacity)))[:, : w.shape[1]] += w
        most[s] = max(most.get(s, 0), int(length[r]))
    if weights is None:
        return
    group = q.shape[1] // cache.kv_heads
    for s in range(cache.slots):
        n = most.get(s, 0)
        want = weights[s, :, :n].astype(np.float64) + sums[s][:, :n] if n else weights[s, :, :0]
        # a weight errs like an output whose values are 1 (see out_error); the scores of these tests stay below 60
        rel = 2 * (2 * cache.dim + 12) * P.U32 * 60 + 2 * (1024 + 256) * P.U32
        rows = sum(int(t) == s for t in slot)
        bound = rel * (sums[s][:, :n] if n else 0) + (rows * group + 2) * P.U32 * np.abs(want)
        assert (np.abs(got_w[s, :, :n] - want) <= bound + 1e-30).all(), s
        rest = before[s, :, n:]
        assert np.array_equal(got_w[s, :, n:], rest), "entries beyond the rows' lengths changed"
