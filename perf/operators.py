"""Serving operators around a key / value cache in pages, and the scores of what a model answers with:

    append   new keys and values into the cache's pages, keys (and queries) rotated by their positions
    attend   attention of single tokens over the pages, optionally adding up every entry's attention weight
    evict    the entries with the largest accumulated weight stay, the others give up their place
    score    log probabilities of given tokens, their ranks, the entropy, the most likely alternatives

`run` computes them in plain torch operations, or, where `own` is set, by the C entry points a user calls. All data is made on
the GPU from the seed.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DEV = "cuda"
_TYPES = {"f16": torch.float16, "f32": torch.float32}
VOCAB = 32000
# q heads, kv heads, head size
HEADS = ((32, 8, 128), (32, 4, 64), (16, 2, 128), (8, 2, 64))


def listed():
    return [
        # one decode step of a batch of chats: each sequence's new token
        {"name": "append-32", "op": "append", "rows": 32, "slots": 32, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "start": 5003,
         "pairs": 64, "split": False, "type": "f16"},
        # a portion of two prompts at far positions, rotation of a part of the head, small pages
        {"name": "append-prompt", "op": "append", "rows": 2001, "slots": 2, "q_heads": 16, "kv_heads": 2, "dim": 128, "page": 16, "start": 30011,
         "pairs": 32, "split": True, "type": "f16"},
        # one chat on a small model: latency
        {"name": "attend-1", "op": "attend", "rows": 1, "low": 700, "high": 700, "q_heads": 32, "kv_heads": 4, "dim": 64, "page": 16,
         "weights": False, "type": "f16"},
        # one very long document
        {"name": "attend-long", "op": "attend", "rows": 1, "low": 130001, "high": 130001, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "weights": False, "type": "f16"},
        # a server's batch, contexts from nearly nothing to long
        {"name": "attend-32", "op": "attend", "rows": 32, "low": 128, "high": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "weights": False, "type": "f16"},
        # a batch in the 32-bit mode of the layer stacks, one slot still empty
        {"name": "attend-f32", "op": "attend", "rows": 9, "low": 0, "high": 4097, "q_heads": 16, "kv_heads": 2, "dim": 128, "page": 32,
         "weights": False, "type": "f32"},
        # a batch whose caches are kept short by their weights
        {"name": "attend-weights", "op": "attend", "rows": 12, "low": 509, "high": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "weights": True, "type": "f16"},
        # four prompts have come in: what stays of each
        {"name": "evict-prompts", "op": "evict", "slots": 4, "low": 900, "high": 8192, "kv_heads": 8, "dim": 128, "page": 64, "keep": 1024,
         "first": 4, "recent": 128, "again": False, "type": "f16"},
        # a long answer outgrew its share once more
        {"name": "evict-long", "op": "evict", "slots": 1, "low": 32768, "high": 32768, "kv_heads": 8, "dim": 128, "page": 32, "keep": 4099,
         "first": 16, "recent": 1000, "again": True, "type": "f16"},
        # one new token with its alternatives
        {"name": "score-1", "op": "score", "rows": 1, "n": VOCAB, "top": 20, "masked": False},
        # a batch's new tokens over a large vocabulary under a grammar's mask
        {"name": "score-32", "op": "score", "rows": 32, "n": 131077, "top": 5, "masked": True},
        # a prompt's tokens
        {"name": "score-prompt", "op": "score", "rows": 2048, "n": VOCAB, "top": 1, "masked": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "evict", "score"))
    q_heads, kv_heads, dim = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    kind = rng.choice(("f16", "f16", "f16", "f32"))
    if op == "append":
        slots = _log(rng, 1, 64)
        return {"op": op, "rows": max(slots, _log(rng, 1, 2048)), "slots": slots, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "start": rng.randint(0, 40000), "pairs": rng.choice((0, dim // 4, dim // 2)), "split": rng.random() < 0.5, "type": kind}
    if op == "attend":
        rows = _log(rng, 1, 48)
        high = _log(rng, 1, min(131072, 240000 // rows if kind == "f16" else 100000 // rows))
        return {"op": op, "rows": rows, "low": high // _log(rng, 1, 64) if rng.random() < 0.8 else 0, "high": high, "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "page": page, "weights": rng.random() < 0.3, "type": kind}
    if op == "evict":
        slots = _log(rng, 1, 8)
        high = _log(rng, 100, 40000 // slots)
        keep = max(16, int(high * rng.uniform(0.05, 0.95)))
        return {"op": op, "slots": slots, "low": max(1, high // _log(rng, 1, 8)), "high": high, "kv_heads": kv_heads, "dim": dim, "page": page,
                "keep": keep, "first": rng.randint(0, keep // 4), "recent": rng.randint(0, keep // 2), "again": rng.random() < 0.5, "type": kind}
    n = _log(rng, 1000, 160000)
    return {"op": op, "rows": _log(rng, 1, min(2048, 64000000 // n)), "n": n, "top": rng.choice((0, 1, 5, 20)), "masked": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _lens(case, count):
    """`count` lengths from low to high, evenly spread; their order is the seed's."""
    if count == 1:
        return [case["high"]]
    low, high = case["low"], case["high"]
    return [low + (high - low) * i // (count - 1) for i in range(count)]


def _u32(values):
    return torch.as_tensor(values, dtype=torch.int64, device=_DEV).to(torch.int32)


def _pool(gen, case, slots, entries, filled=True):
    """Keys and values of `slots` sequences with room for `entries` each, their pages in the pool in any order."""
    per = -(-entries // case["page"])
    pages = slots * per + 3
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    make = (lambda: torch.randn(shape, generator=gen, device=_DEV, dtype=_TYPES[case["type"]])) if filled else \
        (lambda: torch.zeros(shape, device=_DEV, dtype=_TYPES[case["type"]]))
    table = torch.randperm(pages, generator=gen, device=_DEV)[: slots * per].reshape(slots, per).to(torch.int32)
    return {"k": make(), "v": make(), "table": table, "slots": slots, "entries": per * case["page"]}


def _rows_of(case):
    """(slot, entry) of every row of an append: the rows go to the slots in turn."""
    r = np.arange(case["rows"])
    return r % case["slots"], case["start"] + r // case["slots"]


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op == "append":
        rows, width = case["rows"], (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        slot, entry = _rows_of(case)
        s["pool"] = _pool(gen, case, case["slots"], int(entry.max()) + 1 - case["start"] // case["page"] * case["page"], filled=False)
        s["packed"] = torch.randn(rows, width, generator=gen, device=_DEV)
        s["slot"], s["pos"] = _u32(slot), _u32(entry)
        s["entry"] = _u32(entry - case["start"] // case["page"] * case["page"])  # earlier pages were given back: only the last ones are held
        m = max(1, case["pairs"])
        s["turns"] = torch.as_tensor(10000.0 ** (-np.arange(m) / m) / (2 * math.pi), dtype=torch.float64, device=_DEV)
        s["q"] = torch.empty(rows, case["q_heads"] * case["dim"], device=_DEV)
    elif op == "attend":
        rows = case["rows"]
        s["pool"] = _pool(gen, case, rows, max(1, case["high"]))
        s["q"] = 2.0 * torch.randn(rows, case["q_heads"], case["dim"], generator=gen, device=_DEV)
        s["slot"] = torch.randperm(rows, generator=gen, device=_DEV).to(torch.int32)
        order = torch.randperm(rows, generator=gen, device=_DEV)
        s["len"] = _u32(_lens(case, rows))[order].contiguous()
        s["out"] = torch.empty(rows, case["q_heads"], case["dim"], device=_DEV)
        if case["weights"]:
            s["weights"] = torch.rand(rows, case["kv_heads"], s["pool"]["entries"], generator=gen, device=_DEV).square_()
            s["weights_out"] = s["weights"].clone()
    elif op == "evict":
        slots, heads, keep = case["slots"], case["kv_heads"], case["keep"]
        s["pool"] = _pool(gen, case, slots, case["high"])
        s["to"] = _pool(gen, case, slots, keep, filled=False)
        order = torch.randperm(slots, generator=gen, device=_DEV)
        s["seq"] = torch.randperm(slots, generator=gen, device=_DEV).to(torch.int32)
        s["len"] = _u32(_lens(case, slots))[order].contiguous()
        shape = (slots, heads, s["pool"]["entries"])
        w = torch.exp(2.0 * torch.randn(shape, generator=gen, device=_DEV))  # a few entries hold most of the weight
        s["weights"] = torch.where(torch.rand(shape, generator=gen, device=_DEV) < 0.05, torch.zeros((), device=_DEV), w)
        place = torch.rand(shape, generator=gen, device=_DEV).argsort(-1) if case["again"] else torch.arange(shape[2], device=_DEV).expand(shape)
        s["pos"] = place.to(torch.int32).contiguous()
        s["weights_out"], s["pos_out"] = torch.zeros_like(s["weights"]), torch.zeros_like(s["pos"])
        s["from"] = torch.zeros(slots, heads, keep, dtype=torch.int32, device=_DEV)
        s["new_len"] = torch.zeros(slots, dtype=torch.int32, device=_DEV)
    else:
        rows, n, top = case["rows"], case["n"], case["top"]
        s["logits"] = 3.0 * torch.randn(rows, n, generator=gen, device=_DEV)
        if case["masked"]:
            s["logits"].masked_fill_(torch.rand(rows, n, generator=gen, device=_DEV) < 0.9, -math.inf)
        s["tokens"] = torch.randint(n, (rows,), generator=gen, device=_DEV).to(torch.int32)
        likely = torch.rand(rows, generator=gen, device=_DEV) < 0.5  # the greedy choice, as often as another token
        s["tokens"] = torch.where(likely, s["logits"].argmax(-1).to(torch.int32), s["tokens"])
        for name in ("logprob", "entropy"):
            s[name] = torch.empty(rows, device=_DEV)
        s["rank"] = torch.empty(rows, dtype=torch.int32, device=_DEV)
        s["top_ids"] = torch.empty(rows, top, dtype=torch.int32, device=_DEV)
        s["top_logprobs"] = torch.empty(rows, top, device=_DEV)
    return s


# -------------------------------------------------------------------------------------------------------------- plain forms
def _turned(x, pos, turns, pairs, split):
    """Heads x [rows, heads, dim] turned by pos * turns[m] full turns, m the pair: (m, m + pairs), or (2 m, 2 m + 1)."""
    if pairs == 0:
        return x
    t = pos.to(torch.float64)[:, None] * turns[:pairs]
    angle = (2 * math.pi) * (t - torch.round(t))
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if split:
        a, b, rest = x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]
        return torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    a, b, rest = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], x[..., 2 * pairs:]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), rest], -1)


def _plain_append(s):
    c, p = s["case"], s["pool"]
    rows, D = c["rows"], c["dim"]
    q, k, v = (x.reshape(rows, -1, D) for x in s["packed"].split([c["q_heads"] * D, c["kv_heads"] * D, c["kv_heads"] * D], -1))
    q, k = (_turned(x, s["pos"], s["turns"], c["pairs"], c["split"]) for x in (q, k))
    page = p["table"][s["slot"].long(), torch.div(s["entry"], c["page"], rounding_mode="floor").long()].long()
    at = (s["entry"] % c["page"]).long()
    p["k"][page, :, at] = k.to(p["k"].dtype)
    p["v"][page, :, at] = v.to(p["v"].dtype)
    return {"q": q.reshape(rows, -1), "k": p["k"], "v": p["v"]}


def _gathered(pool, heads, dim, slot, entries):
    """[rows, kv heads, entries, dim] in 32 bits"""
    x = pool[slot].permute(0, 2, 1, 3, 4).reshape(slot.shape[0], heads, -1, dim)
    return x[:, :, :entries].float()


def _plain_attend(s):
    c, p = s["case"], s["pool"]
    rows, H, D, most = c["rows"], c["kv_heads"], c["dim"], max(1, c["high"])
    pages = p["table"].long()[s["slot"].long()]
    k, v = (_gathered(p[n], H, D, pages, most) for n in ("k", "v"))
    q = s["q"].reshape(rows, H, -1, D)
    scores = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    seen = torch.arange(most, device=_DEV) < s["len"][:, None, None, None]
    scores = torch.where(seen, scores, torch.full((), -math.inf, device=_DEV))
    top = scores.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros((), device=_DEV))
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total > 0, total, torch.ones_like(total))
    out = {"out": torch.matmul(w, v).reshape(rows, c["q_heads"], D)}
    if c["weights"]:
        grown = s["weights"].clone()
        grown[s["slot"].long(), :, :most] += w.sum(2)
        out["weights"] = grown
    return out


def _plain_evict(s):
    c, p, to = s["case"], s["pool"], s["to"]
    keep, n = c["keep"], p["entries"]
    seq = s["seq"].long()
    w, pos = s["weights"][seq], s["pos"][seq].long()
    entry = torch.arange(n, device=_DEV)
    used = (entry < s["len"][:, None, None]).expand_as(w)
    end = torch.where(used, pos, torch.full_like(pos, -1)).amax(-1, keepdim=True) + 1
    held = (pos < c["first"]) | (pos + c["recent"] >= end)
    order = torch.where(held, torch.full_like(w, math.inf), w)
    order = torch.where(used, order, torch.full_like(w, -math.inf)).sort(dim=-1, descending=True, stable=True).indices
    left = torch.minimum(s["len"], torch.full_like(s["len"], keep))
    stays = torch.zeros_like(used).scatter_(-1, order, entry.expand_as(order) < left[:, None, None])
    # place i of the shortened cache keeps its entry if that stays, else it takes the next one that stays from behind the new end
    place = torch.arange(min(keep, n), device=_DEV)
    here = stays[..., : place.numel()]
    behind = stays & (entry >= left[:, None, None])
    rank = torch.where(behind, behind.long().cumsum(-1) - 1, torch.full_like(order, n))
    sources = torch.zeros(*rank.shape[:2], n + 1, dtype=torch.int64, device=_DEV).scatter_(-1, rank, entry.expand_as(rank))
    hole = (~here).long().cumsum(-1) - 1
    origin = torch.where(here, place, sources.gather(-1, hole.clamp(min=0)))
    valid = (place < left[:, None, None]).expand_as(origin)
    moved = torch.full((*origin.shape[:2], keep), -1, dtype=torch.int32, device=_DEV)
    moved[..., : place.numel()] = torch.where(valid, origin, torch.full_like(origin, -1)).to(torch.int32)
    heads = torch.arange(c["kv_heads"], device=_DEV)[None, :, None]
    src = p["table"].long()[seq][:, None].expand(-1, c["kv_heads"], -1).gather(-1, torch.div(origin, c["page"], rounding_mode="floor"))
    dst = to["table"].long()[seq][:, place // c["page"]][:, None].expand_as(src)
    at = (heads.expand_as(src)[valid], (origin % c["page"])[valid])
    into = (dst[valid], at[0], (place % c["page"]).expand_as(src)[valid])
    for name in ("k", "v"):
        to[name][into] = p[name][src[valid], at[0], at[1]]
    rows = seq[:, None, None].expand_as(src)[valid]
    both = (rows, at[0], place.expand_as(src)[valid])
    s["weights_out"][both] = s["weights"][rows, at[0], origin[valid]]
    s["pos_out"][both] = s["pos"][rows, at[0], origin[valid]]
    return {"from": moved, "new_len": left, "k": to["k"], "v": to["v"], "weights": s["weights_out"], "pos": s["pos_out"]}


def _plain_score(s):
    c, x = s["case"], s["logits"]
    token = s["tokens"].long()[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    lse = top + torch.log(e.sum(-1, keepdim=True))
    p = torch.exp(x - lse)
    entropy = torch.where(p > 0, p * (lse - x), torch.zeros((), device=_DEV)).sum(-1)
    own_x = x.gather(-1, token)
    place = torch.arange(c["n"], device=_DEV)
    rank = 1 + ((x > own_x) | ((x == own_x) & (place < token))).sum(-1)
    out = {"logprob": (own_x - lse)[:, 0], "entropy": entropy, "rank": rank.to(torch.int32)}
    if c["top"]:
        values, ids = x.sort(dim=-1, descending=True, stable=True)
        out["top_ids"] = ids[:, : c["top"]].to(torch.int32)
        out["top_logprobs"] = values[:, : c["top"]] - lse
    return out


# ------------------------------------------------------------------------------------------------------- the framework's calls
def _package():
    """The package's folder carries a hyphen, so it is loaded by path."""
    if "m40_llm_b200" not in sys.modules:
        folder = os.path.join(_ROOT, "m40-llm_b200")
        spec = importlib.util.spec_from_file_location("m40_llm_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules["m40_llm_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["m40_llm_b200"]


_native = None


def _nat():
    """One context per program."""
    global _native
    if _native is None:
        pkg = _package()
        _native = pkg.native.Native(pkg.native.lib(), 0)
    return _native


def _cache(N, case, pool):
    return N.PagedCache(k=pool["k"].data_ptr(), v=pool["v"].data_ptr(), table=pool["table"].data_ptr(), pages=pool["k"].shape[0],
                        page_tokens=case["page"], slots=pool["slots"], max_pages=pool["table"].shape[1], kv_heads=case["kv_heads"],
                        head_dim=case["dim"], elem_dtype=N.DT_F16 if case["type"] == "f16" else N.DT_F32)


def _calls(s):
    """The call's description, made once per state as a program that decodes keeps it, and what the call leaves."""
    nat, N, c = _nat(), _package().native, s["case"]
    ptr = lambda name: s[name].data_ptr() if name in s and s[name].numel() else None  # noqa: E731
    if c["op"] == "append":
        D = c["dim"]
        k_at, v_at = 4 * c["q_heads"] * D, 4 * (c["q_heads"] + c["kv_heads"]) * D
        call = N.PagedAppend(q=ptr("packed"), k=ptr("packed") + k_at, v=ptr("packed") + v_at, q_out=ptr("q"), turns=ptr("turns"),
                             row_slot=ptr("slot"), row_entry=ptr("entry"), row_pos=ptr("pos"), rows=c["rows"], ld=s["packed"].shape[1],
                             q_heads=c["q_heads"], pairs=c["pairs"], rope_layout=1 if c["split"] else 0)
        args, out = (_cache(N, c, s["pool"]), call), {"q": s["q"], "k": s["pool"]["k"], "v": s["pool"]["v"]}
        f = nat.lib.m40llm_paged_append_async
    elif c["op"] == "attend":
        call = N.PagedAttention(q=ptr("q"), out=ptr("out"), row_slot=ptr("slot"), row_len=ptr("len"), weights_in=ptr("weights"),
                                weights_out=ptr("weights_out"), rows=c["rows"], q_heads=c["q_heads"], ld_weights=s["pool"]["entries"],
                                max_len=max(1, c["high"]), scale=1.0 / math.sqrt(c["dim"]))
        args, out = (_cache(N, c, s["pool"]), call), {"out": s["out"]}
        if c["weights"]:
            out["weights"] = s["weights_out"]
        f = nat.lib.m40llm_attention_paged_async
    elif c["op"] == "evict":
        to = _cache(N, c, s["to"])
        call = N.PagedEvict(to=ctypes.addressof(to), seq=ptr("seq"), len=ptr("len"), weights=ptr("weights"), weights_out=ptr("weights_out"),
                            entry_pos=ptr("pos"), entry_pos_out=ptr("pos_out"), origin=ptr("from"), new_len=ptr("new_len"), count=c["slots"],
                            keep=c["keep"], first=c["first"], recent=c["recent"], ld=s["pool"]["entries"], max_len=c["high"])
        args = (_cache(N, c, s["pool"]), call)
        s["keeps"] = to
        out = {"from": s["from"], "new_len": s["new_len"], "k": s["to"]["k"], "v": s["to"]["v"], "weights": s["weights_out"], "pos": s["pos_out"]}
        f = nat.lib.m40llm_paged_evict_async
    else:
        call = N.Logprobs(logits=ptr("logits"), tokens=ptr("tokens"), logprob=ptr("logprob"), rank=ptr("rank"), entropy=ptr("entropy"),
                          top_ids=ptr("top_ids"), top_logprobs=ptr("top_logprobs"), rows=c["rows"], n=c["n"], top=c["top"])
        args, out = (call,), {k: s[k] for k in ("logprob", "entropy", "rank")}
        if c["top"]:
            out |= {"top_ids": s["top_ids"], "top_logprobs": s["top_logprobs"]}
        f = nat.lib.m40llm_logprobs_f32_async
    return f, nat.ctx, args, [ctypes.byref(a) for a in args], out


def run(state):
    if own:
        if "calls" not in state:
            state["calls"] = _calls(state)
        f, ctx, _, refs, out = state["calls"]
        rc = f(ctx, *refs)
        if rc != 0:
            raise RuntimeError(f"call failed: {rc}")
        return out
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "score": _plain_score}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------------------- definitions
def work(case):
    op = case["op"]
    elem = 4 if case.get("type") == "f32" else 2
    if op == "append":
        rows, q, kv = case["rows"], case["q_heads"] * case["dim"], case["kv_heads"] * case["dim"]
        return {"bytes": rows * (4 * (q + 2 * kv) + 4 * q + 2 * elem * kv + 12), "flops": rows * 6 * case["pairs"] * (case["q_heads"] + case["kv_heads"])}
    if op == "attend":
        total, kv = sum(_lens(case, case["rows"])), case["kv_heads"] * case["dim"]
        bytes_ = 2 * elem * total * kv + 8 * case["rows"] * case["q_heads"] * case["dim"]
        return {"bytes": bytes_ + (8 * total * case["kv_heads"] if case["weights"] else 0), "flops": 4 * total * case["q_heads"] * case["dim"]}
    if op == "evict":
        lens = _lens(case, case["slots"])
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": case["kv_heads"] * (8 * sum(lens) + kept * (4 * elem * case["dim"] + 8 + 4)), "flops": 0}
    return {"bytes": case["rows"] * (4 * case["n"] + 16 + 8 * case["top"]), "flops": 4 * case["rows"] * case["n"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "score": _exact_score}[case["op"]](s)


def _exact_append(s):
    c, p = s["case"], s["pool"]
    x = s["packed"].double().cpu().numpy()
    D, H, KV, m = c["dim"], c["q_heads"], c["kv_heads"], c["pairs"]
    pos, turns = s["pos"].cpu().numpy().astype(np.float64), s["turns"].cpu().numpy()
    z = x[:, : (H + KV) * D].reshape(len(x), H + KV, D).copy()
    first = np.arange(m) if c["split"] else 2 * np.arange(m)
    second = first + (m if c["split"] else 1)
    # as complex numbers: a pair turns by a unit one
    t = np.outer(pos, turns[:m]) if m else np.zeros((len(x), 0))
    u = (z[..., first] + 1j * z[..., second]) * np.exp(2j * np.pi * (t - np.rint(t)))[:, None]
    z[..., first], z[..., second] = u.real, u.imag
    k, v = (np.zeros(p["k"].shape) for _ in range(2))
    table, entry, slot = p["table"].cpu().numpy(), s["entry"].cpu().numpy(), s["slot"].cpu().numpy()
    for r in range(len(x)):
        page, at = table[slot[r], entry[r] // c["page"]], entry[r] % c["page"]
        k[page, :, at] = z[r, H:]
        v[page, :, at] = x[r, (H + KV) * D:].reshape(KV, D)
    return {"q": z[:, :H].reshape(len(x), -1), "k": k, "v": v}


def _exact_attend(s):
    c, p = s["case"], s["pool"]
    H, D = c["kv_heads"], c["dim"]
    out = torch.zeros(c["rows"], c["q_heads"], D, dtype=torch.float64, device=_DEV)
    grown = s["weights"].double() if c["weights"] else None
    for r, (slot, n) in enumerate(zip(s["slot"].tolist(), s["len"].tolist())):
        pages = p["table"][slot].long()[: -(-n // c["page"])]
        for h in range(H if n else 0):
            k, v = (p[name][pages, h].reshape(-1, D)[:n].double() for name in ("k", "v"))
            group = slice(h * (c["q_heads"] // H), (h + 1) * (c["q_heads"] // H))
            w = torch.softmax(s["q"][r, group].double() @ k.T / math.sqrt(D), -1)
            out[r, group] = w @ v
            if grown is not None:
                grown[slot, h, :n] += w.sum(0)
    return {"out": out} if grown is None else {"out": out, "weights": grown}


def _exact_evict(s):
    c, p, to = s["case"], s["pool"], s["to"]
    pool = {name: p[name].double().cpu().numpy() for name in ("k", "v")}
    new = {name: np.zeros(to[name].shape) for name in ("k", "v")}
    weights, pos, lens = s["weights"].double().cpu().numpy(), s["pos"].cpu().numpy().astype(np.int64), s["len"].cpu().numpy()
    here, there = p["table"].cpu().numpy(), to["table"].cpu().numpy()
    grown, moved = np.zeros(weights.shape), np.full((c["slots"], c["kv_heads"], c["keep"]), -1)
    places = np.zeros(pos.shape, np.int64)
    for i, slot in enumerate(s["seq"].tolist()):
        n = int(lens[i])
        left = min(n, c["keep"])
        for h in range(c["kv_heads"]):
            end = pos[slot, h, :n].max() + 1
            held = (pos[slot, h, :n] < c["first"]) | (pos[slot, h, :n] + c["recent"] >= end)
            chosen = set(np.lexsort((np.arange(n), -weights[slot, h, :n], ~held))[:left].tolist())
            late = iter(sorted(e for e in chosen if e >= left))
            origin = np.array([e if e in chosen else next(late) for e in range(left)], np.int64)
            moved[i, h, :left] = origin
            grown[slot, h, :left], places[slot, h, :left] = weights[slot, h, origin], pos[slot, h, origin]
            e = np.arange(left)
            for name in ("k", "v"):
                new[name][there[slot, e // c["page"]], h, e % c["page"]] = pool[name][here[slot, origin // c["page"]], h, origin % c["page"]]
    return {"from": moved, "new_len": np.minimum(lens, c["keep"]), "k": new["k"], "v": new["v"], "weights": grown, "pos": places}


def _exact_score(s):
    c = s["case"]
    out = {"logprob": [], "entropy": [], "rank": [], "top_ids": [], "top_logprobs": []}
    for at in range(0, c["rows"], 256):
        logp = torch.log_softmax(s["logits"][at:at + 256].double(), -1)
        token = s["tokens"][at:at + 256].long()[:, None]
        out["logprob"].append(logp.gather(-1, token)[:, 0])
        out["entropy"].append(-torch.special.xlogy(logp.exp(), logp.exp()).sum(-1))
        places = torch.argsort(torch.argsort(-s["logits"][at:at + 256], dim=-1, stable=True), dim=-1)
        out["rank"].append(places.gather(-1, token)[:, 0] + 1)
        ids = torch.argsort(-s["logits"][at:at + 256], dim=-1, stable=True)[:, : c["top"]]
        out["top_ids"].append(ids)
        out["top_logprobs"].append(logp.gather(-1, ids))
    return {k: torch.cat(v) for k, v in out.items() if c["top"] or not k.startswith("top")}
