"""Conversations whose keys and values lie in pages of one pool, as cases that can be timed and checked: a step's rows rotated and appended, and
attention over the pages for one token each of many conversations, for a few tokens, for portions of prompts and for steps that mix them.

A step brings new rows of some conversations, packed one behind another: rows [T, heads, hd].  Row i of a conversation that held n positions stands at
position p = n + i.  Appending rotates q and k by the row of p in the tables cos and sin (pairs (e, e + rot / 2) of the first rot entries; entries behind
them stay), and puts k and v into the conversation's pages.  Attention of a row at position p sees the positions j <= p, with a window w only p - w < j <= p.

``own`` chooses between the framework's calls (``PagedCache.step``, ``append``, ``attend``, ``read``) and plain torch operations in 32 bits over pages that
are found through a table."""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
THETA = 500000.0
SHAPES = {  # query heads, key heads, entries of a head
    "8b": (32, 8, 128), "70b": (64, 8, 128), "0.6b": (16, 8, 128),   # the served models
    "medium": (8, 2, 64),                                            # the tests' middle size
    "single": (16, 16, 128),                                         # a key head per query head
    "wide": (8, 4, 256)}                                             # heads of the widest kind


def _case(kind, shape, dtype, page, n, rows, held, mix=1, window=0, rot=0, ones=False, name=None):
    """n conversations with rows = (least, most) new positions on held = (least, most); the first one has the most of both.  ones: the others bring one."""
    c = dict(kind=kind, shape=shape, dtype=dtype, page=page, n=n, rows_min=rows[0], rows_max=rows[1], held_min=held[0], held_max=held[1], mix=mix, window=window,
             rot=rot or SHAPES[shape][2], ones=ones)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the decode loop's unit: one new position of one conversation
        _case("append", "8b", "bf16", 64, 1, (1, 1), (2048, 2048), name="append one at 2048"),
        # one token each of a batch of conversations of a large model
        _case("append", "70b", "f16", 16, 32, (1, 1), (100, 4000), mix=2, name="append 32 tokens"),
        # prompts of several lengths arrive together
        _case("append", "8b", "bf16", 64, 8, (500, 4096), (0, 0), mix=3, name="append 8 prompts"),
        # heads that are rotated in part, small pages, a second portion of each prompt
        _case("append", "medium", "f16", 16, 12, (1, 700), (1, 999), mix=4, rot=32, name="append portions, half rotated"),
        # one token of a small model with a short conversation: the call where launches and latency count most
        _case("attend", "0.6b", "f16", 64, 1, (1, 1), (998, 998), name="token 0.6b at 998"),
        # batched serving: one token each of conversations of many lengths
        _case("attend", "8b", "bf16", 64, 32, (1, 1), (200, 8191), mix=5, name="32 tokens 8b to 8191"),
        # one token of a very long conversation
        _case("attend", "8b", "bf16", 64, 1, (1, 1), (131071, 131071), name="token 8b at 131071"),
        # many short conversations in small pages, behind a sliding window
        _case("attend", "medium", "f16", 16, 100, (1, 1), (5, 3000), mix=6, window=1024, name="100 tokens medium, window 1024"),
        # a few proposed tokens each are checked at once
        _case("attend", "0.6b", "bf16", 32, 9, (3, 5), (300, 5000), mix=7, name="few tokens 0.6b"),
        # a prompt over its own keys
        _case("attend", "8b", "bf16", 64, 1, (4096, 4096), (0, 0), name="prompt 8b 4096"),
        # the next messages of several conversations
        _case("attend", "70b", "f16", 16, 6, (60, 900), (150, 5000), mix=8, name="portions 70b"),
        # a portion of a prompt runs beside the tokens of the others, heads of the widest kind
        _case("attend", "wide", "bf16", 128, 24, (512, 512), (40, 4000), mix=9, ones=True, name="mixed step wide"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend"])
    shape, dtype, page = rng.choice(sorted(SHAPES)), rng.choice(["bf16", "f16"]), rng.choice([16, 32, 64, 128])
    heads, kv, hd = SHAPES[shape]
    n, mix = rng.choice([1, 2, _log(rng, 3, 64)]), rng.randint(1, 10 ** 6)
    room = 131072 * 8 * 128 // (kv * hd)        # positions of the largest pool
    if kind == "append":
        most = _log(rng, 1, 16384 * 48 * 128 // ((heads + 2 * kv) * hd * n))
        rows = rng.choice([(1, 1), (1, most), (most, most)])
        held = _log(rng, 1, max(1, min(8000, room // n)))
        return _case(kind, shape, dtype, page, n, rows, rng.choice([(0, 0), (1, held), (held, held)]), mix, rot=rng.choice([hd, hd, hd // 2]))
    what = rng.choice(["tokens", "tokens", "few", "portions", "mixed"])
    if what in ("tokens", "few"):
        rows = (1, 1) if what == "tokens" else (1, rng.randint(2, 16))
        most = _log(rng, 1, min(131071, room // n) - 16)
        held = (rng.choice([0, 1, most]), most)
        if held[0] == 0:
            held = (1, most)
    else:
        n = min(n, 8) if what == "portions" else n
        pairs = 4096 * 2048 * 32 // heads * 128 // hd // (n if what == "portions" else 2)
        at = rng.choice([1, _log(rng, 1, max(1, min(8000, room // n // 2)))])
        most = max(2, int(math.sqrt(at * at + 2.0 * pairs) - at))
        most = _log(rng, 2, min(most, 4096))
        rows, held = (_log(rng, 1, most), most), (1, at)
    window = rng.choice([0, 0, _log(rng, 1, 6000)])
    return _case(kind, shape, dtype, page, n, rows, held, mix, window, ones=what == "mixed")


def _conversations(case):
    """(positions held, new rows) of each conversation."""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["n"]):
        lo, hi = case["held_min"], case["held_max"]
        held = hi if i == 0 or lo == hi else _log(rng, max(1, lo), hi)
        rows = case["rows_max"] if i == 0 else 1 if case["ones"] else _log(rng, case["rows_min"], case["rows_max"])
        got.append((held, rows))
    return got


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 8 + what)
    return g


def _rows(case, seed, what, n):
    """n rows of keys (what 0) or values (what 1), [n, kv heads, hd] in D: channels of different widths, some of them off centre, as projections behind
    a norm have them."""
    _, kv, hd = SHAPES[case["shape"]]
    g = _generator(seed, what)
    width = torch.exp(0.5 * torch.randn((kv, hd), generator=g, device=DEV))
    centre = torch.randn((kv, hd), generator=g, device=DEV) * (torch.rand((kv, hd), generator=g, device=DEV) < 0.25)
    return (torch.randn((n, kv, hd), generator=g, device=DEV) * width + centre).to(DT[case["dtype"]])


def _queries(case, seed, n):
    heads, _, hd = SHAPES[case["shape"]]
    return torch.randn((n, heads, hd), generator=_generator(seed, 2), device=DEV).to(DT[case["dtype"]])


def _tables(case):
    """cos and sin [positions, rot / 2]: computed in 64 bits, held in 32."""
    half = case["rot"] // 2
    top = max(held + rows for held, rows in _conversations(case))
    f = THETA ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    a = torch.arange(top, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


# ---------------------------------------------------------------------------------------------- the plain form
def _rotated(x, cos, sin):
    """x [n, heads, hd] in D by the tables' rows cos, sin [n, half], in 32 bits, rounded once."""
    half = cos.shape[1]
    f, c, s = x.float(), cos[:, None], sin[:, None]
    a, b = f[..., :half], f[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, f[..., 2 * half:]], -1).to(x.dtype)


def _attend(q, k, v, at, window):
    """q [rows, heads, hd] at positions at .., k and v [positions, kv heads, hd], in 32 bits."""
    s, heads, hd = q.shape
    n, kv = k.shape[0], k.shape[1]
    q = q.reshape(s, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
    p = (q @ k.permute(1, 2, 0)) * hd ** -0.5
    if s > 1 or window:
        j, i = torch.arange(n, device=q.device), torch.arange(at, at + s, device=q.device)[:, None]
        hidden = j > i
        if window:
            hidden |= j <= i - window
        p = p.unflatten(1, (-1, s)).masked_fill_(hidden, -math.inf).flatten(1, 2)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    o = (p @ v.permute(1, 0, 2)) / p.sum(-1, keepdim=True)
    return o.unflatten(1, (-1, s)).permute(2, 0, 1, 3).reshape(s, heads, hd)


# ---------------------------------------------------------------------------------------------- the framework's calls
_contexts = {}   # a serving program keeps one per model


def _cache(case, positions, tables):
    from cake_b200.config import Config
    from cake_b200.model import Context, PagedCache
    key = (case["shape"], case["dtype"])
    if key not in _contexts:
        heads, kv, hd = SHAPES[case["shape"]]
        _contexts[key] = Context(Config(heads * hd, 64, 256, 1, heads, kv, head_dim=hd, max_seq_len=1 << 18), {}, case["dtype"])
    page = case["page"]
    return PagedCache(_contexts[key], sum((p + page - 1) // page for p in positions), page, max_seqs=len(positions), max_seq=max(positions), rotation=tables)


# ---------------------------------------------------------------------------------------------- the cases
def prepare(case, seed):
    talks, page = _conversations(case), case["page"]
    held, rows = [h for h, _ in talks], [r for _, r in talks]
    new = sum(rows)
    k, v = (_rows(case, seed, what, sum(held) + new) for what in (0, 1))   # what is held first, conversation by conversation, then the step's rows
    tables = _tables(case)
    st = {"case": case, "talks": talks, "q": _queries(case, seed, new)}
    heads, kv, hd = SHAPES[case["shape"]]
    if case["kind"] == "append":   # columns of a fused projection [tokens, heads + 2 kv heads, hd], as a block's product leaves them
        fused = torch.cat([st["q"], k[sum(held):], v[sum(held):]], 1)
        st["q"], st["k"], st["v"] = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    if own:
        cache = _cache(case, [h + r for h, r in talks], tables)
        ids = [cache.add() for _ in talks]
        some = [i for i, h in enumerate(held) if h]
        if some:
            cache.step([ids[i] for i in some], [held[i] for i in some])
            cache.append(0, None, k[:sum(held)], v[:sum(held)], rotate=False)
        cache.step(ids, rows)
        if case["kind"] == "attend":
            cache.append(0, None, k[sum(held):], v[sum(held):], rotate=False)
        st["cache"] = cache
        return st
    count = [(h + r + page - 1) // page for h, r in talks]
    order = torch.randperm(sum(count), generator=_generator(seed, 3), device=DEV)
    st["pages"] = list(order.split(count))
    st["kp"], st["vp"] = (torch.zeros((sum(count), page, kv, hd), dtype=k.dtype, device=DEV) for _ in range(2))
    a, b = 0, sum(held)
    st["positions"], st["places"] = [], []
    for (h, r), pages in zip(talks, st["pages"]):
        p = torch.arange(h + r, device=DEV)
        place = pages[p // page] * page + p % page
        n = h if case["kind"] == "append" else h + r
        for pool, x in ((st["kp"], k), (st["vp"], v)):
            pool.view(-1, kv, hd)[place[:n]] = torch.cat([x[a:a + h], x[b:b + r]])[:n]
        st["positions"].append(p[h:])
        st["places"].append(place[h:])
        a, b = a + h, b + r
    st["positions"], st["places"] = torch.cat(st["positions"]), torch.cat(st["places"])
    st["cos"], st["sin"] = tables
    return st


def run(st):
    case = st["case"]
    if case["kind"] == "append":
        if own:
            q = st["cache"].append(0, st["q"], st["k"], st["v"])
            return q, *st["cache"].read(0)
        cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
        _, kv, hd = SHAPES[case["shape"]]
        kp, vp = st["kp"].view(-1, kv, hd), st["vp"].view(-1, kv, hd)
        kp[st["places"]] = _rotated(st["k"], cos, sin)
        vp[st["places"]] = st["v"]
        return _rotated(st["q"], cos, sin), kp[st["places"]], vp[st["places"]]
    if own:
        return st["cache"].attend(0, st["q"], window=case["window"])
    out, at = [], 0
    for (held, rows), pages in zip(st["talks"], st["pages"]):
        k, v = (pool[pages].flatten(0, 1)[:held + rows].float() for pool in (st["kp"], st["vp"]))
        out.append(_attend(st["q"][at:at + rows].float(), k, v, held, case["window"]))
        at += rows
    return torch.cat(out).to(DT[case["dtype"]])


def _pairs(held, rows, window):
    """Positions seen by a conversation's rows, one row after another, and by any of them."""
    if not window:
        return rows * held + rows * (rows + 1) // 2, held + rows
    short = max(0, min(rows, window - held))       # rows that see everything
    return short * held + short * (short + 1) // 2 + (rows - short) * window, min(held + rows, window + rows - 1)


def work(case):
    heads, kv, hd = SHAPES[case["shape"]]
    talks = _conversations(case)
    new = sum(r for _, r in talks)
    if case["kind"] == "append":   # rows in, q out, k and v into pages; pages in, k and v out; a row of each table
        return {"bytes": new * (2 * hd * (2 * heads + 2 * kv + 2 * kv + 4 * kv) + 4 * case["rot"]), "flops": 3 * new * (heads + kv) * case["rot"]}
    seen = [_pairs(h, r, case["window"]) for h, r in talks]
    return {"bytes": sum(s for _, s in seen) * 4 * kv * hd + 4 * new * heads * hd, "flops": 4 * heads * hd * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    talks = _conversations(case)
    heads, kv, hd = SHAPES[case["shape"]]
    held = sum(h for h, _ in talks)
    new = sum(r for _, r in talks)
    k, v, q = _rows(case, seed, 0, held + new), _rows(case, seed, 1, held + new), _queries(case, seed, new)
    if case["kind"] == "append":
        cos, sin = (t.double() for t in _tables(case))
        half, p = case["rot"] // 2, torch.cat([torch.arange(h, h + r, device=DEV) for h, r in talks])
        turn = torch.complex(cos[p], sin[p])[:, None, :]
        out = []
        for x in (q, k[held:]):
            x = x.double().clone()
            z = torch.complex(x[:, :, :half].contiguous(), x[:, :, half:2 * half].contiguous()) * turn
            x[:, :, :half], x[:, :, half:2 * half] = z.real, z.imag
            out.append(x)
        return out[0], out[1], v[held:].double()
    out = torch.empty((new, heads, hd), dtype=torch.float64, device=DEV)
    a, b = 0, 0
    for h, r in talks:
        kd, vd = (torch.cat([x[a:a + h], x[held + b:held + b + r]]).double() for x in (k, v))
        i, j = torch.arange(h, h + r, device=DEV)[:, None], torch.arange(h + r, device=DEV)[None, :]
        seen = (j <= i) & (j > i - (case["window"] or h + r + 1))
        for g in range(heads):
            qd = q[b:b + r, g].double()
            s = torch.mv(kd[:, g * kv // heads], qd[0])[None] if r == 1 else qd @ kd[:, g * kv // heads].T
            w = torch.softmax(torch.where(seen, s / math.sqrt(hd), torch.full_like(s, -math.inf)), -1)
            out[b:b + r, g] = w @ vd[:, g * kv // heads]
        a, b = a + h, b + r
    return out
