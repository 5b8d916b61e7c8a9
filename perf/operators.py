"""A session's cache in 4 bits, as cases that can be timed and checked: rows of keys and values written into it, rows read back, and
attention over it for one token, a few rows and prompts.

A row of K or V is cut into groups of 32 neighbouring entries.  A group is held as (lo, step) in the model's type D and 32 codes n of four
bits, and stands for lo + step * n:  lo = min x,  step = the smallest D number that is not below (max x - lo) / 15,  n = floor((x - lo) / step + 1/2).
A row of queries at position p sees the positions first <= j <= p.

``own`` chooses between the framework's calls (``Cache.write``, ``Cache.read``, ``Cache.attend``) and plain torch operations in 32 bits."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32
SHAPES = {  # query heads, key heads, entries of a head
    "8b": (32, 8, 128), "70b": (64, 8, 128), "0.6b": (16, 8, 128),   # the served models
    "medium": (8, 2, 64),                                            # the tests' middle size
    "single": (16, 16, 128),                                         # a key head per query head
    "wide": (8, 4, 256)}                                             # heads of the widest kind


def listed():
    return [
        # the decode loop's unit: one new position of one conversation goes into the cache
        dict(name="write one at 2048", kind="write", shape="8b", dtype="bf16", batch=1, seq=1, at=2048),
        # a short prompt of a small model
        dict(name="write 509", kind="write", shape="0.6b", dtype="f16", batch=1, seq=509, at=0),
        # a batch of long prompts, a quarter of the prefill benchmark's
        dict(name="write 8x4096", kind="write", shape="8b", dtype="bf16", batch=8, seq=4096, at=0),
        # part of a small conversation is handed to somebody else, as rows in D
        dict(name="read 1000", kind="read", shape="medium", dtype="f16", batch=2, rows=1000, at=24),
        # a long conversation is
        dict(name="read 32768", kind="read", shape="8b", dtype="bf16", batch=1, rows=32768, at=0),
        # one token of a small model with a short conversation: the call where launches and latency count most
        dict(name="attend step 0.6b 999", kind="attend", shape="0.6b", dtype="f16", batch=1, seq=1, at=998, first=0),
        # one token at the decode benchmark's context
        dict(name="attend step 8b 2048", kind="attend", shape="8b", dtype="bf16", batch=1, seq=1, at=2048, first=0),
        # one token of a very long conversation
        dict(name="attend step 8b 131072", kind="attend", shape="8b", dtype="bf16", batch=1, seq=1, at=131071, first=0),
        # one token each of many conversations: batched serving
        dict(name="attend steps 8b 32x4096", kind="attend", shape="8b", dtype="bf16", batch=32, seq=1, at=4095, first=0),
        # a few tokens at once through a sliding window of 4096
        dict(name="attend 7 rows at 5000", kind="attend", shape="medium", dtype="f16", batch=1, seq=7, at=5000, first=911),
        # the next message of a long conversation
        dict(name="attend portion 200 at 3000", kind="attend", shape="8b", dtype="bf16", batch=1, seq=200, at=3000, first=0),
        # a long prompt over its own keys
        dict(name="attend prompt 4096", kind="attend", shape="8b", dtype="bf16", batch=1, seq=4096, at=0, first=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["write", "read"] + ["attend"] * 4)
    shape, dtype = rng.choice(sorted(SHAPES)), rng.choice(["bf16", "f16"])
    heads, kv, hd = SHAPES[shape]
    batch = rng.choice([1, 1, 1, 2, 3, _log(rng, 4, 32)])
    held = 131072 * 8 * 128 // (kv * hd * batch)   # positions of the largest cache
    if kind == "write":
        return dict(kind=kind, shape=shape, dtype=dtype, batch=batch, seq=_log(rng, 1, min(8192, held // 4)), at=rng.choice([0, 0, _log(rng, 1, 4000)]))
    if kind == "read":
        return dict(kind=kind, shape=shape, dtype=dtype, batch=batch, rows=_log(rng, 1, min(32768, held // 4)), at=rng.choice([0, rng.randint(1, 999)]))
    what = rng.choice(["step", "step", "few", "portion", "prompt"])
    if what in ("step", "few"):
        seq, at = 1 if what == "step" else rng.randint(2, 16), _log(rng, 1, min(131072, held) - 16)
    elif what == "portion":
        batch = min(batch, 3)
        at = _log(rng, 1, 8000)
        seq = _log(rng, 17, min(1000, 4096 * 2048 * 32 // (batch * heads * (at + 1000))))
    else:
        batch, at = 1, 0
        seq = _log(rng, 17, 4096 if heads <= 32 else 2048)
    first = 0
    if rng.random() < 0.3:   # a sliding window that this call's first row fills
        first = rng.randint(0, at)
    return dict(kind=kind, shape=shape, dtype=dtype, batch=batch, seq=seq, at=at, first=first)


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 8 + what)
    return g


def _rows(case, seed, what, n):
    """n positions of keys (what 0) or values (what 1), [batch, n, kv heads, hd] in D: channels of different widths, some of them off centre, as
    projections behind a norm have them."""
    _, kv, hd = SHAPES[case["shape"]]
    g = _generator(seed, what)
    width = torch.exp(0.5 * torch.randn((kv, hd), generator=g, device=DEV))
    centre = torch.randn((kv, hd), generator=g, device=DEV) * (torch.rand((kv, hd), generator=g, device=DEV) < 0.25)
    return (torch.randn((case["batch"], n, kv, hd), generator=g, device=DEV) * width + centre).to(DT[case["dtype"]])


def _queries(case, seed):
    heads, _, hd = SHAPES[case["shape"]]
    return torch.randn((case["batch"], case["seq"], heads, hd), generator=_generator(seed, 2), device=DEV).to(DT[case["dtype"]])


def _held(case):
    """Positions that the cache holds before the call."""
    return case["at"] + {"write": 0, "read": case.get("rows", 0), "attend": case.get("seq", 0)}[case["kind"]]


# ---------------------------------------------------------------------------------------------- the plain form
def _pack(x):
    """Rows [..., hd] in D -> codes [..., hd / 32, 32] (bytes), lo and step [..., hd / 32, 1] in D."""
    f = x.float().unflatten(-1, (-1, GROUP))
    lo = f.amin(-1, keepdim=True)
    span = f.amax(-1, keepdim=True) - lo
    want = span / torch.full_like(span, 15)   # a plain number would be multiplied by 1 / 15, which rounds twice
    near = want.to(x.dtype)
    step = torch.where(near.float() < want, (near.view(torch.int16) + 1).view(x.dtype), near)
    if x.dtype == torch.bfloat16:
        step = torch.where(span > 0, step.clamp_min(2.0 ** -126), step)
    n = torch.floor((f - lo) / torch.where(step > 0, step.float(), 1.0) + 0.5)
    return n.to(torch.uint8), lo.to(x.dtype), step


def _values(packed):
    n, lo, step = packed
    return (lo.float() + step.float() * n.float()).flatten(-2)


def _attend(q, k, v, at, first):
    """q [batch, seq, heads, hd], k and v [batch, positions, kv heads, hd], in 32 bits."""
    b, s, heads, hd = q.shape
    n, kv = k.shape[1], k.shape[2]
    q = q.reshape(b, s, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    p = (q @ k.permute(0, 2, 3, 1)) * hd ** -0.5
    j, i = torch.arange(n, device=q.device), torch.arange(at, at + s, device=q.device)
    p = p.unflatten(2, (-1, s)).masked_fill_(((j > i[:, None]) | (j < first)), -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    o = (p.flatten(2, 3) @ v.permute(0, 2, 1, 3)) / p.sum(-1).flatten(2, 3)[..., None]
    return o.unflatten(2, (-1, s)).permute(0, 3, 1, 2, 4).reshape(b, s, heads, hd)


# ---------------------------------------------------------------------------------------------- the framework's calls
_contexts = {}   # a serving program keeps one per model


def _cache(case, positions):
    from cake_b200.config import Config
    from cake_b200.model import Cache, Context
    key = (case["shape"], case["dtype"])
    if key not in _contexts:
        heads, kv, hd = SHAPES[case["shape"]]
        _contexts[key] = Context(Config(heads * hd, 64, 256, 1, heads, kv, head_dim=hd, max_seq_len=1 << 18), {}, case["dtype"])
    return Cache(_contexts[key], case["batch"], positions, bits=4)


# ---------------------------------------------------------------------------------------------- the cases
def prepare(case, seed):
    held, st = _held(case), {"case": case}
    k, v = (_rows(case, seed, what, held + (case["seq"] if case["kind"] == "write" else 0)) for what in (0, 1))
    if case["kind"] == "write":   # columns of a fused projection [tokens, heads + 2 kv heads, hd], as a block's product leaves them
        heads, kv, hd = SHAPES[case["shape"]]
        fused = torch.zeros((case["batch"], case["seq"], heads + 2 * kv, hd), dtype=k.dtype, device=DEV)
        fused[:, :, heads:heads + kv] = k[:, held:]
        fused[:, :, heads + kv:] = v[:, held:]
        st["k"], st["v"] = fused[:, :, heads:heads + kv], fused[:, :, heads + kv:]
    if case["kind"] == "attend":
        st["q"] = _queries(case, seed)
    if own:
        st["cache"] = _cache(case, held + case.get("seq", 0))
        if held:
            st["cache"].write(0, k[:, :held], v[:, :held], 0)
    elif case["kind"] != "write":
        st["packed"] = _pack(k), _pack(v)
    return st


def run(st):
    case = st["case"]
    at, dtype = case["at"], DT[case["dtype"]]
    if case["kind"] == "write":
        if own:
            st["cache"].write(0, st["k"], st["v"], at)
            return st["cache"].read(0, 0, at, case["seq"]), st["cache"].read(0, 1, at, case["seq"])
        return [_values(_pack(x)).to(dtype).transpose(1, 2) for x in (st["k"], st["v"])]
    if case["kind"] == "read":
        if own:
            return st["cache"].read(0, 0, at, case["rows"]), st["cache"].read(0, 1, at, case["rows"])
        return [_values([t[:, at:] for t in p]).to(dtype).transpose(1, 2) for p in st["packed"]]
    if own:
        return st["cache"].attend(0, st["q"], at, first=case["first"])
    return _attend(st["q"].float(), _values(st["packed"][0]), _values(st["packed"][1]), at, case["first"]).to(dtype)


def work(case):
    heads, kv, hd = SHAPES[case["shape"]]
    entries = 2 * case["batch"] * kv * hd                 # of one position, keys and values
    packed = entries * (GROUP // 2 + 4) / GROUP           # its bytes in the cache
    if case["kind"] == "write":                           # rows in, packed out; packed in, rows out
        return {"bytes": 2 * case["seq"] * (2 * entries + packed), "flops": case["seq"] * entries * 6}
    if case["kind"] == "read":
        return {"bytes": case["rows"] * (2 * entries + packed), "flops": case["rows"] * entries * 2}
    s, at, first = case["seq"], case["at"], case["first"]
    pairs = s * (at - first) + s * (s + 1) // 2
    return {"bytes": (at + s - first) * packed + 2 * 2 * case["batch"] * s * heads * hd, "flops": 4 * case["batch"] * heads * hd * pairs}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _stands_for(x):
    """What rows x [..., hd] in D stand for in the cache, from the definition, in 64 bits."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    bits, least = (8, -126) if x.dtype == torch.bfloat16 else (11, -14)   # of a D number; the exponent of its smallest normal one
    want = (hi - lo) / 15
    ulp = torch.exp2(torch.floor(torch.log2(want.clamp_min(2.0 ** least))).clamp_min(least) - (bits - 1))
    step = torch.ceil(want / ulp) * ulp
    if x.dtype == torch.bfloat16:
        step = torch.where(hi > lo, step.clamp_min(2.0 ** least), step)
    n = torch.where(step > 0, torch.floor((g - lo) / step.clamp_min(2.0 ** -140) + 0.5), torch.zeros_like(g))
    return (lo + step * n).reshape(x.shape)


def exact(case, seed):
    n = _held(case) + (case["seq"] if case["kind"] == "write" else 0)
    k, v = _stands_for(_rows(case, seed, 0, n)), _stands_for(_rows(case, seed, 1, n))
    if case["kind"] != "attend":
        return k[:, case["at"]:].transpose(1, 2), v[:, case["at"]:].transpose(1, 2)
    q = _queries(case, seed).double()
    heads, kv, hd = SHAPES[case["shape"]]
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(case["at"], case["at"] + case["seq"], device=DEV)[:, None]
    seen[:, :case["first"]] = False
    for b in range(case["batch"]):
        for h in range(heads):
            s = torch.mv(k[b, :, h * kv // heads], q[b, 0, h])[None] if case["seq"] == 1 else q[b, :, h] @ k[b, :, h * kv // heads].T
            w = torch.softmax(torch.where(seen, s / math.sqrt(hd), torch.full_like(s, -math.inf)), -1)
            out[b, :, h] = w @ v[b, :, h * kv // heads]
    return out
