"""Calls on caches in pages that are refused or answered on the host."""
import types

import pytest
import torch

from cake_b200 import model
from cake_b200.capi import CakeB200Error, lib
from cake_b200.config import Config
from cake_b200.model import Context, PagedCache

EINVAL, ESTATE = -1, -4


def ctx_for(heads, kv, hd, dtype="bf16", layers=1):
    return Context(Config(heads * hd, 64, 256, layers, heads, kv, head_dim=hd, max_seq_len=4096), {}, dtype)


def hosted(monkeypatch, **calls):
    """A PagedCache of 2 sequences, 2 key heads of 64, in front of a library that is these functions."""
    cache = PagedCache.__new__(PagedCache)
    cache.h, cache.max_seqs, cache._kv, cache._hd, cache._dtype, cache._rows = None, 2, 2, 64, torch.bfloat16, 5
    cache._one = torch.empty(1, dtype=torch.bfloat16)
    cache._kv_like = cache._one.expand(torch.Size((5, 2, 64)))
    cache._lib = types.SimpleNamespace(**calls)
    monkeypatch.setattr(PagedCache, "_stream", lambda self: 1)
    return cache


def refused(code, f, *a, **kw):
    with pytest.raises(CakeB200Error) as e:
        f(*a, **kw)
    assert e.value.code == code, str(e.value)


# ------------------------------------------------------------------------------------------------ reading
@pytest.mark.parametrize("seq", [-1, -2, -2 ** 31, 2 ** 32 - 1, 2 ** 32, 2])
def test_no_sequence_is_read_as_the_step(monkeypatch, seq):
    """The library writes a step's rows where the sequence's number is below 0: room that was made for others never gets there."""
    def read(*a):
        raise AssertionError(f"the library was asked for {a}")
    cache = hosted(monkeypatch, cake_b200_pages_read=read)
    refused(EINVAL, cache.read, 0, seq, 0, 1)


@pytest.mark.gpu
def test_room_for_other_rows_than_the_steps_is_refused():
    ctx = ctx_for(8, 2, 64)
    cache = PagedCache(ctx, 8, 16, max_seqs=2, max_seq=60)
    s = cache.add()
    cache.step([s], [5])
    x = torch.randn(5, 2, 64, device="cuda").bfloat16()
    cache.append(0, None, x, -x)
    k, v = torch.empty_like(x), torch.empty_like(x)
    for n in (-1, 1, 4, 6):   # refused in front of any launch; there is room for all five rows here in any case
        assert lib().cake_b200_pages_read(cache.h, 0, -1, 0, n, k.data_ptr(), v.data_ptr(), cache._stream()) == EINVAL
    for n in (0, 5):
        k.zero_(), v.zero_()
        assert lib().cake_b200_pages_read(cache.h, 0, -1, 0, n, k.data_ptr(), v.data_ptr(), cache._stream()) == 0
        assert torch.equal(v, -x) and torch.equal(k, cache.read(0, s)[0])
    refused(EINVAL, cache.read, 0, -1, 0, 1)
    refused(EINVAL, cache.read, 0, -1)
    ctx.close()


# ------------------------------------------------------------------------------------------------ results on their inputs
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3])
def test_queries_rotated_onto_rows_that_are_still_read_are_refused(rows):
    """A fused projection [rows, q | k | v]: results that would lie on rows of it are no call; a contiguous q in place, and room beside it, are."""
    heads, kv, hd = 8, 2, 64
    wide, row = (heads + 2 * kv) * hd, heads * hd
    ctx = ctx_for(heads, kv, hd)
    cache = PagedCache(ctx, 8, 16, max_seqs=2, max_seq=60)
    s = cache.add()
    cache.step([s], [4])
    x = torch.randn(4, kv, hd, device="cuda").bfloat16()
    cache.append(0, None, x, x)
    cache.step([s], [rows])
    buf = torch.randn(8 * wide, device="cuda").bfloat16()
    fused = buf[wide:(1 + rows) * wide].view(rows, heads + 2 * kv, hd)
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    want, before = cache.append(0, q, k, v), buf.clone()
    wk, wv = cache.read(0)
    at = fused.data_ptr()

    def call(out, q_at=at, tok=wide, k_at=at + 2 * row, v_at=at + 2 * (row + kv * hd), kv_tok=wide):
        return lib().cake_b200_pages_append(cache.h, 0, q_at, tok, k_at, kv_tok, v_at, kv_tok, out, 1, cache._stream())
    torch.cuda.synchronize()
    inside = [at + 16, at + 2 * (row - 8), at - 16, at + 2 * row, at + 2 * (wide - 8)]
    if rows > 1:
        inside += [at, at + 2 * wide, at + 2 * ((rows - 1) * wide + 8)]
    for out in inside:
        assert call(out) == EINVAL, (out - at) / 2
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    free = buf.data_ptr() + 2 * (1 + rows) * wide   # right behind, and right in front
    for out in (free, at - 2 * rows * row):
        if out < buf.data_ptr():
            continue
        assert call(out) == 0
        torch.cuda.synchronize()
        first = (out - buf.data_ptr()) // 2
        assert torch.equal(buf[first:first + rows * row].view(rows, heads, hd), want)
        buf.copy_(before)
    qc, kc, vc = (t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    for k_at, v_at in ((kc.data_ptr(), qc.data_ptr()), (qc.data_ptr(), vc.data_ptr())):   # its keys, or values, are its queries
        assert call(qc.data_ptr(), qc.data_ptr(), row, k_at, v_at, kv * hd) == EINVAL
    assert call(qc.data_ptr(), qc.data_ptr(), row, kc.data_ptr(), vc.data_ptr(), kv * hd) == 0
    assert torch.equal(qc, want)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0), (wk, wv)))
    if rows == 1:   # one row is contiguous at any stride
        assert call(at) == 0
        torch.cuda.synchronize()
        assert torch.equal(fused[:, :heads], want)
    ctx.close()


# ------------------------------------------------------------------------------------------------ replays
@pytest.mark.gpu
@pytest.mark.parametrize("how", ["drop", "truncate"])
def test_a_replay_behind_a_step_that_was_ended_touches_no_sequence(how):
    """One of a step's sequences goes, the graph is replayed all the same: rows of all that are left stay, calls are refused, and what comes next is as if it had not run."""
    heads, kv, hd = 8, 2, 64
    ctx = ctx_for(heads, kv, hd)
    cache = PagedCache(ctx, 24, 16, max_seqs=4, max_seq=100)
    g = torch.Generator(device="cuda").manual_seed(3)

    def rows(n, x):
        return torch.randn((n, x, hd), generator=g, device="cuda").bfloat16()
    a, b, other = cache.add(), cache.add(), cache.add()
    held = [37, 30, 45]
    cache.step([a, b, other], held)
    k, v = rows(sum(held), kv), rows(sum(held), kv)
    cache.append(0, None, k, v, rotate=False)
    cache.step([a, b], [1, 3])
    q, nk, nv = rows(4, heads), rows(4, kv), rows(4, kv)

    def calls():
        cache.append(0, None, nk, nv, rotate=False)
        return cache.attend(0, q)
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    graph.replay()
    want = out.clone()
    kept = {s: cache.read(0, s) for s in (a, other)}
    if how == "drop":
        cache.drop(b)
        fresh = cache.add()   # in the same row of the table
        assert fresh == b
    else:
        cache.truncate(b, 20)
        kept[b] = cache.read(0, b)
    nk.neg_(), nv.neg_()
    nk[0].neg_(), nv[0].neg_()   # (the rows of the one that is left)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0])
    refused(ESTATE, cache.attend, 0, q)
    refused(ESTATE, cache.append, 0, None, nk, nv, False)
    for s, (x, y) in kept.items():
        assert all(torch.equal(p, r) for p, r in zip(cache.read(0, s), (x, y)))
    grow = 33 if how == "drop" else 13   # b, or the one in its place, up to the same length: over pages that the replay wrote to
    cache.step([b], [grow])
    k2, v2 = rows(grow, kv), rows(grow, kv)
    cache.append(0, None, k2, v2, rotate=False)
    x, y = (k2, v2) if how == "drop" else (torch.cat(p) for p in zip(kept[b], (k2, v2)))
    got = cache.read(0, b)
    assert torch.equal(got[0], x) and torch.equal(got[1], y)
    for s in (a, other):
        assert all(torch.equal(p, r) for p, r in zip(cache.read(0, s), kept[s]))
    del graph
    ctx.close()


# ------------------------------------------------------------------------------------------------ streams
@pytest.mark.gpu
@pytest.mark.parametrize("copied", [False, True])
def test_rotation_tables_that_are_still_on_their_way(copied):
    """Tables made on one stream, where the cache is made too, and used on another one at once; copied: into the order that the library takes."""
    ctx = ctx_for(8, 2, 64)
    angles = torch.arange(60, device="cuda", dtype=torch.float64)[:, None] * 10.0 ** -torch.linspace(0, 4, 32, device="cuda", dtype=torch.float64)
    cos, sin = angles.cos().float(), angles.sin().float()
    q, k = (torch.randn(40, x, 64, device="cuda").bfloat16() for x in (8, 2))

    def rows(cache):
        cache.step([cache.add()], [40])
        return cache.append(0, q, k, k)
    want = rows(PagedCache(ctx, 4, 16, max_seqs=1, max_seq=60, rotation=(cos, sin)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.zeros(32, 60, device="cuda").T if copied else torch.zeros(60, 32, device="cuda") for _ in range(2)]
        torch.cuda._sleep(50_000_000)   # some 30 ms
        late[0].copy_(cos), late[1].copy_(sin)
        cache = PagedCache(ctx, 4, 16, max_seqs=1, max_seq=60, rotation=tuple(late))
    got = rows(cache)
    assert torch.equal(got, want)
    ctx.close()
