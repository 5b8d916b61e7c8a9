"""Caches in four bits: calls one after another that no other test makes."""
from ctypes import byref, c_float, c_int, c_void_p

import pytest
import torch

from cake_b200.capi import CakeB200Error, check, lib
from cake_b200.model import Cache, Context, TextModelBase
from tests.test_packed_cache import EINVAL, ESTATE, check_attention, ctx_for, filled, queries, rows
from tests.util import checkpoint, medium_config


@pytest.mark.gpu
def test_a_refused_begin_leaves_the_graph_refused():
    """Rows were written behind the decode graph's back; a begin that is refused does not make it runnable."""
    cfg = medium_config(num_hidden_layers=1)
    ctx = Context(cfg, checkpoint(cfg, "bf16", std=0.05, peaked=True), "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    m.forward([[1, 2, 3, 4, 5, 6, 7, 8]], 0)
    m.index_pos = 8
    m.decode_build()
    m.decode_greedy(5, 2)
    k = rows(1, 3, 2, 64, "bf16", 1)
    ctx.cache.write(0, k, k, 6)
    for token, pos, code in ((cfg.vocab_size, 9, EINVAL), (5, 8, ESTATE)):
        with pytest.raises(CakeB200Error) as e:
            check(lib().cake_b200_decode_begin(ctx.h, token, pos))
        assert e.value.code == code
        with pytest.raises(CakeB200Error) as e:
            check(lib().cake_b200_decode_run(ctx.h, 1))
        assert e.value.code == ESTATE
    m.index_pos = 9
    assert len(m.decode_greedy(5, 2)) == 2 and ctx.cache.len(0) == 11
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,s", [(8, 2, 128, 1), (8, 2, 64, 6), (4, 2, 256, 3), (32, 8, 128, 150)])
def test_values_of_any_size_of_bf16(heads, kv, hd, s):
    """Powers of two on V alone change nothing but the result's exponent."""
    ctx = ctx_for(heads, kv, hd, "bf16")
    n = s + 50
    k, v, q = rows(1, n, kv, hd, "bf16", 1), rows(1, n, kv, hd, "bf16", 2), queries(1, s, heads, hd, "bf16", 3)
    cache, want = Cache(ctx, 1, n, bits=4), None
    for e in (0, -100, 60, 114):
        cache.write(0, k, v * 2.0 ** e, 0)
        got = cache.attend(0, q, n - s) * 2.0 ** -e
        if want is None:
            want = got
            check_attention(got, q, k, v, n - s, 0, "bf16")
        assert torch.equal(got, want), e
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("s", [1, 5, 200])
def test_queries_of_any_stride(s):
    """Tokens and batch rows on any multiple of 8 entries, one over another, and one for all."""
    ctx = ctx_for(32, 8, 128, "bf16")
    cache, k, v = filled(ctx, 2, 400, 3, "bf16")
    row = 32 * 128
    buf = queries(1, 2 * s + 2, 40, 128, "bf16", 4).reshape(-1)
    for tok, batch in ((row + 8, (row + 8) * s + 16), (row, row * s + 8), (row, 0), (0, row), (8, 24), (1032, 8)):
        q = buf.as_strided((2, s, 32, 128), (batch, tok, 128, 1))
        check_attention(cache.attend(0, q, 400 - s), q.clone(), k, v, 400 - s, 0, "bf16")
    ctx.close()


@pytest.mark.gpu
def test_calls_on_two_streams_and_the_context_in_turn():
    """Writes on one stream, attention on another, blocks on the context's own, without a wait of the host between them."""
    ctx = ctx_for(32, 8, 128, "f16")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    cache, k, v = filled(ctx, 1, 900, 3, "f16")
    q = queries(1, 300, 32, 128, "f16", 4)
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(a):
            for _ in range(3):
                cache.write(0, k, v if i % 2 else -v, 0)
        with torch.cuda.stream(b):
            got.append((cache.attend(0, q, 600), cache.attend(0, q[:, 299:], 899)))
        with torch.cuda.stream(ctx.torch_stream):
            got[-1] += (cache.attend(0, q, 600),)
    torch.cuda.synchronize()
    for i, (many, one, again) in enumerate(got):
        assert torch.equal(many, again) and torch.equal(many, got[i % 2][0]) and torch.equal(one, got[i % 2][1])
    check_attention(got[1][0], q, k, v, 600, 0, "f16")
    check_attention(got[1][1], q[:, 299:], k, v, 899, 0, "f16")
    check_attention(got[0][0], q, k, -v, 600, 0, "f16")
    ctx.close()


@pytest.mark.gpu
def test_the_attention_kernel_timed_over_a_batch():
    """cake_b200_bench_kernel times one token's attention: it has one row, whatever the cache's batch, and that row is the first batch row's."""
    cfg = medium_config(num_hidden_layers=2)
    ctx = Context(cfg, checkpoint(cfg, "bf16", std=0.05), "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    cache = Cache(ctx, 3, 100)
    cache.fill_synthetic([0, 1], 50)
    before = [cache.read(l, w).clone() for l in (0, 1) for w in (0, 1)]
    n, ms = len(m.blocks), c_float()
    hs, ix = (c_void_p * n)(*[b.h for b in m.blocks]), (c_int * n)(*range(n))
    check(lib().cake_b200_bench_kernel(ctx.h, hs, ix, n, cache.h, 4, 3, byref(ms)))
    assert 0 < ms.value < 10 and cache.len(0) == 50
    after = [cache.read(l, w) for l in (0, 1) for w in (0, 1)]
    for a, b in zip(after, before):
        assert torch.equal(a[1:], b[1:]) and torch.equal(a[0, :, :49], b[0, :, :49])
    ctx.close()
