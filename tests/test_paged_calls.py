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
