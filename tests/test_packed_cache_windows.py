"""Caches in four bits: calls whose window leaves nothing, in every form that the launch takes."""
import pytest
import torch

from tests.test_packed_cache import check_attention, ctx_for, filled, queries


def attend_over_rubbish(cache, q, at, **kw):
    """The call's result lies where NaN lay before."""
    torch.cuda.synchronize()
    rubbish = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    del rubbish
    return cache.attend(0, q, at, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,b,n,s", [(1, 1, 64, 1 << 16, 1, 1),                       # more batch rows than a grid's third side has
                                               (32, 8, 128, 1, 1 << 15, 1 << 15),                 # more pieces of rows than its second one has
                                               (8, 2, 64, 2, 40, 1), (8, 2, 64, 1, 40, 20), (16, 8, 128, 3, 300, 200), (4, 2, 256, 1, 70, 30)])
def test_rows_that_see_nothing_are_zero(heads, kv, hd, b, n, s):
    ctx = ctx_for(heads, kv, hd, "bf16", max_seq=n)
    cache, k, v = filled(ctx, b, n, 3, "bf16")
    q = queries(1, s, heads, hd, "bf16", 4).expand(b, -1, -1, -1).contiguous()
    for first in (n, n + 1, 2 ** 31 - 1):
        assert not attend_over_rubbish(cache, q, n - s, first=first).any()
    got = attend_over_rubbish(cache, q, n - s, first=n - 1)     # the last row alone sees one position
    assert not got[:, :-1].any()
    # (not a read: the value is the sum of p step (n - 8) and p (lo + 8 step), so near zero a difference of numbers of the group's size, 2^-24 of them off)
    check_attention(got[:, -1:], q[:, -1:], k[:, n - 1:], v[:, n - 1:], 0, 0, "bf16")
    ctx.close()
