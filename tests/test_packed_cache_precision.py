"""Caches in four bits: how many bits the attention over them keeps, for many rows (entries rounded to D, everything else finer) and for a few (codes)."""
import pytest
import torch

from tests.test_packed_cache import HALF, attention, ctx_for, filled, queries, stands_for


def rounded(x):
    """What rows x [b, n, kv, hd] stand for, rounded to D: the operands of a call of many rows."""
    return stands_for(x).to(x.dtype).double().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("b,s,at,first", [(1, 200, 0, 0), (2, 130, 40, 0), (1, 150, 2000, 700)])
def test_many_rows_round_entries_and_the_result_only(b, s, at, first, dtype):
    """Over entries rounded to D, a row of n keys differs from 64 bits by the result's rounding, h, and by
      weights in two D operands: h^2 of each, and 2^-25 of the largest where a small one has fp16's last bits (|v| <= big);
      scores: 8 products of 16 added one behind the other, 2^-22 each of at most mag: a weight changes by e^(2 ds), ds = mag 2^-19 + mag 2^-20 for the exponent;
      2^x to 2^-22; sums of weights, 64 a tile and then the tiles; sums of values, n / 8 additions of 2^-22 of at most the mass."""
    ctx = ctx_for(32, 8, 128, dtype)
    n, h = at + s, HALF[dtype]
    cache, k, v = filled(ctx, b, n, 3, dtype)
    q = queries(b, s, 32, 128, dtype, 4)
    ref, mass, mag, big = attention(q.double().cpu(), rounded(k), rounded(v), at, first, 128 ** -0.5)
    keys = (torch.arange(at, at + s) + 1 - first).double()[None, :, None, None]
    bound = 1.01 * h * ref.abs() + mass * (2 * h * h + torch.expm1(2 * mag * (2.0 ** -19 + 2.0 ** -20)) + 2.0 ** -21 + (64 + keys / 64) * 2.0 ** -23 + keys / 8 * 2.0 ** -22)
    bound = bound + keys * 2.0 ** -25 * big + 2.0 ** -25
    err = (cache.attend(0, q, at, first=first).double().cpu() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    ctx.close()
