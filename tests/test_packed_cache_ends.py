"""Caches in four bits: entries at the ends of the type, and what they do to rows that see them and rows that do not."""
import pytest
import torch

from cake_b200.model import Cache
from cake_b200.synth import TORCH_DTYPES
from tests.test_packed_cache import HALF, check_attention, ctx_for, filled, queries, rows, stands_for


def at_the_end(b, n, kv, hd, D, seed):
    """Groups that reach D's largest number from zero and from anywhere, its neighbours, both signs."""
    most = torch.finfo(D).max
    x = torch.rand((b, n, kv, hd), generator=torch.Generator().manual_seed(seed)) * most / 4
    x[..., ::32] = most
    x[..., 1::64] = 0.0
    x[:, 1::3, :, ::32] = most * (1 - torch.finfo(D).eps / 2)
    x[:, 2::3] = -x[:, 2::3]
    return x.to(D).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_entries_at_the_end_stay_numbers(hd, dtype):
    ctx = ctx_for(2, 2, hd, dtype)
    x = at_the_end(2, 50, 2, hd, TORCH_DTYPES[dtype], hd)
    most = torch.finfo(x.dtype).max
    cache = Cache(ctx, 2, 50, bits=4)
    cache.write(0, x, x.flip(1), 0)
    for which, y in ((0, x), (1, x.flip(1))):
        got, ref = cache.read(0, which).double(), stands_for(y).transpose(1, 2).clamp(max=most)
        assert torch.isfinite(got).all()
        assert ((got - ref).abs() <= ref.abs() * (HALF[dtype] + 2.0 ** -23)).all()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("s", [1, 3, 150])
def test_a_row_over_entries_at_the_end(s, dtype):
    """One position, so the result is the value: on codes, and expanded.  The value's rounding, h, and the result's.  On codes a weight p is 1 to 2^-22 (2^x, its argument's
    rounding), p step rounds to step itself, and (step (n - 8) + p (lo + 8 step)) / p has 2^-22 of step |n - 8| <= V and three roundings of 2^-24 of at most 2 V:
    2^-20 V, V = D's largest number, where a value near zero is the difference of large ones."""
    ctx = ctx_for(32, 8, 128, dtype)
    x = at_the_end(1, s, 8, 128, TORCH_DTYPES[dtype], s)
    most = torch.finfo(x.dtype).max
    cache = Cache(ctx, 1, s, bits=4)
    cache.write(0, rows(1, s, 8, 128, dtype, 1), x, 0)
    got = cache.attend(0, queries(1, s, 32, 128, dtype, 2), 0)[:, 0].double().cpu()
    ref = stands_for(x[:, 0]).cpu().clamp(max=most).repeat_interleave(4, 1)
    assert ((got - ref).abs() <= 2.02 * HALF[dtype] * ref.abs() + 2.0 ** -20 * most).all()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("s,at", [(150, 0), (200, 900), (5, 30)])
def test_rows_do_not_see_what_lies_behind_them(s, at, dtype):
    """Positions at the type's end come after the others: the rows in front of them are, to the bit, what they are without them (or on codes, where the
    order of sums is the same too)."""
    ctx = ctx_for(32, 8, 128, dtype)
    n, late = at + s, 3 if s == 5 else 40
    cache, k, v = filled(ctx, 1, n, 4, dtype)
    q = queries(1, s, 32, 128, dtype, 5)
    clean = cache.attend(0, q, at)
    check_attention(clean, q, k, v, at, 0, dtype)
    x = at_the_end(1, late, 8, 128, TORCH_DTYPES[dtype], 6)
    cache.write(0, k[:, n - late:], x, n - late)
    got = cache.attend(0, q, at)
    assert torch.equal(got[:, :s - late], clean[:, :s - late])
    if dtype == "f16":
        assert torch.isfinite(got).all()
    cache.write(0, x, v[:, n - late:], n - late)
    got = cache.attend(0, q, at)
    assert torch.equal(got[:, :s - late], clean[:, :s - late])
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,s,n", [(4, 2, 128, 1, 10), (4, 2, 128, 1, 700), (4, 2, 128, 1, 20000), (8, 2, 64, 3, 100), (8, 1, 128, 3, 40), (4, 2, 256, 1, 3000), (32, 8, 128, 150, 400)])
def test_nan_reaches_a_row_through_any_weight(heads, kv, hd, s, n, dtype):
    """A key whose score is 700 below the others': its weight is no number of fp32, but a value that is NaN still is one that the rows see."""
    ctx = ctx_for(heads, kv, hd, dtype, max_seq=n)
    k, v = torch.zeros((1, n, kv, hd)), rows(1, n, kv, hd, dtype, 2)
    at = n - s
    q = torch.ones((1, s, heads, hd)).to(TORCH_DTYPES[dtype]).cuda()
    for far in {0, at // 2, at - 1, at}:
        kf, vf = k.clone(), v.clone()
        kf[:, far] = -700.0 * hd ** -0.5
        kf = kf.to(v.dtype).cuda()
        cache = Cache(ctx, 1, n, bits=4)
        cache.write(0, kf, vf, 0)
        clean = cache.attend(0, q, at)
        assert torch.isfinite(clean).all()
        vf[:, far, 0, 40] = torch.nan
        cache.write(0, kf, vf, 0)
        got = cache.attend(0, q, at)
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[:, :, :heads // kv, 32:64] = True
        assert torch.equal(got.isnan(), bad), far
        assert torch.equal(got[~bad], clean[~bad])
        cache.close()
    ctx.close()
