"""Caches in four bits: how many bits the attention over them keeps, for many rows (entries rounded to D, everything else finer) and for a few (codes)."""
import pytest
import torch

from cake_b200.model import Cache
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


def few_rows(q, kx, vx, at, first, dtype):
    """In 64 bits: the attention of q [b, s, heads, hd] over what rows kx, vx [b, n, kv, hd] stand for, and how far a call on codes may be from it.  With u = step |n - 8|
    of an entry, a row of `keys` keys rounds: the result, h; a weight times a step to one operand of fp16 (bf16: 2^-11 of p u) or to two (f16: 2^-22), or, where it has
    fp16's last bits, 2^-25 of the power of two that puts the largest step of the group which the row sees at 8 or more: 2^-25 / 8 of that step, times 8;
    the sums of u and of lo + 8 step, 230 * 2^-24 of V, the largest entry of the group that the row sees; scores: four products behind one another of at
    most 8 steps times the sum of |q|, 2^-22 each, eight additions of them of 2^-24 each, and 2^-20 of mag for lo + 8 step and the exponent; a weight changes by e^(2 ds)."""
    b, s, heads, hd = q.shape
    n, G, scale, h = kx.shape[1], heads // kx.shape[2], hd ** -0.5, HALF[dtype]

    def parts(x):   # values, step per entry
        x = x.double().cpu()
        g = x.unflatten(-1, (-1, 32))
        y = stands_for(x.to(kx.dtype)).double()
        want = (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) / 15
        step = want.to(kx.dtype)
        step = torch.where(step.double() < want, (step.view(torch.int16) + 1).view(kx.dtype), step).double().expand_as(g).flatten(-2)
        lo = g.amin(-1, keepdim=True).expand_as(g).flatten(-2)
        return [t.repeat_interleave(G, 2).transpose(1, 2) for t in (y, step, (y - lo - 8 * step).abs())]

    (k, ks, _), (v, vs, u) = parts(kx), parts(vx)
    q = q.double().cpu().transpose(1, 2)
    j, i = torch.arange(n)[None], torch.arange(at, at + s)[:, None]
    seen = (j >= first) & (j <= i)
    p = torch.softmax(torch.where(seen, q @ k.transpose(2, 3) * scale, -torch.inf), -1)
    ds = scale * (4 * 2.0 ** -22 * 8 + 8 * 2.0 ** -24 * 8) * q.abs() @ ks.transpose(2, 3) + scale * 2.0 ** -20 * q.abs() @ k.abs().transpose(2, 3)
    ds = torch.where(seen, ds, 0.0).amax(-1, keepdim=True)
    group = lambda t: t.unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(*t.shape[:-1], t.shape[-1] // 32, 32).flatten(-2)
    most = lambda t: torch.stack([group(t[:, :, first:at + r + 1].amax(2)) for r in range(s)], 2)   # of what row r sees
    keys = (i + 1 - first).double()
    ref, mass = p @ v, p @ v.abs()
    bound = 1.01 * h * ref.abs() + 1.01 * (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22) * (p @ u) + keys * 2.0 ** -25 * most(vs) + 2.0 ** -16 * most(v.abs()) + mass * torch.expm1(2 * ds) + 2.0 ** -25
    return ref.transpose(1, 2), bound.transpose(1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,s", [(4, 2, 128, 1), (8, 2, 64, 1), (8, 1, 128, 1), (4, 1, 128, 4), (4, 1, 64, 5), (2, 1, 256, 1), (2, 1, 256, 4), (1, 1, 128, 12), (2, 2, 64, 16), (8, 8, 128, 7)])
def test_groups_of_values_keep_their_bits_whatever_else_there_is(heads, kv, hd, s, dtype):
    """Values of one head whose groups differ in size by 2^30 (f16: 2^24, which is most of its range); positions whose values are far larger than those in
    front of them, which the rows in front do not see.  Keys of one value per group, so that scores are all but exact."""
    ctx = ctx_for(heads, kv, hd, dtype)
    D = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    for n in (s, 6 + s, 300):
        g = torch.Generator().manual_seed(n)
        k = (0.3 * torch.randn((1, n, kv, hd // 32, 1), generator=g)).expand(-1, -1, -1, -1, 32).flatten(-2).to(D).cuda()
        v = torch.randn((1, n, kv, hd), generator=g)
        q = queries(1, s, heads, hd, dtype, n)
        exps = torch.tensor([0, 30, 15, 3] * 2 if dtype == "bf16" else [-10, 13, 0, 7] * 2)[:hd // 32]
        sizes = v * torch.exp2(exps.double()).float().repeat_interleave(32)
        later = v * torch.exp2(torch.where(torch.arange(n) > n - s, 40.0 if dtype == "bf16" else 13.0, 0.0))[None, :, None, None] * (1.0 if dtype == "bf16" else 2.0 ** -8)
        rising = v * torch.exp2((torch.arange(n) - (n - s)).clamp(min=0) * (7.0 if dtype == "bf16" else 1.3))[None, :, None, None] * (1.0 if dtype == "bf16" else 2.0 ** -8)
        for x in (sizes, sizes.flip(3), later, later.flip(1), rising, rising.flip(1)):
            x = x.clamp(-60000, 60000).to(D).cuda() if dtype == "f16" else x.to(D).cuda()
            cache = Cache(ctx, 1, n, bits=4)
            cache.write(0, k, x, 0)
            ref, bound = few_rows(q, k, x, n - s, 0, dtype)
            err = (cache.attend(0, q, n - s).double().cpu() - ref).abs()
            assert (err <= bound).all(), (n, float((err / bound).max()))
            cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 2, 64), (4, 2, 256)])
def test_few_rows_keep_the_codes(heads, kv, hd, dtype):
    ctx = ctx_for(heads, kv, hd, dtype)
    for b, s, at, first in ((1, 1, 0, 0), (2, 1, 700, 0), (1, 3, 1500, 33), (2, 4, 9, 2)):
        cache, k, v = filled(ctx, b, at + s, at, dtype)
        q = queries(b, s, heads, hd, dtype, at + 1)
        ref, bound = few_rows(q, k, v, at, first, dtype)
        err = (cache.attend(0, q, at, first=first).double().cpu() - ref).abs()
        assert (err <= bound).all(), (at, float((err / bound).max()))
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,s,at", [(32, 8, 128, 1, 30), (8, 2, 64, 3, 100), (5, 5, 128, 5, 60), (4, 2, 256, 2, 400), (8, 1, 128, 4, 20)])
def test_few_rows_in_f16_are_off_by_the_result(heads, kv, hd, s, at):
    """All but the result keeps 20 bits and more (few_rows), so the distance to 64 bits is that of rounding the result once, up to 2^-8 of it for what falls to the other side."""
    ctx = ctx_for(heads, kv, hd, "f16")
    cache, k, v = filled(ctx, 4, at + s, at, "f16")
    q = queries(4, s, heads, hd, "f16", at + 1)
    ref, _ = few_rows(q, k, v, at, 0, "f16")
    rms = lambda t: float(t.square().mean().sqrt())
    own, err = rms(ref.half().double() - ref), rms(cache.attend(0, q, at).double().cpu() - ref)
    assert err <= (1 + 2.0 ** -8) * own, (err, own)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_row_of_many_and_the_row_alone(dtype):
    """The same row on entries rounded to D and on codes: each within its own bound of its own formula, and so near one another."""
    ctx = ctx_for(32, 8, 128, dtype)
    s, at = 180, 60
    cache, k, v = filled(ctx, 1, at + s, 8, dtype)
    q = queries(1, s, 32, 128, dtype, 9)
    many = cache.attend(0, q, at).double().cpu()
    for t in (0, 1, 63, 64, 179):
        one = q[:, t:t + 1]
        ref, bound = few_rows(one, k[:, :at + t + 1], v[:, :at + t + 1], at + t, 0, dtype)
        alone = cache.attend(0, one, at + t).double().cpu()
        assert ((alone - ref).abs() <= bound).all(), t
        # entries rounded to D: h |v| of each value, and e^(2 h mag) of a weight
        _, mass, mag, _ = attention(one.double().cpu(), rounded(k), rounded(v), at + t, 0, 128 ** -0.5)
        h = HALF[dtype]
        wide = 1.01 * h * ref.abs() + mass * (torch.expm1(2 * mag * (h + 2.0 ** -18)) + 1.01 * h + 2.0 ** -14) + 2.0 ** -25
        assert ((many[:, t:t + 1] - ref).abs() <= wide).all(), t
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,s", [(32, 8, 128, 1), (64, 8, 64, 1), (8, 4, 256, 1), (32, 4, 128, 1), (4, 4, 128, 3), (8, 8, 64, 12)])
def test_scores_whose_sums_cancel(heads, kv, hd, s, dtype):
    """Keys of one size and both signs against queries whose neighbours are alike: the codes' sums come to little, the scores to the steps' roundings.  Values of one number
    per group, so that nothing but scores and the result is rounded.  With S = scale times the sum of step |q|, a group's sum has four products behind one another
    and two additions, each off by 2^-24 of 8 times its share of S at most (n - 8 and 8 steps), rms 1 / sqrt 3 of that, half of it on the way: sqrt 6 / 2 / sqrt 3 * 8 * 2^-24
    S / sqrt groups < 1.5 * 2^-21 S / sqrt groups, and half of that where one of few keys' weights p moves by p (1 - p) <= 1 / 4 of it, to either side of |v|."""
    ctx = ctx_for(heads, kv, hd, dtype)
    D, b, n, groups = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype], 8, 2 + s, hd // 32
    g = torch.Generator().manual_seed(hd + s)
    size = 500 + 1000 * torch.rand((b, n, kv, 1), generator=g)
    k = (size * (1 - 2 * (torch.arange(hd) % 2))).to(D).cuda()
    q = torch.randn((b, s, heads, hd // 2, 1), generator=g).expand(-1, -1, -1, -1, 2).flatten(-2).to(D).cuda()
    v = torch.randn((b, n, kv, groups, 1), generator=g).expand(-1, -1, -1, -1, 32).flatten(-2).to(D).cuda()
    cache = Cache(ctx, b, n, bits=4)
    cache.write(0, k, v, 0)
    ref, _ = few_rows(q, k, v, n - s, 0, dtype)
    S = hd ** -0.5 * q.double().abs().sum(-1, keepdim=True).cpu() * (2 * float(size.max()) / 15 * (1 + 2 * HALF[dtype]))
    rms = lambda t: float(t.square().mean().sqrt())
    own = rms(ref.to(D).double() - ref)
    err = rms(cache.attend(0, q, n - s).double().cpu() - ref)
    assert err ** 2 <= 1.2 * own ** 2 + rms(float(v.abs().max()) * 0.75 * 2.0 ** -21 * S / groups ** 0.5) ** 2, (err, own)
    ctx.close()
