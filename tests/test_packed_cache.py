"""Caches in four bits: rows written, read back and attended over, against the definition in 64 bits; refusals; the same cache under a block, a whole
generation and the decode graph."""
import os
import subprocess

import numpy as np
import pytest
import torch

from cake_b200.capi import CakeB200Error, check, lib, ptr
from cake_b200.config import Config
from cake_b200.model import B200Transformer, Cache, Context, Master, Sessions, TextModelBase
from cake_b200.synth import TORCH_DTYPES
from tests.util import checkpoint, medium_config

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ESTATE = -1, -4
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step of D, relative


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def stands_for(x):
    """What rows [..., hd] in D stand for."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    lo, span = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
    want = span / 15
    step = want.to(x.dtype)
    up = (step.view(torch.int16) + 1).view(x.dtype)
    step = torch.where(step.double() < want, up, step).double()
    if x.dtype is torch.bfloat16:
        step = torch.where(span > 0, step.clamp_min(2.0 ** -126), step)
    n = torch.floor((g - lo) / torch.where(step > 0, step, 1.0) + 0.5)
    y = torch.where(torch.isfinite(span.float()), lo + step * n, torch.nan)
    return y.reshape(x.shape)


def attention(q, k, v, at, first, scale):
    """q [b, s, heads, hd], k, v [b, n, kv, hd] in 64 bits -> (out, sum p |v|, largest sum |q||k| * scale of a row's seen keys, largest |v| of an
    entry's group that any row sees)."""
    b, s, heads, hd = q.shape
    n, G = k.shape[1], heads // k.shape[2]
    k, v = (t.repeat_interleave(G, 2).transpose(1, 2) for t in (k, v))
    q = q.transpose(1, 2)
    j, i = torch.arange(n)[None], torch.arange(at, at + s)[:, None]
    seen = (j >= first) & (j <= i)
    k, v = (torch.where((torch.arange(n) < at + s)[:, None], t, torch.zeros(())) for t in (k, v))   # what nobody sees, whatever it is
    sc = torch.where(seen, (q @ torch.nan_to_num(k, nan=0.0).transpose(2, 3)) * scale, -torch.inf)
    some = seen.any(1)
    p = torch.zeros_like(sc)
    p[:, :, some] = torch.softmax(sc[:, :, some], -1)
    mag = torch.where(seen, (q.abs() @ torch.nan_to_num(k, nan=0.0).abs().transpose(2, 3)) * scale, 0.0).amax(-1, keepdim=True)
    v = torch.nan_to_num(v, nan=0.0)
    big = torch.where(((torch.arange(n) >= first) & (torch.arange(n) < at + s))[:, None], v.abs(), 0.0).amax(2, keepdim=True)
    big = big.unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, -1, -1, 32).flatten(-2)
    return (p @ v).transpose(1, 2), (p @ v.abs()).transpose(1, 2), mag.transpose(1, 2), big.transpose(1, 2)


def check_attention(got, q, kx, vx, at, first, dtype, scale=None):
    """kx, vx: the rows written [b, n, kv, hd] in D.  Three things round: the held entries to D where a product takes them so (half a step each; of a
    score that is at most h mag, which changes a weight by e^(2 h mag)), a weight to D's half step or finer, and the result.  The sums are fp32.  Where
    a value is summed as p step (n - 8) and p (lo + 8 step), a sum that comes to nothing still has terms: with V the largest entry of the group, 8 step <= 1.08 V
    (the span is at most 2 V) and |lo + 8 step| <= 1.07 V + step / 2, 2.3 V together, over at most 100 additions one behind the other of 2^-24 each (16 in a
    product, one per block of a warp, the warps, the CTAs): 230 * 2^-24 V < 2^-16 V."""
    h = HALF[dtype]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ref, mass, mag, big = attention(q.double().cpu(), stands_for(kx).cpu(), stands_for(vx).cpu(), at, first, scale)
    got = got.double().cpu()
    ds = mag * (h + 2.0 ** -16) + 1e-5
    bound = 1.01 * h * ref.abs() + mass * (torch.expm1(2 * ds) + 2 * h + 1e-5) + 2.0 ** -16 * big + 2.0 ** -24
    assert torch.isfinite(got).all()
    err = (got - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # roundings are independent: their root mean square is h / sqrt 3 of what is rounded, for each of the four kinds at most
    rms = lambda t: float(t.square().mean().sqrt())
    assert rms(err) <= 2.4 * h * rms(ref) + 1e-6, (rms(err), rms(ref))


# ---------------------------------------------------------------------------------------------- inputs
def ctx_for(heads, kv, hd, dtype, max_seq=4096, **kw):
    return Context(Config(heads * hd, 64, 64, 2, heads, kv, head_dim=hd, max_seq_len=max_seq), {}, dtype, **kw)


def rows(b, n, kv, hd, dtype, seed, width=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((b, n, kv, hd), generator=g) * torch.exp(0.5 * torch.randn((kv, hd), generator=g)) + torch.randn((kv, hd), generator=g)
    return (x * width).to(TORCH_DTYPES[dtype]).cuda()


def queries(b, s, heads, hd, dtype, seed):
    return torch.randn((b, s, heads, hd), generator=torch.Generator().manual_seed(seed)).to(TORCH_DTYPES[dtype]).cuda()


def filled(ctx, b, n, seed, dtype, cap=None, block=0):
    c = ctx.config
    k, v = (rows(b, n, c.num_key_value_heads, c.hd, dtype, seed + i) for i in (0, 1))
    cache = Cache(ctx, b, cap or n, bits=4)
    cache.write(block, k, v, 0)
    return cache, k, v


def close_to_rows(got, x, dtype):
    """got [b, kv, n, hd] in D: what rows x [b, n, kv, hd] stand for, formed in fp32 and rounded to D once."""
    ref, got = stands_for(x).transpose(1, 2), got.double()
    nan = ref.isnan()
    assert torch.equal(nan, got.isnan())
    h, least = HALF[dtype], 2.0 ** -134 if dtype == "bf16" else 2.0 ** -25
    assert ((got - ref).abs()[~nan] <= ref.abs()[~nan] * (h + 2.0 ** -23) + least).all()


# ---------------------------------------------------------------------------------------------- the format (no GPU)
def test_every_word_of_a_block_has_its_own_place(tmp_path):
    src = tmp_path / "place.cpp"
    src.write_text(r'''
#include "packed_cache.cuh"
#include <cstdio>
#include <set>
using namespace cake::pc;
int main() {
  for (int hd : {64, 128, 256}) {
    std::set<int> k, v, p;
    for (int r = 0; r < BLOCK; r++) {
      for (int u = 0; u < hd / 8; u++) k.insert(k_word(hd, r, u));
      for (int g = 0; g < 8; g++)
        for (int j = 0; j < hd / 32; j++) v.insert(v_half(hd, r, g, j));
      for (int j = 0; j < hd / 32; j++) p.insert(pair_word(hd, r, j));
    }
    const int words = BLOCK * hd / 8;
    if ((int)k.size() != words || *k.begin() != 0 || *k.rbegin() != words - 1) return 1;
    if ((int)v.size() != 2 * words || *v.begin() != 0 || *v.rbegin() != 2 * words - 1) return 2;
    if ((int)p.size() != BLOCK * hd / 32 || *p.begin() != 0 || *p.rbegin() != BLOCK * hd / 32 - 1) return 6;
    const int codes = 4 * words, pairs = 4 * BLOCK * hd / GROUP;
    if (k_pairs(hd) != codes || v_codes(hd) != codes + pairs || v_pairs(hd) != 2 * codes + pairs || block_bytes(hd) != 2 * (codes + pairs)) return 3;
    if (block_bytes(hd) % 16) return 4;
  }
  for (int cap : {1, 15, 16, 63, 64, 65, 4096, 131072})
    if (cap_blocks(cap) * BLOCK < cap || cap_blocks(cap) % 4) return 5;
  return 0;
}
''')
    exe = tmp_path / "place"
    subprocess.check_call(["g++", "-std=c++17", "-x", "c++", str(src), "-I", os.path.join(ROOT, "cake_b200", "csrc"), "-I", "/usr/local/cuda/include", "-o", str(exe)])
    assert subprocess.call([str(exe)]) == 0


def test_definition_holds_what_it_says():
    """The oracle's own properties: within half a step, exact at the ends, groups of one value exact, no code beyond 15."""
    for dtype in ("bf16", "f16"):
        x = torch.randn((64, 128), generator=torch.Generator().manual_seed(3)).to(TORCH_DTYPES[dtype])
        x[0] = 2.5
        y = stands_for(x)
        g, r = x.double().reshape(64, 4, 32), y.reshape(64, 4, 32)
        step = (g.amax(-1) - g.amin(-1)) / 15 * (1 + 2 * HALF[dtype])
        assert ((r - g).abs().amax(-1) <= step / 2 + 1e-12).all()
        assert torch.equal(r.amin(-1), g.amin(-1)) and torch.equal(y[0], x[0].double())


# ---------------------------------------------------------------------------------------------- write and read
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (3, 3, 128), (16, 8, 128), (2, 1, 256)])
def test_rows_come_back_as_what_they_stand_for(heads, kv, hd, dtype):
    ctx = ctx_for(heads, kv, hd, dtype)
    for b, n in ((1, 1), (2, 17), (3, 64), (1, 333)):
        cache, k, v = filled(ctx, b, n, 7 + n, dtype, cap=n + 3)
        assert cache.len(0) == n and cache.len(1) == 0
        for which, x in ((0, k), (1, v)):
            close_to_rows(cache.read(0, which), x, dtype)
            lo, m = n // 3, n - n // 3 - n // 5
            close_to_rows(cache.read(0, which, lo, m), x[:, lo:lo + m], dtype)
        kh, vh = cache.kv(0)   # the host's view of the same
        assert torch.equal(kh, cache.read(0, 0).cpu()) and torch.equal(vh, cache.read(0, 1).cpu())
        cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_rows_of_every_kind(dtype):
    """Groups of one value, zeros, one outlier, both signs of zero, the type's extremes, subnormals, ties between codes, NaN and infinities."""
    ctx = ctx_for(2, 2, 64, dtype)
    D = TORCH_DTYPES[dtype]
    x = torch.randn((1, 20, 2, 64), generator=torch.Generator().manual_seed(1))
    x[0, 0], x[0, 1, 0], x[0, 1, 1] = 0.0, 3.25, -0.0
    x[0, 2, :, 5] = 1000.0
    x[0, 3, 0] *= 2.0 ** -24 if dtype == "f16" else 2.0 ** -130
    x[0, 3, 1] *= 2.0 ** -14 if dtype == "f16" else 2.0 ** -126
    x[0, 4, :, ::2], x[0, 4, :, 1::2] = torch.finfo(D).max / 2, -torch.finfo(D).max / 2
    x[0, 5] = torch.randint(0, 31, (2, 64), generator=torch.Generator().manual_seed(2)) / 2.0     # steps of one, every other value a tie
    x[0, 5, :, 0], x[0, 5, :, 1], x[0, 5, :, 32], x[0, 5, :, 33] = 0.0, 15.0, 0.0, 15.0
    x[0, 6, 0, 3], x[0, 7, 0, 40], x[0, 8, 1, 63] = torch.nan, torch.inf, -torch.inf
    x[0, 9, 0, :32] = torch.inf
    x[0, 10, 0, 2], x[0, 10, 0, 3] = torch.inf, -torch.inf
    x[0, 11] += 300.0
    for row, unit in ((13, 1.0), (14, 3.0), (15, 0.8125)):       # entries just below, on and above a tie: the ends are 7.5 steps from zero
        x[0, row, :, :32] = torch.tensor([-2.0, -1.0, 0.0, 1.0, 2.0, -4.0, 4.0, 8.0] * 4) * 2.0 ** -20 * unit
        x[0, row, :, 0], x[0, row, :, 1] = -7.5 * unit, 7.5 * unit
    x = x.to(D).cuda()
    if dtype == "bf16":
        x[0, 12, :, 0], x[0, 12, :, 1] = torch.finfo(D).max, -torch.finfo(D).max   # a span beyond fp32
    cache = Cache(ctx, 1, 20, bits=4)
    cache.write(0, x, x.flip(1), 0)
    close_to_rows(cache.read(0, 0), x, dtype)
    close_to_rows(cache.read(0, 1), x.flip(1), dtype)
    ctx.close()


@pytest.mark.gpu
def test_columns_of_a_projection_and_other_strides():
    ctx = ctx_for(4, 2, 128, "bf16")
    fused = rows(2, 50, 8, 128, "bf16", 5)
    cache = Cache(ctx, 2, 64, bits=4)
    for k, v in ((fused[:, :, 4:6], fused[:, :, 6:]),                       # as a block's projection holds them
                 (fused[:, ::2, 4:6], fused[:, 1::2, 6:]),                  # every other token
                 (fused[:1, :25, 4:6].expand(2, -1, -1, -1), fused[:, :25, 0:2]),   # one row for the whole batch
                 (fused.flip(1)[:, :25, 4:6], fused[:, :25, ::4]),          # heads apart: copied
                 (fused.reshape(-1)[4:4 + 2 * 25 * 256].view(2, 25, 2, 128), fused[:, 25:, :2])):   # off the 16-byte grid: copied
        cache.clear()
        cache.write(0, k, v, 0)
        close_to_rows(cache.read(0, 0), k, "bf16")
        close_to_rows(cache.read(0, 1), v, "bf16")
    ctx.close()


@pytest.mark.gpu
def test_rows_in_pieces_are_the_rows_at_once():
    ctx = ctx_for(4, 2, 128, "f16")
    n = 45
    cache, k, v = filled(ctx, 2, n, 11, "f16", cap=64)
    whole = [cache.read(0, w).clone() for w in (0, 1)]
    at = 0
    other = Cache(ctx, 2, 64, bits=4)
    for m in (1, 1, 14, 3, 16, 10):
        other.write(1, k[:, at:at + m], v[:, at:at + m], at)
        at += m
    assert at == n and all(torch.equal(other.read(1, w), whole[w]) for w in (0, 1))
    # from 20 on anew: what is in front stays, what was behind is gone
    k2, v2 = rows(2, 5, 2, 128, "f16", 91), rows(2, 5, 2, 128, "f16", 92)
    other.write(1, k2, v2, 20)
    assert other.len(1) == 25
    for w, x in ((0, k2), (1, v2)):
        got = other.read(1, w)
        assert torch.equal(got[:, :, :20], whole[w][:, :, :20])
        close_to_rows(got[:, :, 20:], x, "f16")
    new = other.as_new()
    assert new.bits == 4 and new.len(1) == 0
    ctx.close()


# ---------------------------------------------------------------------------------------------- attention
SHAPES = [(8, 2, 64), (5, 5, 128), (16, 8, 128), (32, 8, 128), (8, 1, 128), (4, 2, 256), (2, 2, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_one_token(heads, kv, hd, dtype):
    ctx = ctx_for(heads, kv, hd, dtype)
    for b, n in ((1, 1), (1, 2), (2, 15), (1, 16), (3, 17), (1, 63), (2, 64), (1, 65), (1, 127), (5, 129), (1, 1000), (2, 2049)):
        cache, k, v = filled(ctx, b, n, n, dtype, cap=n + 1)
        q = queries(b, 1, heads, hd, dtype, n + 9)
        check_attention(cache.attend(0, q, n - 1), q, k, v, n - 1, 0, dtype)
        for first in (n // 2, n - 1):
            check_attention(cache.attend(0, q, n - 1, first=first), q, k, v, n - 1, first, dtype)
        assert torch.equal(cache.attend(0, q, n - 1, first=n), torch.zeros_like(q))   # a row that sees nothing
        cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_several_rows(heads, kv, hd, dtype):
    ctx = ctx_for(heads, kv, hd, dtype)
    for b, s, at in ((1, 2, 0), (2, 3, 14), (1, 5, 60), (1, 8, 1000), (1, 17, 0), (1, 33, 31), (2, 70, 5), (1, 130, 0), (1, 131, 200), (1, 300, 77)):
        n = at + s
        cache, k, v = filled(ctx, b, n + 3, n, dtype, cap=n + 5)     # positions behind the rows are there already
        q = queries(b, s, heads, hd, dtype, n + 9)
        check_attention(cache.attend(0, q, at), q, k, v, at, 0, dtype)
        for first in {max(0, at - 7), at + s // 2}:                   # the second: the rows in front see nothing
            got = cache.attend(0, q, at, first=first)
            check_attention(got, q, k, v, at, first, dtype)
            assert not got[:, :max(0, first - at)].any()
        cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("s", [1, 4, 40, 150])
def test_what_no_row_sees_may_be_anything(hd, s):
    """NaN and infinities in front of `first`, behind the last row, and, for a row, behind that row: K or V, every place of a tile."""
    ctx = ctx_for(4, 2, hd, "bf16")
    at, first, n = 100, 37, 100 + s + 9
    k, v = rows(1, n, 2, hd, "bf16", 1), rows(1, n, 2, hd, "bf16", 2)
    k[:, :first], v[:, :first] = torch.nan, torch.inf
    k[:, at + s:], v[:, at + s:] = torch.inf, torch.nan
    cache = Cache(ctx, 1, n, bits=4)
    cache.write(0, k, v, 0)
    q = queries(1, s, 4, hd, "bf16", 3)
    check_attention(cache.attend(0, q, at, first=first), q, k, v, at, first, "bf16")
    if s > 1:   # the last row's own position: the rows in front of it are as before
        v[:, at + s - 1] = torch.nan
        k[:, at + s - 1] = torch.nan
        cache.write(0, k[:, at + s - 1:], v[:, at + s - 1:], at + s - 1)
        got = cache.attend(0, q, at, first=first)
        check_attention(got[:, :-1], q[:, :-1], k, v, at, first, "bf16")
        assert got[:, -1].isnan().all()
    # large finite rows there leave the seen ones their precision
    x = torch.full((1, n, 2, hd), 2.0 ** 100, dtype=torch.bfloat16, device="cuda") * torch.randn((1, n, 2, hd), device="cuda").bfloat16()
    k, v = rows(1, n, 2, hd, "bf16", 1), rows(1, n, 2, hd, "bf16", 2)
    for t in (k, v):
        t[:, :first], t[:, at + s:] = x[:, :first], x[:, at + s:]
    cache.write(0, k, v, 0)
    check_attention(cache.attend(0, q, at, first=first), q, k, v, at, first, "bf16")
    # seen NaN: the entries of V's group, or the whole row for K
    v[:, at - 1, 0, 3] = torch.nan
    cache.write(0, k[:, :at], v[:, :at], 0)
    cache.write(0, rows(1, s, 2, hd, "bf16", 8), rows(1, s, 2, hd, "bf16", 9), at)
    got = cache.attend(0, q, at, first=first)
    assert got[:, :, :2, :32].isnan().all() and torch.isfinite(got[:, :, :2, 32:]).all() and torch.isfinite(got[:, :, 2:]).all()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("b,s,at,first", [(1, 150, 100, 0), (1, 150, 100, 37), (1, 150, 2000, 1003), (2, 260, 0, 0), (1, 77, 3000, 16)])
def test_nan_in_a_prompt_reaches_the_rows_that_see_it(b, s, at, first, dtype):
    """Rows enough for keys and values to be expanded for the prompt's kernel, in one piece and with the keys cut: a NaN of K makes the rows from its
    position on NaN, one of V its group's entries of theirs; nothing else, whatever lies in front of `first` and behind the rows."""
    ctx = ctx_for(32, 8, 128, dtype)
    n = at + s + 5
    q = queries(b, s, 32, 128, dtype, 3)
    k0, v0 = rows(b, n, 8, 128, dtype, 1), rows(b, n, 8, 128, dtype, 2)
    k0[:, :first], v0[:, at + s:] = torch.inf, torch.nan
    cache = Cache(ctx, b, n, bits=4)
    for spots in ([], [("v", 0, 2, 70, at + s // 2)], [("k", 0, 0, 5, at + s - 1), ("v", b - 1, 7, 127, first)], [("v", 0, 3, 0, at + 16), ("v", 0, 3, 40, at + 31), ("k", 0, 4, 9, at + 47)]):
        k, v = k0.clone(), v0.clone()
        bad = torch.zeros((b, s, 32, 128), dtype=torch.bool)
        for which, bi, h, d, pos in spots:
            (k if which == "k" else v)[bi, pos, h, d] = torch.nan
            d0, d1 = (0, 128) if which == "k" else (d // 32 * 32, d // 32 * 32 + 32)
            bad[bi, max(0, pos - at):, 4 * h:4 * h + 4, d0:d1] = True
        cache.write(0, k, v, 0)
        got = cache.attend(0, q, at, first=first).cpu()
        assert torch.equal(got.isnan(), bad), spots
        if not spots:
            check_attention(got, q, k, v, at, first, dtype)
        clean = got if not spots else clean
        assert torch.equal(got[~bad], clean[~bad])
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_and_sizes_of_entries(dtype):
    """Sharp and flat softmaxes; values so small or large that weights times steps leave fp16; a step that grows by 2^12 on the way."""
    ctx = ctx_for(8, 2, 128, dtype)
    n, s = 700, 1
    k, v = rows(1, n, 2, 128, dtype, 1), rows(1, n, 2, 128, dtype, 2)
    q = queries(1, s, 8, 128, dtype, 3)
    cache = Cache(ctx, 1, n, bits=4)
    sizes = (1.0, 2.0 ** -9, 2.0 ** 9) if dtype == "f16" else (1.0, 2.0 ** -60, 2.0 ** 60)
    for size in sizes:
        for scale in (None, 1e-3, 1.0, 1e-30):
            w = v * size
            cache.write(0, k, w, 0)
            check_attention(cache.attend(0, q / 4 if scale == 1.0 else q, n - 1, scale=scale or 0.0) / size, q / 4 if scale == 1.0 else q, k, w / size, n - 1, 0, dtype, scale)
    grown = v * torch.where(torch.arange(n, device="cuda") >= n // 2, 1.0, 2.0 ** -12)[None, :, None, None].to(v.dtype)
    for t in (grown, grown.flip(1)):
        cache.write(0, k, t, 0)
        check_attention(cache.attend(0, q, n - 1), q, k, t.contiguous(), n - 1, 0, dtype)
    ctx.close()


@pytest.mark.gpu
def test_query_strides_and_repeats():
    ctx = ctx_for(4, 2, 128, "f16")
    cache, k, v = filled(ctx, 2, 90, 3, "f16")
    fused = queries(2, 120, 8, 128, "f16", 4)
    for s in (1, 6, 60):
        want = None
        for q in (fused[:, :s, :4].contiguous(), fused[:, :s, :4]):
            got = cache.attend(0, q, 90 - s)
            check_attention(got, q, k, v, 90 - s, 0, "f16")
            want = got if want is None else want
            assert torch.equal(got, want)                                   # the same call, the same bits
    q = fused[:, ::30, 4:]
    check_attention(cache.attend(0, q, 86), q, k, v, 86, 0, "f16")
    ctx.close()


@pytest.mark.gpu
def test_one_head_group_row_by_row_is_the_rows_at_once():
    """A prompt may be cut anywhere: row t of a long call is that row alone, up to the roundings of the two forms."""
    ctx = ctx_for(8, 2, 128, "f16")
    cache, k, v = filled(ctx, 1, 200, 21, "f16")
    q = queries(1, 200, 8, 128, "f16", 5)
    whole = cache.attend(0, q, 0)
    check_attention(whole, q, k, v, 0, 0, "f16")
    for t in (0, 1, 16, 63, 64, 150, 199):
        check_attention(cache.attend(0, q[:, t:t + 1], t), q[:, t:t + 1], k, v, t, 0, "f16")
    ctx.close()


@pytest.mark.gpu
def test_a_long_cache():
    """Offsets beyond 32 bits: the last rows of a cache of 4.5 GB."""
    ctx = ctx_for(8, 8, 256, "bf16", max_seq=1 << 16)
    b, n = 28, 1 << 16
    cache = Cache(ctx, b, n, bits=4)
    cache.fill_synthetic([0], 17)
    assert cache.len(0) == 17
    k, v = rows(b, 40, 8, 256, "bf16", 1), rows(b, 40, 8, 256, "bf16", 2)
    x = torch.zeros((b, 1, 8, 256), dtype=torch.bfloat16, device="cuda").expand(b, n - 40, 8, 256)
    cache.write(0, x, x, 0)
    cache.write(0, k, v, n - 40)
    got = cache.read(0, 0, n - 40)
    close_to_rows(got, k, "bf16")
    q = queries(b, 1, 8, 256, "bf16", 3)
    got = cache.attend(0, q, n - 1, first=n - 40)
    check_attention(got[-2:], q[-2:], k[-2:], v[-2:], 39, 0, "bf16")
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 128), (8, 1, 64), (2, 1, 256), (6, 2, 128), (5, 5, 64)])
def test_a_few_heads_over_many_positions(heads, kv, hd):
    """A head's keys are cut between many CTAs: more parts than shared memory holds at a time, and CTAs with parts of two heads.
    (Up to 157 parts are added one behind the other, 230 + 2.3 * 157 < 600 halves of 2^-23 V; the bound's mass * 2 h, mass > 0.5 here, is 2^-11, V < 5.)"""
    n = 20011
    ctx = ctx_for(heads, kv, hd, "f16", max_seq=n)
    cache, k, v = filled(ctx, 1, n, 5, "f16")
    for s, at, first in ((1, n - 1, 3), (2, 17003, 17), (5, 15001, 0)):
        q = queries(1, s, heads, hd, "f16", at)
        got = cache.attend(0, q, at, first=first)
        check_attention(got, q, k, v, at, first, "f16")
        assert torch.equal(cache.attend(0, q, at, first=first), got)
    v[:, 11000, 0, :32] = float("nan")          # one part's
    cache.write(0, k[:, 11000:], v[:, 11000:], 11000)     # (a write ends the cache behind its rows)
    q = queries(1, 1, heads, hd, "f16", 1)
    got = cache.attend(0, q, n - 1)
    assert got[..., :heads // kv, :32].isnan().all() and not got[..., :heads // kv, 32:].isnan().any() and not got[..., heads // kv:, :].isnan().any()
    ctx.close()


# ---------------------------------------------------------------------------------------------- streams and graphs
@pytest.mark.gpu
def test_rows_made_and_read_on_another_stream():
    ctx = ctx_for(8, 2, 128, "bf16")
    side = torch.cuda.Stream()
    cache = Cache(ctx, 1, 4096, bits=4)
    big = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    for stream in (side, ctx.torch_stream, torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            for _ in range(20):
                big = big @ big * 1e-4                        # the rows are not there yet when the call is made
            k, v, q = (rows(1, 500, h, 128, "bf16", i) + big[0, 0].to(torch.bfloat16) * 0 for i, h in ((1, 2), (2, 2), (3, 8)))
            q = q[:, 499:]
            cache.write(0, k, v, 0)
            out = cache.attend(0, q, 499)
            copy = out.clone()                               # behind the kernel on the caller's stream
        stream.synchronize()
        check_attention(copy, q, k, v, 499, 0, "bf16")
    ctx.close()


@pytest.mark.gpu
def test_captured_calls_share_a_context():
    """Two graphs of one context, replayed in turn and beside eager calls, with new rows in the captured buffers."""
    ctx = ctx_for(8, 2, 128, "bf16")
    caches, bufs, graphs, outs = [], [], [], []
    for i, s in enumerate((1, 40)):
        cache = Cache(ctx, 1, 2048, bits=4)
        n = 1500
        k, v = rows(1, n, 2, 128, "bf16", i), rows(1, n, 2, 128, "bf16", i + 5)
        q = queries(1, s, 8, 128, "bf16", i + 9)
        cache.write(0, k, v, 0)
        cache.attend(0, q, n - s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.write(0, k[:, n - s:], v[:, n - s:], n - s)
            outs.append(cache.attend(0, q, n - s))
        caches.append(cache); bufs.append((k, v, q, s)); graphs.append(g)
    for turn in range(3):
        for i, (k, v, q, s) in enumerate(bufs):
            q.copy_(queries(1, s, 8, 128, "bf16", 40 + turn + i))
            k[:, -s:], v[:, -s:] = rows(1, s, 2, 128, "bf16", 50 + turn), rows(1, s, 2, 128, "bf16", 60 + turn)
        for g in graphs + graphs[::-1]:
            g.replay()
        for i, (k, v, q, s) in enumerate(bufs):
            check_attention(outs[i], q, k, v, 1500 - s, 0, "bf16")
            check_attention(caches[i].attend(0, q, 1500 - s), q, k, v, 1500 - s, 0, "bf16")
    torch.cuda.synchronize()
    del graphs, g
    ctx.close()


@pytest.mark.gpu
def test_first_calls_inside_a_capture():
    """Memory that a call has to make cannot come in a capture: the call is refused, and the refusal leaves the capture usable."""
    ctx = ctx_for(32, 8, 128, "bf16")
    cache = Cache(ctx, 1, 600, bits=4)
    k, v = rows(1, 600, 8, 128, "bf16", 1), rows(1, 600, 8, 128, "bf16", 2)
    q = queries(1, 600, 32, 128, "bf16", 3)
    cache.write(1, k[:, :1], v[:, :1], 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(CakeB200Error) as e:
            cache.write(0, k, v, 0)
        assert e.value.code == ESTATE and cache.len(0) == 0
        cache.write(1, k, v, 0)
        one = cache.attend(1, q[:, 599:], 599)
        with pytest.raises(CakeB200Error) as e:
            cache.attend(1, q, 0)
        assert e.value.code == ESTATE
    g.replay()
    check_attention(one, q[:, 599:], k, v, 599, 0, "bf16")
    check_attention(cache.attend(1, q, 0), q, k, v, 0, 0, "bf16")
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        many = cache.attend(1, q, 0)
    q.copy_(queries(1, 600, 32, 128, "bf16", 4))
    g2.replay()
    check_attention(many, q, k, v, 0, 0, "bf16")
    torch.cuda.synchronize()
    del g, g2
    ctx.close()


@pytest.mark.gpu
def test_closed_caches_and_contexts():
    """A closed cache's memory is the next one's; caches may outlive their context; the calling thread keeps its device and stream."""
    ctx = ctx_for(8, 2, 128, "bf16")
    for i in range(6):
        cache, k, v = filled(ctx, 1 + i % 2, 700, i, "bf16")
        q = queries(1 + i % 2, 1, 8, 128, "bf16", i)
        check_attention(cache.attend(0, q, 699), q, k, v, 699, 0, "bf16")
        cache.close()
    left, k, v = filled(ctx, 1, 50, 9, "bf16")
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    h, left.h = left.h, None                     # the library's own order: the context first
    ctx._children = []
    ctx.sync()
    lib().cake_b200_ctx_destroy(ctx.h)
    lib().cake_b200_cache_free(h)
    ctx.h = None
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_decode_graph_asks_for_its_position_after_rows_were_written():
    cfg = medium_config(num_hidden_layers=1)
    ctx = Context(cfg, checkpoint(cfg, "bf16", std=0.05, peaked=True), "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    m.forward([[1, 2, 3, 4, 5, 6, 7, 8]], 0)
    m.index_pos = 8
    m.decode_build()
    m.decode_greedy(5, 2)
    k = rows(1, 3, 2, 64, "bf16", 1)
    ctx.cache.write(0, k, k, 6)
    with pytest.raises(CakeB200Error) as e:
        check(lib().cake_b200_decode_run(ctx.h, 1))
    assert e.value.code == ESTATE
    m.index_pos = 9
    assert len(m.decode_greedy(5, 2)) == 2 and ctx.cache.len(0) == 11
    ctx.close()


# ---------------------------------------------------------------------------------------------- refusals
@pytest.mark.gpu
def test_refusals():
    ctx = ctx_for(8, 2, 64, "bf16")
    k = rows(1, 4, 2, 64, "bf16", 1)
    q = queries(1, 4, 8, 64, "bf16", 2)

    def refused(code, call):
        with pytest.raises(CakeB200Error) as e:
            call()
        assert e.value.code == code, e.value

    for bits in (1, 2, 3, 5, 8, -4):
        refused(EINVAL, lambda: Cache(ctx, 1, 64, bits=bits))
    refused(EINVAL, lambda: Cache(ctx, 0, 64, bits=4))
    refused(EINVAL, lambda: Cache(ctx, 1, ctx.max_seq + 1, bits=4))
    plain, cache = Cache(ctx, 1, 64), Cache(ctx, 1, 6, bits=4)
    for c in (plain,):
        refused(EINVAL, lambda: c.write(0, k, k, 0))
        refused(EINVAL, lambda: c.attend(0, q, 0))
        refused(EINVAL, lambda: c.read(0, 0, 0, 1))
    refused(ESTATE, lambda: cache.attend(0, q, 0))       # nothing held
    refused(ESTATE, lambda: cache.read(0, 0, 0, 1))
    refused(ESTATE, lambda: cache.write(0, k, k, 1))     # a gap
    refused(EINVAL, lambda: cache.write(2, k, k, 0))     # no such block
    refused(EINVAL, lambda: cache.write(-1, k, k, 0))
    cache.write(0, k, k, 0)
    refused(ESTATE, lambda: cache.write(0, k, k, 4))     # beyond the capacity
    refused(ESTATE, lambda: cache.write(0, k, k, -1))
    refused(ESTATE, lambda: cache.attend(0, q, 1))
    refused(ESTATE, lambda: cache.attend(0, q, -1))
    refused(EINVAL, lambda: cache.attend(0, q, 0, first=-1))
    for scale in (-1.0, float("nan"), float("inf")):
        refused(EINVAL, lambda: cache.attend(0, q, 0, scale=scale))
    for w, first, n in ((0, 0, 5), (0, 4, 1), (1, -1, 2), (1, 0, 0), (0, 2, -1)):
        refused(ESTATE, lambda: cache.read(0, w, first, n))
    refused(EINVAL, lambda: cache.read(0, 2, 0, 1))
    refused(EINVAL, lambda: check(lib().cake_b200_cache_write(cache.h, 0, ptr(k) + 2, 128, 512, ptr(k), 128, 512, 1, 0, None)))
    refused(EINVAL, lambda: check(lib().cake_b200_cache_write(cache.h, 0, ptr(k), 127, 512, ptr(k), 128, 512, 1, 0, None)))
    refused(EINVAL, lambda: check(lib().cake_b200_cache_write(cache.h, 0, ptr(k), 128, 512, None, 128, 512, 1, 0, None)))
    refused(EINVAL, lambda: check(lib().cake_b200_cache_write(cache.h, 0, ptr(k), 128, 512, ptr(k), 128, 512, 0, 0, None)))
    refused(EINVAL, lambda: check(lib().cake_b200_cache_attend(cache.h, 0, ptr(q), 512, 2048, ptr(q) + 8, 1, 0, 0, 0.0, None)))
    for bad in (k.float(), k.cpu(), k[..., :32], k[:, :, :1], k[0], k.expand(2, -1, -1, -1)):
        with pytest.raises(ValueError):
            cache.write(0, bad, k, 0)
        with pytest.raises(ValueError):
            cache.write(0, k, bad, 0)
    with pytest.raises(ValueError):
        cache.attend(0, k, 0)
    assert cache.len(0) == 4                             # no refused call has moved it
    close_to_rows(cache.read(0, 1), k, "bf16")
    ctx.close()
    for cfg in (Config(128, 64, 64, 1, 4, 2, head_dim=32, max_seq_len=64), Config(256, 64, 64, 1, 4, 2, head_dim=64, max_seq_len=64, partial_rotary_factor=0.375)):
        other = Context(cfg, {}, "bf16")
        refused(EINVAL, lambda: Cache(other, 1, 64, bits=4))
        other.close()


# ---------------------------------------------------------------------------------------------- under blocks
def _model_pair(cfg, dtype, **kw):
    sd = checkpoint(cfg, dtype, std=0.05, peaked=True)
    return [(c, TextModelBase.load(c, **kw)) for c in (Context(cfg, sd, dtype), Context(cfg, sd, dtype, cache_bits=4))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cfg", [dict(), dict(head_dim=128, num_attention_heads=4, num_key_value_heads=2), dict(head_dim=256, num_attention_heads=4, num_key_value_heads=4),
                                 dict(head_dim=128, num_attention_heads=4, num_key_value_heads=1, use_qk_norm=True, partial_rotary_factor=0.75)])
def test_block_writes_the_rows_of_its_plain_cache(cfg, dtype):
    """The first block's rows are those that a cache in D holds, in four bits; a step's attention is that of the rows held (the block's other parts
    are those of the plain cache): seen through `attend` on the rotated queries of the same call."""
    cfg = medium_config(num_hidden_layers=1, **cfg)
    (pc, plain), (qc, packed) = _model_pair(cfg, dtype)
    x = (torch.randn((1, 40, cfg.hidden_size), generator=torch.Generator().manual_seed(2))).to(TORCH_DTYPES[dtype]).cuda()
    at = 0
    for s in (33, 1, 1, 5):
        for ctx, m in ((pc, plain), (qc, packed)):
            m.blocks[0].forward_batch(x[:, at:at + s], [(m.blocks[0].name, at, 0)], ctx, blocks=m.blocks)
            ctx.sync()
        at += s
    for which in (0, 1):
        want = pc.cache.kv(0)[which]                     # [1, kv, n, hd] in D
        got = qc.cache.read(0, which).cpu()
        ref = stands_for(want)
        # a key next to a rounding line of D may lie a step of D apart where the norm's sum has another order; its code then too
        same = (got.double() - ref).abs() <= ref.abs() * (HALF[dtype] + 2.0 ** -23) + 2.0 ** -25
        if not cfg.use_qk_norm:
            assert same.all()
        assert same.float().mean() > 0.99
    pc.close()
    qc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,heads,kv,window", [(64, 8, 2, None), (128, 4, 1, None), (64, 8, 2, 23), (128, 4, 2, 23)])
def test_block_output_is_that_of_the_rows_held(dtype, hd, heads, kv, window):
    """One block against its formula in 64 bits over the rows that the cache holds: prompt, portion and steps, with a sliding window too (the first call
    sees all it stores, a later one the last `window` positions at its end)."""
    cfg = medium_config(num_hidden_layers=1, head_dim=hd, num_attention_heads=heads, num_key_value_heads=kv, sliding_window=window)
    sd = checkpoint(cfg, dtype, std=0.05)
    ctx = Context(cfg, sd, dtype, cache_bits=4)
    m = TextModelBase.load(ctx)
    W = {n.split("layers.0.")[1]: t.double() for n, t in sd.items() if "layers.0." in n}
    g = torch.Generator().manual_seed(3)
    x = torch.randn((1, 61, cfg.hidden_size), generator=g).to(TORCH_DTYPES[dtype])
    r = lambda t: t.to(TORCH_DTYPES[dtype]).double()
    rms = lambda t, w: r(t / torch.sqrt(t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * w)
    at = 0
    for s in (50, 1, 9, 1):
        xs = x[:, at:at + s]
        y = m.blocks[0].forward_batch(xs.cuda(), [(m.blocks[0].name, at, 0)], ctx, blocks=m.blocks)
        ctx.sync()
        xd = xs.double()
        h = rms(xd, W["input_layernorm.weight"])
        q = r(h @ W["self_attn.q_proj.weight"].T).view(1, s, heads, hd)
        f = cfg.rope_theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        ang = torch.arange(at, at + s, dtype=torch.float64)[:, None] * f
        c, sn = r(ang.cos())[:, None], r(ang.sin())[:, None]
        q = torch.cat([r(r(q[..., :hd // 2] * c) - r(q[..., hd // 2:] * sn)), r(r(q[..., hd // 2:] * c) + r(q[..., :hd // 2] * sn))], -1)
        k, v = (t.double().transpose(1, 2) for t in ctx.cache.kv(0))
        att = r(attention(q, k, v, at, max(0, at + s - window) if window and at else 0, hd ** -0.5)[0].reshape(1, s, -1))
        x1 = r(r(att @ W["self_attn.o_proj.weight"].T) + xd)
        h2 = rms(x1, W["post_attention_layernorm.weight"])
        gate, up = r(h2 @ W["mlp.gate_proj.weight"].T), r(h2 @ W["mlp.up_proj.weight"].T)
        out = r(r(r(gate * torch.sigmoid(gate)) * up) @ W["mlp.down_proj.weight"].T) + x1
        err = (y.double().cpu() - out).abs()
        top = float(out.abs().max())
        # a rounding on the way that falls to the other side is a whole step of D at the size of the sums; three sums of the stream follow one another
        assert float(err.max()) <= 4 * 2 * HALF[dtype] * 2.0 ** np.floor(np.log2(top)), (s, float(err.max()), top)
        at += s
    if window:
        with pytest.raises(CakeB200Error) as e:   # a portion longer than the window, on a cache that is not empty
            m.blocks[0].forward_batch(x[:, :window + 1].cuda(), [(m.blocks[0].name, at, 0)], ctx, blocks=m.blocks)
        assert e.value.code == EINVAL
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_generation_steps_and_graph_agree(dtype):
    """The prompt and then token by token; prompt cut in two; the decode graph: the same tokens (logits of random weights stand apart)."""
    cfg = medium_config(num_hidden_layers=2)
    sd = checkpoint(cfg, dtype, std=0.05, peaked=True)
    ctx = Context(cfg, sd, dtype, cache_bits=4)
    m = TextModelBase.load(ctx)
    prompt = np.random.default_rng(1).integers(0, cfg.vocab_size, 37).tolist()
    want = Master(m).generate_text(prompt, 12)["tokens"]
    assert ctx.cache.bits == 4 and ctx.cache.len(0) == 37 + len(want) - 1
    ctx.cache.clear()
    m.forward([prompt[:20]], 0)
    lg = m.forward([prompt[20:]], 20)
    ctx.sync()
    first = int(lg.float().argmax())
    m.index_pos = 37
    m.decode_build()
    got = [first] + m.decode_greedy(first, len(want) - 1)
    assert got == want
    assert ctx.cache.len(0) == 37 + len(want) - 1 and ctx.cache.len(1) == ctx.cache.len(0)
    s = Sessions(m)
    assert s.cache_of("a").bits == 4
    ctx.close()


@pytest.mark.gpu
def test_graph_and_steps_agree_where_capacity_is_large():
    """The graph cuts keys as the capacity asks, steps as the length does."""
    cfg = medium_config(num_hidden_layers=2, max_seq_len=40000, head_dim=128, num_attention_heads=4, num_key_value_heads=2)
    ctx = Context(cfg, checkpoint(cfg, "bf16", std=0.05, peaked=True), "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    for n in (5, 130, 1500):
        ids = np.random.default_rng(n).integers(0, cfg.vocab_size, n).tolist()
        want = Master(m).generate_text(ids, 8)["tokens"]
        ctx.cache.clear()
        logits = m.forward([ids], 0)
        ctx.sync()
        first = int(logits.float().argmax())
        m.index_pos = n
        m.decode_build()
        assert [first] + m.decode_greedy(first, len(want) - 1) == want
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["olmo2", "gemma3", "exaone4"])
def test_sibling_blocks(kind):
    """Per layer: norms, rotation or none and the layer's window are those of the plain cache.  Rows as there, in four bits; what lies in front of a local
    layer's window changes nothing, of a global layer's something."""
    from tests.test_gpu_parity import SIBLINGS
    cfg = medium_config(num_hidden_layers=4, **SIBLINGS[kind])
    (pc, plain), (qc, packed) = _model_pair(cfg, "bf16")
    xs = [torch.randn((1, 14, cfg.hidden_size), generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in (1, 2)]
    xs[1][:, 4:] = xs[0][:, 4:]                          # the first four tokens differ
    for layer in range(4):
        last = []
        for x in xs:
            for ctx, m in ((pc, plain), (qc, packed)):
                ctx.cache.clear()
                for at, n in ((0, 4), (4, 3), (7, 1), (8, 1), (9, 4), (13, 1)):
                    y = m.blocks[layer].forward(x[:, at:at + n], at, layer, ctx)
                ctx.sync()
            last.append(y.clone())
            for which in (0, 1):
                got, ref = qc.cache.read(layer, which).cpu().double(), stands_for(pc.cache.kv(layer)[which])
                assert ((got - ref).abs() <= ref.abs() * (HALF["bf16"] + 2.0 ** -23) + 2.0 ** -25).float().mean() > 0.99
        local = bool(cfg.sliding_window) and not cfg.global_layers[layer]
        assert torch.equal(last[0], last[1]) == local, layer
    pc.close(), qc.close()


@pytest.mark.gpu
def test_batch_rows_are_their_own():
    cfg = medium_config(num_hidden_layers=2)
    sd = checkpoint(cfg, "bf16", std=0.05, peaked=True)
    ctx = Context(cfg, sd, "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    ids = np.random.default_rng(2).integers(0, cfg.vocab_size, (3, 30))
    alone = []
    for r in range(3):
        ctx.cache.clear()
        m.forward([ids[r, :25].tolist()], 0)
        alone.append([])
        for i, t in enumerate(ids[r, 25:]):
            lg = m.forward([[int(t)]], 25 + i)
            ctx.sync()
            alone[-1].append(lg.float()[0].cpu())
    ctx.cache = Cache(ctx, 3, 64)
    assert ctx.cache.bits == 4
    m.forward(ids[:, :25], 0)
    for i in range(5):
        lg = m.forward(ids[:, 25 + i:26 + i], 25 + i)
        ctx.sync()
        lg = lg.float().cpu()
        for r in range(3):
            assert torch.nn.functional.cosine_similarity(lg[r], alone[r][i], dim=0) > 0.999
    ctx.close()


def test_command_lines_name_the_choice():
    from cake_b200 import run, worker
    for main in (run.main, worker.main):
        with pytest.raises(SystemExit):
            main(["x", "--cache-bits", "3"])


@pytest.mark.gpu
def test_compiled_host_gives_the_same_tokens(tmp_path):
    from tests.test_cpp_host import RUN, _write_model
    from cake_b200.build import build
    build()
    cfg = medium_config(num_hidden_layers=2)
    sd = checkpoint(cfg, "bf16", std=0.05, peaked=True)
    _write_model(tmp_path, cfg, sd)
    prompt = np.random.default_rng(5).integers(0, cfg.vocab_size - 1, 21).tolist()
    out = [subprocess.run([RUN, str(tmp_path), "--prompt-ids", ",".join(map(str, prompt)), "-n", "10", "--cache-bits", bits], capture_output=True, text=True,
                          timeout=120) for bits in ("4", "3")]
    assert out[0].returncode == 0, out[0].stderr
    assert out[1].returncode == 1 and "4 bits" in out[1].stderr
    ctx = Context(cfg, sd, "bf16", cache_bits=4)
    assert [int(t) for t in out[0].stdout.splitlines()[0].split(":")[1].split()] == Master(TextModelBase.load(ctx)).generate_text(prompt, 10)["tokens"]
    ctx.close()
