"""Caches in pages: rows appended with their rotation, attention over pages of sequences of many lengths, against plain arithmetic in 64 bits."""
import math
import os
import random
import subprocess

import pytest
import torch

from cake_b200.capi import CakeB200Error, byref, c_void_p, lib
from cake_b200.config import Config
from cake_b200.model import Context, PagedCache
from cake_b200.synth import TORCH_DTYPES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ESTATE, ENOMEM = -1, -4, -5
HALF_ULP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # of a rounding to D, relative
LEAST = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24}    # D's smallest number


def ctx_for(heads, kv, hd, dtype, layers=1, **kw):
    return Context(Config(heads * hd, 64, 256, layers, heads, kv, head_dim=hd, max_seq_len=kw.pop("max_seq_len", 1 << 16), rope_theta=500000.0, **kw), {}, dtype)


def normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(TORCH_DTYPES[dtype])


def tables(n, rot, theta=500000.0):
    f = theta ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") / (rot // 2))
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float(), a.sin().float()


class Talks:
    """Sequences of a cache and what their pages should hold, position by position."""

    def __init__(self, cache, kv, hd, dtype):
        self.cache, self.kv, self.hd, self.dtype, self.k, self.v = cache, kv, hd, dtype, {}, {}
        self.empty = torch.empty(0, kv, hd, dtype=TORCH_DTYPES[dtype], device="cuda")

    def add(self):
        s = self.cache.add()
        self.k[s] = self.v[s] = self.empty
        return s

    def step(self, ids, counts, seed=1, k=None, v=None, block=0):
        """New rows as they are."""
        n = sum(counts)
        k = normal((n, self.kv, self.hd), self.dtype, 2 * seed) if k is None else k
        v = normal((n, self.kv, self.hd), self.dtype, 2 * seed + 1) if v is None else v
        self.cache.step(ids, counts)
        assert self.cache.append(block, None, k, v, rotate=False) is None
        for s, a, b in zip(ids, k.split(counts), v.split(counts)):
            self.k[s], self.v[s] = torch.cat([self.k[s], a]), torch.cat([self.v[s], b])

    def check(self, q, ids, counts, window=0, scale=0.0, out=None, block=0):
        got = self.cache.attend(block, q, window=window, scale=scale) if out is None else out
        assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
        for s, g, x in zip(ids, got.split(counts), q.split(counts)):
            check_rows(g, x, self.k[s], self.v[s], window, scale, self.dtype)
        return got


def check_rows(got, q, k, v, window, scale, dtype):
    """got, q [rows, heads, hd] of a sequence's last rows; k, v [positions, kv, hd].  What the bound counts, for a weighted mean of values with A = sum p |v|: one
    rounding of the result (half an ulp); weights as two operands of 8 bits or more (2^-16 A); a score's sum of hd products in fp32, at most hd / 2 + 8
    roundings of 2^-24 of sum |q k| in any order of pairs or chains of accumulators, twice for numerator and denominator; exponentials to 2^-21; sums over
    n positions in chains of 64 or more in parallel, (n / 64 + 80) roundings of 2^-24."""
    rows, heads, hd = q.shape
    n, kv = k.shape[0], k.shape[1]
    sc = scale or hd ** -0.5
    i, j = torch.arange(n - rows, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (j <= i) & (j > i - (window or n + 1))
    for h in range(heads):
        kd, vd, qd = k[:, h * kv // heads].double(), v[:, h * kv // heads].double(), q[:, h].double()
        s = torch.where(seen, qd @ torch.nan_to_num(kd.T) * sc, -math.inf)
        p = torch.softmax(s, -1)
        want, A = p @ torch.nan_to_num(vd, 0, 0, 0), p @ torch.nan_to_num(vd, 0, 0, 0).abs()
        size = torch.where(seen, qd.abs() @ torch.nan_to_num(kd.T, 0, 0, 0).abs() * sc, 0).amax(-1, keepdim=True)
        tol = HALF_ULP[dtype] * want.abs() * 1.001 + A * (2.0 ** -16 + 2 * size * (hd / 2 + 8) * 2.0 ** -24 + 2.0 ** -20 + (n / 64 + 80) * 2.0 ** -24) + LEAST[dtype]
        far = (got[:, h].double() - want).abs() - tol
        assert far.max() <= 0, (h, float(far.max()), float((got[:, h].double() - want).abs().max()))


# ------------------------------------------------------------------------------------------------ the book of pages, without a GPU
BOOK = r'''
#include "paged_plan.hpp"
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
using namespace cake::pg;
#define IS(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
static unsigned rnd_state = 7;
static int rnd(int n) { rnd_state = rnd_state * 1664525u + 1013904223u; return (int)((rnd_state >> 8) % (unsigned)n); }
static int bad;
int first_of(const SeqRow &s, const Window &w, int tok) {   // what token tok sees first, from the definition
  if (w.w <= 0) return 0;
  if (w.by_call) return s.pos0 == 0 ? 0 : std::max(0, s.pos0 + s.count - w.w);
  return std::max(0, s.pos0 + tok - w.w + 1);
}
int main() {
  {  // refusals leave everything as it was
    Book b;
    b.init(4, 16, 3, 40);
    int s0 = b.add(), s1 = b.add(), s2 = b.add();
    IS(s0 == 0 && s1 == 1 && s2 == 2 && b.add() == -1);
    int w[3] = {s0, s1, 7}, c[3] = {5, 5, 5};
    IS(b.plan(w, c, 3, 4, &bad) == Book::NOT_LIVE && bad == 2);
    w[2] = -1;
    IS(b.plan(w, c, 3, 4, &bad) == Book::NOT_LIVE);
    w[2] = s0;
    IS(b.plan(w, c, 3, 4, &bad) == Book::TWICE && bad == 2);
    c[1] = 0;
    IS(b.plan(w, c, 2, 4, &bad) == Book::COUNT && bad == 1);
    c[1] = -3;
    IS(b.plan(w, c, 2, 4, &bad) == Book::COUNT);
    c[1] = 41;
    IS(b.plan(w, c, 2, 4, &bad) == Book::TOO_LONG && bad == 1);
    c[1] = 2147483647;
    IS(b.plan(w, c, 2, 4, &bad) == Book::TOO_LONG);
    c[0] = 40; c[1] = 17;   // 3 + 2 pages of 4
    IS(b.plan(w, c, 2, 4, &bad) == Book::NO_PAGES);
    IS(b.free_pages.size() == 4 && b.seqs[0].len == 0 && b.step.empty() && b.n_rows == 0);
    c[0] = 33; c[1] = 16;
    IS(b.plan(w, c, 2, 4, &bad) == Book::OK && b.free_pages.empty() && b.n_rows == 49 && b.updates.size() == 8);
    const uint64_t shape = b.shape;
    c[0] = 7; c[1] = 1;     // seven fit their pages, one does not
    IS(b.plan(w, c, 2, 4, &bad) == Book::NO_PAGES && b.shape == shape && b.seqs[0].len == 33 && b.step.size() == 2);
    IS(b.plan(w, c, 1, 4, &bad) == Book::OK && b.seqs[0].len == 40 && b.updates.empty());
    b.cut(0, 32);           // ends the step
    IS(b.step.empty() && b.free_pages.size() == 1 && b.seqs[0].pages.size() == 2);
    b.drop(1);
    IS(b.free_pages.size() == 2 && !b.has(1) && b.add() == 1 && b.seqs[1].len == 0);
  }
  for (int round = 0; round < 400; round++) {   // any steps: pages belong to one sequence each, and the cuts cover every tile once
    const int page = 16 << rnd(4), G = 1 + rnd(20), n_kv = 1 + rnd(8), seqs = 1 + rnd(12);
    Book b;
    b.init(3 + rnd(400), page, seqs, 1 + rnd(6000));
    std::vector<int> ids;
    std::map<int, int> table;
    for (int step = 0; step < 12; step++) {
      while ((int)ids.size() < seqs && rnd(3)) ids.push_back(b.add());
      if (ids.empty()) continue;
      std::vector<int> w, c;
      for (int s : ids) if (rnd(4)) { w.push_back(s); c.push_back(1 + (rnd(3) ? rnd(3) : rnd(300))); }
      if (w.empty()) continue;
      std::vector<int> before;
      for (int s : w) before.push_back(b.seqs[s].len);
      if (b.plan(w.data(), c.data(), (int)w.size(), G, &bad) == Book::OK) {
        for (size_t i = 0; i < b.updates.size(); i += 2) table[b.updates[i]] = b.updates[i + 1];
        std::set<int> used(b.free_pages.begin(), b.free_pages.end());
        size_t n = b.free_pages.size();
        for (int s : ids) {
          n += b.seqs[s].pages.size();
          IS((int)b.seqs[s].pages.size() == (b.seqs[s].len + page - 1) / page);
          for (size_t i = 0; i < b.seqs[s].pages.size(); i++) {
            used.insert(b.seqs[s].pages[i]);
            IS(table[s * b.per_seq + (int)i] == b.seqs[s].pages[i] && (int)i < b.per_seq);
          }
        }
        IS((int)n == b.n_pages && (int)used.size() == b.n_pages);
        IS(b.step.size() == w.size());
        std::set<int> rows;
        for (const SeqRow &s : b.step) {
          int i = 0;
          while (w[i] != s.slot) i++;
          int row0 = 0;
          for (int k = 0; k < i; k++) row0 += c[k];
          IS(s.pos0 == before[i] && s.count == c[i] && s.row0 == row0 && b.seqs[s.slot].len == s.pos0 + s.count);
        }
        for (int i = 0; i < (int)b.step.size(); i++) IS((b.step[i].count * G <= TOKEN_COLS) == (i < b.n_few));
        for (int k = 0; k < 3; k++) {
          const Window win{k ? 1 + rnd(500) : 0, k == 2};
          bool none = false;   // (a call whose rows exceed its window is refused in front of this)
          for (const SeqRow &s : b.step) none = none || (win.by_call && s.pos0 > 0 && s.count > win.w);
          if (none) continue;
          std::vector<Worker> ws;
          std::vector<Cut> cuts;
          const int most = 1 + rnd(300);
          int total = 0;
          for (int s = 0; s < b.n_few; s++) total += tiles_of(b.step[s], win) * n_kv;
          b.cut_few(win, n_kv, most, &ws, &cuts);
          IS((int)ws.size() <= most && (ws.empty() == (b.n_few == 0)));
          int i = 0, h = 0, t = 0, sum = 0;   // the workers follow one another through (sequence, key head, tile)
          std::vector<std::vector<int>> pieces;   // of the runs, in whose shares
          for (size_t j = 0; j < ws.size(); j++) {
            const Worker &x = ws[j];
            IS(x.i == i && x.kvh == h && x.tile == t && x.left >= 1 && x.s.slot == b.step[i].slot && x.s.pos0 == b.step[i].pos0);
            bool fresh = true;
            for (int y = 0; y < x.left; y++) {
              if (t == 0) pieces.push_back({});
              if (t == 0 || fresh) pieces.back().push_back((int)j);
              fresh = false;
              sum++;
              if (++t == tiles_of(b.step[i], win)) { t = 0; fresh = true; if (++h == n_kv) { h = 0; i++; } }
            }
          }
          size_t cut = 0;
          for (size_t y = 0; y < pieces.size(); y++) {
            const std::vector<int> &p = pieces[y];
            for (size_t z = 0; z < p.size(); z++) IS(p[z] == p[0] + (int)z);
            if (p.size() == 1) continue;
            IS(cut < cuts.size());
            const Cut &x = cuts[cut++];
            IS(x.kvh == (int)y % n_kv && x.s.slot == b.step[y / n_kv].slot && x.first == p[0] && x.parts == (int)p.size());
          }
          IS(cut == cuts.size() && (int)cut <= most);
          IS(sum == total && i == b.n_few && h == 0 && t == 0);
          for (int s = 0; s < b.n_few; s++) {
            IS(tile_first(b.step[s], win) * TILE <= first_of(b.step[s], win, 0) && tiles_of(b.step[s], win) >= 1);
            IS((tile_first(b.step[s], win) + 1) * TILE > first_of(b.step[s], win, 0));
          }
          std::vector<Item> it;
          const int room = 1 + rnd(80), parts = b.cut_many(win, G, room, &it), tpt = TILE_ROWS / G;
          std::map<std::pair<int, int>, std::vector<Item>> of;
          for (const Item &x : it) of[{x.i, x.tok0}].push_back(x);
          size_t whole = 0;
          std::set<int> places;
          for (int s = b.n_few; s < (int)b.step.size(); s++)
            for (int tok = 0; tok < b.step[s].count; tok += tpt, whole++) {
              const std::vector<Item> &v = of[{s, tok}];
              IS(!v.empty() && (int)v.size() == v[0].parts);
              IS(v[0].t0 == first_of(b.step[s], win, tok) / TILE);
              IS(v.back().t1 == (b.step[s].pos0 + std::min(tok + tpt, b.step[s].count) - 1) / TILE + 1);
              for (size_t x = 0; x < v.size(); x++) {
                IS(v[x].part == (int)x && v[x].t1 > v[x].t0 && (x == 0 || v[x].t0 == v[x - 1].t1) && v[x].tile == v[0].tile);
                if (v[x].parts > 1) IS(v[x].part0 == v[0].part0 && places.insert(v[x].part0 + v[x].part).second && v[x].part0 + v[x].part < parts);
              }
            }
          IS(of.size() == whole && (int)places.size() == parts);
          IS(it.size() <= whole + 2 * (size_t)room && it.size() <= Book::most_items(b.n_rows, seqs, G, room));
          IS(parts <= 2 * room && (whole > (size_t)room || it.size() <= (size_t)room));
        }
      }
      if (!rnd(3)) {
        const int at = rnd((int)ids.size()), s = ids[at];
        if (rnd(2)) { b.drop(s); ids.erase(ids.begin() + at); }
        else b.cut(s, rnd(b.seqs[s].len + 1));
      }
    }
  }
  return 0;
}
'''


def test_pages_and_cuts_of_any_steps(tmp_path):
    src = tmp_path / "book.cpp"
    src.write_text(BOOK)
    exe = tmp_path / "book"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-Wall", "-x", "c++", str(src), "-I", os.path.join(ROOT, "cake_b200", "csrc"), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ appending
def rotated(x, cos, sin, at):
    """[rows, heads, hd] at positions at, in 64 bits, and what the roundings in 32 bits may add."""
    half = cos.shape[1]
    x, c, s = x.double(), cos[at].double()[:, None], sin[at].double()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    want = torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), torch.zeros_like(x[..., 2 * half:])], -1)
    return want, size * 2.0 ** -22


def close_to(got, want, slack, dtype):
    assert ((got.double() - want).abs() <= HALF_ULP[dtype] * want.abs() * 1.001 + slack + LEAST[dtype] / 2).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,rot,page,dtype", [
    (32, 8, 128, 128, 64, "bf16"), (16, 8, 128, 128, 16, "f16"), (8, 2, 64, 64, 32, "bf16"), (8, 2, 64, 32, 16, "f16"), (8, 4, 256, 256, 128, "bf16"),
    (8, 4, 256, 64, 1024, "f16"), (5, 5, 128, 16, 16, "bf16"), (7, 1, 64, 48, 32, "f16"), (3, 1, 256, 16, 16, "bf16"), (12, 3, 128, 96, 16, "bf16")])
def test_append(heads, kv, hd, rot, page, dtype):
    ctx = ctx_for(heads, kv, hd, dtype)
    steps = [([0, 1, 2], [1, 40, 17]), ([0, 1, 2], [1, 1, 1]), ([2, 0], [200, 15]), ([1], [1]), ([1, 2, 0], [300, 2, 1])]
    cos, sin = tables(600, rot)
    cache = PagedCache(ctx, 3 * (600 // page + 1), page, max_seqs=3, max_seq=600, rotation=(cos, sin))
    for _ in range(3):
        cache.add()
    held, want_k, want_v = [0, 0, 0], [[], [], []], [[], [], []]
    for n, (ids, counts) in enumerate(steps):
        rows = sum(counts)
        fused = normal((rows, heads + 2 * kv, hd), dtype, n)
        q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
        if n == 2:   # rows of their own, a copy that is needed
            k = k.contiguous().transpose(0, 1).contiguous().transpose(0, 1)
            v = torch.cat([v.reshape(-1)[:3], v.reshape(-1)])[3:].view(rows, kv, hd)
        at = torch.cat([torch.arange(held[s], held[s] + c, device="cuda") for s, c in zip(ids, counts)])
        cache.step(ids, counts)
        kept = fused.clone()
        got_q = cache.append(0, q, k, v)
        assert torch.equal(kept, fused)
        got_k, got_v = cache.read(0)
        close_to(got_q, *rotated(q, cos, sin, at), dtype)
        close_to(got_k, *rotated(k, cos, sin, at), dtype)
        assert torch.equal(got_v, v)
        for s, c, a, b in zip(ids, counts, got_k.split(counts), got_v.split(counts)):
            held[s] += c
            want_k[s].append(a)
            want_v[s].append(b)
            assert cache.len(s) == held[s]
    for s in range(3):   # what was written before stays as it was
        k, v = cache.read(0, s)
        assert torch.equal(k, torch.cat(want_k[s])) and torch.equal(v, torch.cat(want_v[s]))
        k, v = cache.read(0, s, 7, 11)
        assert torch.equal(k, torch.cat(want_k[s])[7:18]) and torch.equal(v, torch.cat(want_v[s])[7:18])
    ctx.close()


@pytest.mark.gpu
def test_the_contexts_own_tables():
    """Without tables of its own a cache rotates by the model's: held in D, as the reference has them."""
    ctx, rot = ctx_for(8, 2, 64, "bf16", partial_rotary_factor=0.5), 32
    f = torch.tensor(500000.0) ** -(torch.arange(rot // 2, dtype=torch.float32) * 2 / rot)
    a = torch.arange(50, dtype=torch.float32)[:, None] * f
    cache = PagedCache(ctx, 8, 16, max_seqs=2, max_seq=50)
    s = cache.add()
    x = normal((50, 10, 64), "bf16", 3)
    cache.step([s], [50])
    q = cache.append(0, x[:, :8], x[:, 8:9].repeat(1, 2, 1), x[:, 8:])
    want, slack = rotated(x[:, :8], a.cos().cuda(), a.sin().cuda(), torch.arange(50, device="cuda"))
    size = x[:, :8].double().abs().amax(-1, keepdim=True) * 2 * 2.0 ** -8   # tables of 8 bits
    close_to(q, want, slack + size, "bf16")
    ctx.close()


@pytest.mark.gpu
def test_append_without_rotation_or_queries():
    ctx = ctx_for(8, 2, 128, "f16")
    cache = PagedCache(ctx, 40, 16, max_seqs=2)
    t = Talks(cache, 2, 128, "f16")
    a, b = t.add(), t.add()
    t.step([b, a], [33, 5], seed=1)
    q = normal((38, 8, 128), "f16", 9)
    assert torch.equal(cache.append(0, q, torch.cat([t.k[b], t.k[a]]), torch.cat([t.v[b], t.v[a]]), rotate=False), q)
    for s in (a, b):
        k, v = cache.read(0, s)
        assert torch.equal(k, t.k[s]) and torch.equal(v, t.v[s])
    ctx.close()


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [(32, 8, 128), (16, 8, 128), (8, 2, 64), (8, 4, 256), (6, 6, 64), (5, 1, 128), (8, 1, 64), (7, 1, 128), (3, 3, 256), (24, 8, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page,dtype", [(16, "bf16"), (64, "f16"), (256, "bf16")])
def test_tokens_of_many_lengths(heads, kv, hd, page, dtype):
    """One token each at lengths around the pages' and the tiles' ends."""
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 200, 255, 256, 257, 700, 1501]
    ctx = ctx_for(heads, kv, hd, dtype)
    cache = PagedCache(ctx, sum(-(-n // page) for n in lengths), page, max_seqs=len(lengths), max_seq=1501)
    t = Talks(cache, kv, hd, dtype)
    ids = [t.add() for _ in lengths]
    order = random.Random(5).sample(range(1, len(ids)), len(ids) - 1)
    t.step([ids[i] for i in order], [lengths[i] - 1 for i in order], 1)
    t.step(ids, [1] * len(ids), 2)
    assert cache.available == 0
    q = normal((len(ids), heads, hd), dtype, 3)
    out = t.check(q, ids, [1] * len(ids))
    assert torch.equal(out, cache.attend(0, q))   # the same every time
    for window in (1, 16, 64, 100):
        t.check(q, ids, [1] * len(ids), window=window)
    t.check(q, ids, [1] * len(ids), scale=0.31)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page,dtype", [(16, "f16"), (64, "bf16"), (128, "f16")])
def test_rows_of_every_number(heads, kv, hd, page, dtype):
    """Steps that mix one token, a few and many, on nothing, a little and more."""
    talk = [(0, 1), (0, 2), (0, 63), (0, 64), (0, 65), (0, 200), (1, 1), (1, 3), (5, 16), (61, 4), (63, 2), (64, 128), (100, 33), (300, 1), (511, 130), (640, 5)]
    ctx = ctx_for(heads, kv, hd, dtype)
    cache = PagedCache(ctx, sum(-(-(h + r) // page) for h, r in talk), page, max_seqs=len(talk), max_seq=800)
    t = Talks(cache, kv, hd, dtype)
    ids = [t.add() for _ in talk]
    some = [i for i, (h, _) in enumerate(talk) if h]
    t.step([ids[i] for i in some], [talk[i][0] for i in some], 1)
    order = random.Random(7).sample(range(len(ids)), len(ids))
    who, counts = [ids[i] for i in order], [talk[i][1] for i in order]
    t.step(who, counts, 2)
    q = normal((sum(counts), heads, hd), dtype, 3)
    out = t.check(q, who, counts)
    assert torch.equal(out, cache.attend(0, q))
    for window in (1, 50, 64, 129):
        t.check(q, who, counts, window=window)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,rows,held,window", [
    (32, 8, 128, 1, 40000, 0), (8, 2, 64, 1, 65534, 0), (8, 4, 256, 2, 20000, 7000), (16, 8, 128, 40, 30000, 0), (8, 2, 64, 3, 30000, 20001), (8, 4, 256, 70, 9000, 0)])
def test_long_sequences(heads, kv, hd, rows, held, window):
    """A few rows on many keys: the keys are cut over the chip, and the sums joined."""
    ctx = ctx_for(heads, kv, hd, "bf16")
    cache = PagedCache(ctx, -(-(held + rows) // 64) + 1, 64, max_seqs=2, max_seq=held + rows)
    t = Talks(cache, kv, hd, "bf16")
    a, b = t.add(), t.add()
    t.step([a], [held], 1)
    t.step([b, a], [1, rows], 2)
    q = normal((1 + rows, heads, hd), "bf16", 3)
    out = t.check(q, [b, a], [1, rows], window=window)
    for _ in range(3):
        assert torch.equal(out, cache.attend(0, q, window=window))
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,rows", [(32, 8, 128, 1), (8, 2, 64, 2), (8, 4, 256, 1), (32, 8, 128, 150), (8, 2, 64, 300), (8, 4, 256, 140)])
def test_scores_that_lie_far_apart(heads, kv, hd, rows):
    """Keys whose scores rise, fall and jump by far more than an exponential's range, and values of two sizes."""
    ctx = ctx_for(heads, kv, hd, "bf16")
    n = 700
    for kind in range(4):
        cache = PagedCache(ctx, n // 16 + 1, 16, max_seqs=1, max_seq=n)
        t = Talks(cache, kv, hd, "bf16")
        s = t.add()
        k, v = normal((n, kv, hd), "bf16", kind), normal((n, kv, hd), "bf16", 9)
        j = torch.arange(n, device="cuda").float()
        lift = [j / 8, -j / 8, (j % 97 == 96).float() * 60, torch.where(j > 400, -1e4, 0.0)][kind]
        k[..., 0] = lift[:, None].to(k.dtype)
        v = (v.float() * torch.where(j % 2 == 0, 1.0, 64.0)[:, None, None]).to(v.dtype)
        t.step([s], [n - rows], k=k[:n - rows], v=v[:n - rows])
        t.step([s], [rows], k=k[n - rows:], v=v[n - rows:])
        q = normal((rows, heads, hd), "bf16", 4)
        q[..., 0] = 8
        t.check(q, [s], [rows])
        cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_weights_far_below_the_largest(rows, dtype):
    """One position with nearly all the weight and 60000 with 2^-25 of it each, whose values are larger: together they are a good part of the result."""
    ctx = ctx_for(8, 2, 64, dtype)
    n = 60000
    cache = PagedCache(ctx, n // 64 + 2, 64, max_seqs=1, max_seq=n + rows)
    t = Talks(cache, 2, 64, dtype)
    s = t.add()
    k, v = torch.zeros(n + rows, 2, 64, device="cuda", dtype=TORCH_DTYPES[dtype]), normal((n + rows, 2, 64), dtype, 1) + 4
    k[123, :, 0], v[123] = 25 * math.log(2), 0.125
    t.step([s], [n], k=k[:n], v=v[:n])
    t.step([s], [rows], k=k[n:], v=v[n:])
    q = torch.zeros(rows, 8, 64, device="cuda", dtype=TORCH_DTYPES[dtype])
    q[:, :, 0] = 8
    t.check(q, [s], [rows])
    ctx.close()


@pytest.mark.gpu
def test_more_windows_than_plans():
    """Windows in any order, more of them than the cache keeps plans for, one captured; other windows after eight captured ones are refused."""
    ctx = ctx_for(8, 2, 128, "bf16")
    cache = PagedCache(ctx, 60, 16, max_seqs=3, max_seq=400)
    t = Talks(cache, 2, 128, "bf16")
    ids = [t.add() for _ in range(3)]
    counts = [1, 30, 2]
    t.step(ids, [100, 250, 7], 1)
    t.step(ids, counts, 2)
    q = normal((33, 8, 128), "bf16", 3)
    rng = random.Random(2)
    cache.attend(0, q, window=77)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cache.attend(0, q, window=77)
    for turn in range(3):
        for w in rng.sample(range(1, 300), 14):
            t.check(q, ids, counts, window=w)
        t.step(ids, counts, 10 + turn)
        q.copy_(normal((33, 8, 128), "bf16", 20 + turn))
        g.replay()
        t.check(q, ids, counts, window=77, out=out)
    for w in range(1, 8):
        cache.attend(0, q, window=w)
        torch.cuda.synchronize()
        h = torch.cuda.CUDAGraph()
        with torch.cuda.graph(h):
            cache.attend(0, q, window=w)
        del h
    t.check(q, ids, counts, window=5)
    with pytest.raises(CakeB200Error) as e:
        cache.attend(0, q, window=300)
    assert e.value.code == EINVAL
    del g
    ctx.close()


BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 2, 64), (8, 4, 256)])
@pytest.mark.parametrize("rows", [1, 3, 150])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_what_a_row_does_not_see_counts_for_nothing(heads, kv, hd, rows, dtype):
    """Infinities and NaN in pages of a former owner, behind a sequence's last row, in front of a window and in later rows of the step itself."""
    ctx = ctx_for(heads, kv, hd, dtype)
    cache = PagedCache(ctx, 60, 16, max_seqs=3, max_seq=960)
    t = Talks(cache, kv, hd, dtype)
    gone = t.add()
    dirt = torch.tensor(BAD, device="cuda")[torch.arange(960 * kv * hd, device="cuda") % 3].view(960, kv, hd).to(TORCH_DTYPES[dtype])
    t.step([gone], [960], k=dirt, v=dirt)
    cache.drop(gone)
    a, b = t.add(), t.add()
    n = 330
    k, v = normal((n + rows, kv, hd), dtype, 1), normal((n + rows, kv, hd), dtype, 2)
    t.step([b, a], [7, n], k=torch.cat([k[:7], k[:n]]), v=torch.cat([v[:7], v[:n]]))
    t.step([a, b], [rows, rows], k=torch.cat([k[n:], k[:rows]]), v=torch.cat([v[n:], v[:rows]]))
    q = normal((2 * rows, heads, hd), dtype, 3)
    t.check(q, [a, b], [rows, rows])
    want = cache.attend(0, q, window=90)[:rows]
    cache.truncate(a, 0)
    k[:n - 100], v[:n - 100] = dirt[:n - 100], dirt[:n - 100]
    cache.step([a], [n])
    cache.append(0, None, k[:n], v[:n], rotate=False)
    cache.step([a], [rows])
    cache.append(0, None, k[n:], v[n:], rotate=False)
    got = cache.attend(0, q[:rows], window=90)
    assert torch.isfinite(got).all()
    t.k[a], t.v[a] = k, v
    check_rows(got, q[:rows], k[n - 99:], v[n - 99:], 90, 0.0, dtype)
    if rows > 1:   # later rows of the step
        for first in (1, rows // 2, rows - 1):
            k2, v2 = k.clone(), v.clone()
            k2[n + first:], v2[n + first:] = dirt[:rows - first], dirt[:rows - first]
            cache.append(0, None, k2[n:], v2[n:], rotate=False)
            got = cache.attend(0, q[:rows], window=90)
            assert torch.isfinite(got[:first]).all() and torch.isnan(got[first:]).all()
            check_rows(got[:first], q[:first], k[n - 99:n + first], v[n - 99:n + first], 90, 0.0, dtype)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 2, 64), (8, 4, 256)])
@pytest.mark.parametrize("rows", [1, 2, 140])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_infinite_values_that_a_row_sees(heads, kv, hd, rows, dtype):
    """One entry of one position: an infinity stays one in that entry of the rows that see it, a NaN makes NaN, two infinities of both signs NaN."""
    ctx = ctx_for(heads, kv, hd, dtype)
    cache = PagedCache(ctx, 40, 32, max_seqs=1, max_seq=900)
    t = Talks(cache, kv, hd, dtype)
    s = t.add()
    n = 250
    k, v, q = normal((n, kv, hd), dtype, 1) * 0.1, normal((n, kv, hd), dtype, 2), normal((rows, heads, hd), dtype, 3)
    clean = v.clone()
    at = [70, n - rows, n - 1]
    for p, d, x in ((at[0], 3, float("inf")), (at[1], 5, -float("inf")), (at[1], hd - 1, float("nan")), (at[2], 3, -float("inf"))):
        v[p, :, d] = x
    t.step([s], [n - rows], k=k[:n - rows], v=v[:n - rows])
    t.step([s], [rows], k=k[n - rows:], v=v[n - rows:])
    got = cache.attend(0, q).double()
    want = torch.zeros(rows, hd, device="cuda", dtype=torch.float64)
    for i in range(rows):
        seen = v[:n - rows + i + 1, 0].double()
        want[i] = torch.where(torch.isfinite(seen), 0.0, seen).sum(0)   # (+inf, -inf, NaN or 0)
    for h in range(heads):
        odd = ~torch.isfinite(want)
        assert torch.equal(torch.nan_to_num(got[:, h][odd], 7, 8, 9), torch.nan_to_num(want[odd], 7, 8, 9)), h
        assert torch.isfinite(got[:, h][~odd]).all()
    other = torch.isfinite(v.double()).all(0).all(0)
    check_rows(torch.where(other, got, 0).to(q.dtype), q, k, torch.where(other, clean, 0), 0, 0.0, dtype)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 200])
def test_strides_streams_and_other_rows(rows):
    """Rows of any stride, one for all, calls on another stream than the cache's first; what belongs to others stays as it is."""
    ctx = ctx_for(32, 8, 128, "bf16")
    cache = PagedCache(ctx, 200, 16, max_seqs=3, max_seq=1000)
    t = Talks(cache, 8, 128, "bf16")
    a, b, c = t.add(), t.add(), t.add()
    t.step([a, b, c], [300, 77, 16], 1)
    held = {s: cache.read(0, s) for s in (b, c)}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        t.step([a], [rows], 2)
        buf = normal((rows, 48, 128), "bf16", 3)
        first = cache.attend(0, buf[:, 4:36])
    t.check(buf[:, 4:36], [a], [rows])
    torch.cuda.synchronize()
    assert torch.equal(first, cache.attend(0, buf[:, 4:36].contiguous()))
    assert torch.equal(cache.attend(0, buf[:1, 4:36].expand(rows, 32, 128))[-1:], cache.attend(0, buf[:1, 4:36].repeat(rows, 1, 1))[-1:])
    flat = normal((40 + rows * 8 + 32 * 128,), "bf16", 5)
    over = flat.as_strided((rows, 32, 128), (8, 128, 1), 8)   # rows over one another
    t.check(over.clone(), [a], [rows], out=cache.attend(0, over))
    for s in (b, c):
        assert all(torch.equal(x, y) for x, y in zip(cache.read(0, s), held[s]))
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 100])
def test_pools_beyond_32_bits(rows):
    """Pages whose bytes lie behind 2^32."""
    ctx = ctx_for(32, 8, 128, "bf16", max_seq_len=1 << 22)
    pages = 18000   # of 262144 bytes each
    cache = PagedCache(ctx, pages, 64, max_seqs=3, max_seq=64 * 17500)
    t = Talks(cache, 8, 128, "bf16")
    hog, a = cache.add(), t.add()
    t.step([a], [100], 1)
    cache.step([hog], [64 * 17400])   # takes its pages, writes none
    t.step([a], [800], 2)
    t.step([a], [rows], 3)
    assert cache.available < 600 and 17400 * 262144 > 1 << 32
    q = normal((rows, 32, 128), "bf16", 4)
    t.check(q, [a], [rows])
    k, v = cache.read(0, a)
    assert torch.equal(k, t.k[a]) and torch.equal(v, t.v[a])
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("max_seq", [2500, 65000])   # (what a run can have at most decides how a captured call is cut)
@pytest.mark.parametrize("heads,kv,hd,counts", [(32, 8, 128, [1, 1, 1]), (8, 2, 64, [2, 1, 3]), (16, 8, 128, [1, 90, 1])])
def test_captured_and_replayed(heads, kv, hd, counts, max_seq):
    """A step's calls captured once, replayed for steps of other sequences and lengths; a step of other counts is refused."""
    ctx = ctx_for(heads, kv, hd, "bf16")
    cache = PagedCache(ctx, 400, 16, max_seqs=5, max_seq=max_seq)
    t = Talks(cache, kv, hd, "bf16")
    ids = [t.add() for _ in range(5)]
    t.step(ids, [40, 700, 3, 64, 1500], 1)
    n = sum(counts)
    q, k, v = (normal((n, x, hd), "bf16", 2 + i) for i, x in enumerate((heads, kv, kv)))
    cache.step(ids[:3], counts)
    torch.cuda.synchronize()
    with pytest.raises(CakeB200Error) as e:   # nothing like it has run outside a capture for attention yet: what it needs is not there
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.step(ids[:3], counts)
    assert e.value.code == ESTATE
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache.append(0, None, k, v, rotate=False)
        for w in (0, 200):
            cache.attend(0, q, window=w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append(0, None, k, v, rotate=False)
        outs = [cache.attend(0, q, window=w) for w in (0, 200)]
        rk, rv = cache.read(0)
    for s, x, y in zip(ids, k.split(counts), v.split(counts)):
        t.k[s], t.v[s] = torch.cat([t.k[s], x]), torch.cat([t.v[s], y])
    for i, who in enumerate(([0, 1, 2], [4, 2, 3], [1, 4, 0], [2, 3, 4])):
        who = [ids[j] for j in who]
        for j, x in enumerate((q, k, v)):
            x.copy_(normal(x.shape, "bf16", 50 + 10 * i + j))
        cache.step(who, counts)
        g.replay()
        for s, x, y in zip(who, k.split(counts), v.split(counts)):
            t.k[s], t.v[s] = torch.cat([t.k[s], x]), torch.cat([t.v[s], y])
        assert torch.equal(rk, k) and torch.equal(rv, v)
        for w, out in zip((0, 200), outs):
            t.check(q, who, counts, window=w, out=out)   # (the call itself may cut its keys by these lengths, and so sum in another order)
            t.check(q, who, counts, window=w)
    before = [o.clone() for o in outs]
    cache.step(ids[:2], [1, 1])
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(CakeB200Error) as e:
        cache.read(0)
    assert e.value.code == ESTATE and "replayed" in str(e.value)
    assert all(torch.equal(x, y) for x, y in zip(before, outs))
    kk, vv = cache.read(0, ids[0], 0, t.k[ids[0]].shape[0])
    assert torch.equal(kk, t.k[ids[0]]) and torch.equal(vv, t.v[ids[0]])
    del g
    ctx.close()


@pytest.mark.gpu
def test_two_caches_and_two_blocks():
    """Caches of one context, and blocks of one cache, keep apart; sequences come and go."""
    ctx = ctx_for(8, 2, 128, "f16", layers=2)
    talks = [Talks(PagedCache(ctx, 40, 16, max_seqs=4, max_seq=300), 2, 128, "f16") for _ in range(2)]
    ids = [[t.add() for _ in range(3)] for t in talks]
    rng = random.Random(3)
    other = [{s: t.empty for s in x} for t, x in zip(talks, ids)]
    for turn in range(30):
        i = turn % 2
        t, who = talks[i], ids[i]
        pick = rng.sample(who, rng.randint(1, 3))
        counts = [rng.choice([1, 1, 2, 20]) for _ in pick]
        t.step(pick, counts, 100 + turn)
        k1 = normal((sum(counts), 2, 128), "f16", 500 + turn)
        t.cache.append(1, None, k1, -k1, rotate=False)
        for s, x in zip(pick, k1.split(counts)):
            other[i][s] = torch.cat([other[i][s], x])
        q = normal((sum(counts), 8, 128), "f16", 900 + turn)
        t.check(q, pick, counts)
        got = t.cache.attend(1, q)
        for s, g, x in zip(pick, got.split(counts), q.split(counts)):
            check_rows(g, x, other[i][s], -other[i][s], 0, 0.0, "f16")
        if turn % 5 == 4:   # one goes back a little, one goes
            a = rng.choice(who)
            n = rng.randint(0, t.cache.len(a))
            t.cache.truncate(a, n)
            t.k[a], t.v[a], other[i][a] = t.k[a][:n], t.v[a][:n], other[i][a][:n]
            gone = who.pop(rng.randrange(3))
            t.cache.drop(gone)
            new = t.add()
            other[i][new] = t.empty
            who.append(new)
            assert t.cache.len(new) == 0
    ctx.close()


@pytest.mark.gpu
def test_refusals():
    ctx = ctx_for(8, 2, 128, "bf16", layers=2)

    def refused(code, f, *a, **kw):
        with pytest.raises(CakeB200Error) as e:
            f(*a, **kw)
        assert e.value.code == code, str(e.value)

    for kw in (dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(max_seqs=0), dict(max_seq=-1), dict(max_seq=1 << 17)):
        refused(EINVAL, PagedCache, ctx, 4, **{"page_size": 16, **kw})
    refused(EINVAL, PagedCache, ctx, 0, 16)
    refused(EINVAL, PagedCache, ctx, 1 << 30, 16)
    for shape in ((30, 64), (40, 64, 1), (40, 0)):
        with pytest.raises(ValueError):
            PagedCache(ctx, 4, 16, max_seq=40, rotation=(torch.zeros(shape, device="cuda"),) * 2)
    with pytest.raises(ValueError):
        PagedCache(ctx, 4, 16, max_seq=40, rotation=(torch.zeros(40, 64),) * 2)
    with pytest.raises(ValueError):
        PagedCache(ctx, 4, 16, max_seq=40, rotation=(torch.zeros(40, 64, device="cuda", dtype=torch.float64),) * 2)
    table = torch.zeros(40, 64, device="cuda")
    for pages, page, seqs, n in ((4, 16, 1, 2147483647), (4, 16, 1 << 20, 1 << 20), (1 << 27, 16, 1, 40)):
        rc = lib().cake_b200_pages_create(ctx.h, pages, page, seqs, n, table.data_ptr(), table.data_ptr(), 128, byref(c_void_p()))
        assert rc == EINVAL
    assert lib().cake_b200_pages_create(ctx.h, 4, 16, 1, 40, table.data_ptr(), None, 128, byref(c_void_p())) == EINVAL
    assert lib().cake_b200_pages_create(ctx.h, 4, 16, 1, 40, table.data_ptr() + 4, table.data_ptr(), 128, byref(c_void_p())) == EINVAL
    for half in (4, 72):
        refused(EINVAL, PagedCache, ctx, 4, 16, max_seq=40, rotation=(torch.zeros(40, half, device="cuda"),) * 2)
    cache = PagedCache(ctx, 4, 16, max_seqs=2, max_seq=40)
    a, b = cache.add(), cache.add()
    refused(ESTATE, cache.add)
    x = normal((3, 2, 128), "bf16", 1)
    q = normal((3, 8, 128), "bf16", 2)
    with pytest.raises(ValueError):
        cache.append(0, None, x, x)   # no step
    cache.step([a], [3])
    refused(ESTATE, cache.attend, 0, q)     # no rows
    refused(ESTATE, cache.read, 0)
    refused(EINVAL, cache.append, 2, q, x, x)
    refused(EINVAL, cache.append, -1, q, x, x)
    cache.append(0, q, x, x)
    refused(EINVAL, cache.attend, 0, q, window=-1)
    for scale in (-1.0, float("nan"), float("inf")):
        refused(EINVAL, cache.attend, 0, q, scale=scale)
    refused(ESTATE, cache.attend, 1, q)
    for bad in (q[:2], q[:, :4], q[..., :64], q[0]):
        with pytest.raises(ValueError):
            cache.attend(0, bad)
    for bad in (q.half(), q.cpu()):
        with pytest.raises(ValueError):
            cache.attend(0, bad)
    with pytest.raises(ValueError):
        cache.append(0, q, x, x[:2])
    with pytest.raises(ValueError):
        cache.step([a], [1, 2])
    refused(EINVAL, cache.step, [], [])
    refused(EINVAL, cache.step, [a, a], [1, 1])
    refused(EINVAL, cache.step, [a, 2], [1, 1])
    refused(EINVAL, cache.step, [-1], [1])
    refused(EINVAL, cache.step, [a], [0])
    refused(ESTATE, cache.step, [a], [38])
    refused(ENOMEM, cache.step, [a, b], [30, 17])
    assert cache.len(a) == 3 and cache.len(b) == 0 and cache.available == 3
    cache.attend(0, q)                       # the step still stands
    refused(ESTATE, cache.read, 0, a, 0, 4)
    refused(ESTATE, cache.read, 0, a, -1, 2)
    refused(ESTATE, cache.read, 0, b, 0, 1)
    refused(EINVAL, cache.read, 0, 5, 0, 1)
    cache.step([a], [3])
    refused(ESTATE, cache.append, 1, q, x, x)   # block 1 has no rows in front of these
    cache.append(0, q, x, x)
    refused(ESTATE, cache.truncate, a, 7)
    refused(ESTATE, cache.truncate, a, -1)
    refused(EINVAL, cache.truncate, 3, 0)
    cache.truncate(a, 4)
    refused(ESTATE, cache.attend, 0, q)         # its step is gone
    cache.drop(b)
    refused(EINVAL, cache.drop, b)
    assert cache.len(b) < 0 and cache.len(a) == 4 and cache.read(0, a)[0].shape[0] == 4
    cache.close()
    refused(EINVAL, cache.add)
    ctx.close()
    ctx = ctx_for(4, 2, 32, "bf16")
    refused(EINVAL, PagedCache, ctx, 4, 16)
    ctx.close()


@pytest.mark.gpu
def test_a_result_on_its_queries_is_refused():
    """Several CTAs read the same queries: a result that covers any of them is no call, one right beside them is."""
    ctx = ctx_for(8, 2, 64, "bf16")
    cache = PagedCache(ctx, 8, 16, max_seqs=2, max_seq=60)
    s = cache.add()
    cache.step([s], [2])
    x = normal((2, 2, 64), "bf16", 1)
    q = normal((4, 8, 64), "bf16", 2)
    cache.append(0, None, x, x)
    want = cache.attend(0, q[1:3])
    at, row = q.data_ptr(), 8 * 64 * 2

    def call(first, out, tok=8 * 64):
        return lib().cake_b200_pages_attend(cache.h, 0, at + first * row, tok, at + out * row, 0, 0.0, cache._stream())
    torch.cuda.synchronize()
    for first, out, tok in ((1, 1, 512), (1, 0, 512), (1, 2, 512), (0, 1, 1024), (1, 0, 0)):
        assert call(first, out, tok) == EINVAL
    q[3] = q[1]
    assert call(2, 0) == 0
    torch.cuda.synchronize()
    assert torch.equal(q[0:2], cache.attend(0, q[2:4])) and torch.isfinite(want.float()).all()
    cache.close()
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 64, 1024), (32, 8, 128, 512), (8, 4, 256, 1024)])
def test_pages_that_are_many_tiles(heads, kv, hd, page):
    ctx = ctx_for(heads, kv, hd, "f16")
    talk = [(1000, 1), (1023, 2), (1024, 40), (0, 1100), (3000, 1), (511, 513), (2047, 130)]
    cache = PagedCache(ctx, sum(-(-(h + r) // page) for h, r in talk), page, max_seqs=len(talk), max_seq=3001)
    t = Talks(cache, kv, hd, "f16")
    ids = [t.add() for _ in talk]
    some = [i for i, (h, _) in enumerate(talk) if h]
    t.step([ids[i] for i in some], [talk[i][0] for i in some], 1)
    counts = [r for _, r in talk]
    t.step(ids, counts, 2)
    q = normal((sum(counts), heads, hd), "f16", 3)
    t.check(q, ids, counts)
    t.check(q, ids, counts, window=700)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (8, 8, 128), (8, 1, 256)])
def test_hundreds_of_sequences(heads, kv, hd):
    """More runs than CTAs, of every length up to a few tiles; then a few rows and portions of them mixed in any order."""
    rng = random.Random(heads + hd)
    ctx = ctx_for(heads, kv, hd, "bf16")
    cache = PagedCache(ctx, 4000, 16, max_seqs=400, max_seq=400)
    t = Talks(cache, kv, hd, "bf16")
    ids = [t.add() for _ in range(400)]
    t.step(ids, [rng.randint(1, 140) for _ in ids], 1)
    who = rng.sample(ids, 333)
    t.step(who, [1] * 333, 2)
    q = normal((333, heads, hd), "bf16", 3)
    out = cache.attend(0, q)
    for i in rng.sample(range(333), 40):
        check_rows(out[i:i + 1], q[i:i + 1], t.k[who[i]], t.v[who[i]], 0, 0.0, "bf16")
    who = rng.sample(ids, 350)
    counts = [rng.choice([1, 1, 2, 3, 17, 60]) for _ in who]
    t.step(who, counts, 4)
    q = normal((sum(counts), heads, hd), "bf16", 5)
    for window in (0, 33):
        out = cache.attend(0, q, window=window)
        for i in rng.sample(range(350), 40):
            a = sum(counts[:i])
            check_rows(out[a:a + counts[i]], q[a:a + counts[i]], t.k[who[i]], t.v[who[i]], window, 0.0, "bf16")
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 2, 64), (8, 4, 256)])
def test_a_query_that_is_no_number_stays_alone(heads, kv, hd):
    ctx = ctx_for(heads, kv, hd, "bf16")
    cache = PagedCache(ctx, 80, 16, max_seqs=3, max_seq=400)
    t = Talks(cache, kv, hd, "bf16")
    ids, counts = [t.add() for _ in range(3)], [1, 2, 150]
    t.step(ids, [200, 100, 77], 1)
    t.step(ids, counts, 2)
    q = normal((153, heads, hd), "bf16", 3)
    want = cache.attend(0, q)
    for row, head, bad in ((0, 0, float("nan")), (2, heads - 1, float("inf")), (3, 1, float("nan")), (90, 0, -float("inf")), (152, heads - 1, float("nan"))):
        p = q.clone()
        p[row, head, 5] = bad
        got = cache.attend(0, p)
        odd = torch.zeros(153, heads, dtype=torch.bool, device="cuda")
        odd[row, head] = True
        assert torch.equal(got[~odd], want[~odd]) and not torch.equal(got[odd], want[odd])
    ctx.close()


@pytest.mark.gpu
def test_memory_comes_back():
    """Caches that are made and closed leave the device's memory as it was."""
    ctx = ctx_for(32, 8, 128, "bf16")

    def once():
        cache = PagedCache(ctx, 12000, 64, max_seqs=2, max_seq=1000)   # 3 GB
        s = cache.add()
        x = normal((10, 8, 128), "bf16", 1)
        cache.step([s], [10])
        cache.append(0, None, x, x)
        cache.attend(0, normal((10, 32, 128), "bf16", 2))
        cache.close()
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]

    first = once()
    assert all(once() >= first - (64 << 20) for _ in range(5))
    ctx.close()
