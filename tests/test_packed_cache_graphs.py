"""Caches in four bits: what captured calls leave behind in their graphs."""
import os
import subprocess

import pytest
import torch

from tests.test_packed_cache import ROOT, check_attention, ctx_for, filled, queries


def test_memory_that_captures_have_used_is_kept(tmp_path):
    """No GPU: what is made and released, over calls that grow, outside and inside captures."""
    src = tmp_path / "kept.cpp"
    src.write_text(r'''
#include "kept_memory.cuh"
#include <cstdio>
#include <cstdlib>
#include <map>
std::map<void *, size_t> live;
size_t room = 1 << 30;
int released = 0;
void *make(size_t n) {
  if (n > room) return nullptr;
  void *p = malloc(1);
  live[p] = n;
  return p;
}
void release(void *p) {
  if (!live.erase(p)) { printf("released twice\n"); exit(9); }
  released++;
  free(p);
}
#define IS(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  cake::KeptMemory m;
  const size_t most = 1000;
  IS(m.short_of(10, true));                                   // a capture cannot make it: refused, nothing noted
  IS(m.short_of(10, false));
  void *a = m.grow(10, most, make, release);
  IS(a && m.now == a && m.cap == 10 && live.size() == 1);
  IS(!m.short_of(7, false) && !m.short_of(10, false) && m.short_of(11, true));
  void *b = m.grow(11, most, make, release);                  // no capture has used it: given back
  IS(b && m.cap == 20 && live.size() == 1 && live.count(b) && released == 1);
  IS(!m.short_of(15, true));                                  // a captured call
  IS(!m.short_of(15, false) && m.short_of(21, false));
  void *c = m.grow(300, most, make, release);
  IS(c != b && live.count(b) && live[b] == 20 && m.cap == 300);  // the graph's memory is still there
  void *d = m.grow(301, most, make, release);                 // c is in no graph
  IS(m.cap == 600 && live.size() == 2 && live.count(b) && live.count(d));
  IS(!m.short_of(600, true));
  m.grow(700, most, make, release);
  IS(m.cap == 1000 && live.size() == 3 && live.count(d));
  room = 2500;
  IS(!m.short_of(1000, true));
  m.grow(2000, 10000, make, release);                         // twice as much fits not beside, exactly as much does not either way: as asked
  IS(m.cap == 2000);
  room = 100;
  IS(!m.short_of(5, true));
  IS(!m.grow(3000, 10000, make, release) && !m.now && m.cap == 0);   // none: but the graphs' memory stays
  IS(live.count(b) && live.count(d) && live.size() == 4);
  IS(m.short_of(1, false));
  IS(m.grow(50, 10000, make, release) && m.cap == 50);
  m.release_all(release);
  IS(live.empty() && !m.now && m.short_of(1, false));
  return 0;
}
''')
    exe = tmp_path / "kept"
    subprocess.check_call(["g++", "-std=c++17", "-x", "c++", str(src), "-I", os.path.join(ROOT, "cake_b200", "csrc"), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


@pytest.mark.gpu
def test_a_graph_outlives_calls_that_need_more():
    """Captured over many rows, then calls with more positions, then replayed: the graph's own memory is still its own."""
    ctx = ctx_for(32, 8, 128, "bf16")
    cache, k, v = filled(ctx, 1, 700, 5, "bf16")
    q = queries(1, 300, 32, 128, "bf16", 6)
    cache.attend(0, q, 400)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cache.attend(0, q, 400)
    held = []
    for n in (1500, 4000):
        big, bk, bv = filled(ctx, 1, n, n, "bf16")
        bq = queries(1, 200, 32, 128, "bf16", n)
        check_attention(big.attend(0, bq, n - 200), bq, bk, bv, n - 200, 0, "bf16")
        held.append(torch.full((1 << 24,), float("nan"), device="cuda"))   # what was given back would be somebody else's now
        q.copy_(queries(1, 300, 32, 128, "bf16", n + 1))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_attention(out, q, k, v, 400, 0, "bf16")
        assert all(x.isnan().all() for x in held)
        check_attention(big.attend(0, bq, n - 200), bq, bk, bv, n - 200, 0, "bf16")
    del g
    ctx.close()
