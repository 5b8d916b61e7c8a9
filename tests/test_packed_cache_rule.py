"""Caches in four bits: which way a call of many rows goes (no GPU)."""
import os
import subprocess

from tests.test_packed_cache import ROOT

# query heads a key head, key heads, batch rows, rows a call, position, device microseconds on codes and expanded
MEASURED = [(4, 8, 1, 5, 0, 4.5, 7.2), (4, 8, 1, 16, 16000, 42.4, 64.3), (4, 8, 1, 64, 16000, 131.2, 74.9), (4, 8, 1, 64, 4000, 40.7, 34.2),
            (8, 1, 1, 16, 4000, 13.3, 21.5), (8, 1, 8, 32, 16000, 130.9, 75.8), (4, 32, 1, 5, 16000, 73.8, 152.9), (4, 32, 1, 64, 1000, 58.5, 30.4),
            (4, 8, 8, 5, 4000, 40.2, 65.9), (8, 8, 8, 3, 16000, 132.3, 229.6), (4, 8, 8, 32, 4000, 150.0, 72.1), (4, 8, 8, 32, 0, 27.5, 10.1),
            (4, 8, 32, 5, 4000, 149.2, 217.2), (4, 8, 32, 5, 16000, 492.5, 861.9), (4, 8, 32, 5, 0, 25.4, 9.6), (4, 8, 32, 16, 4000, 283.2, 218.7),
            (1, 8, 32, 17, 16000, 494.3, 869.8), (4, 32, 32, 5, 16000, 1922.6, 3662.0), (4, 32, 32, 8, 250, 118.6, 78.9), (4, 32, 32, 16, 1000, 410.2, 234.0),
            (4, 32, 32, 64, 16000, 15407.8, 5578.6), (4, 8, 1, 16, 2000, 13.1, 16.4), (4, 8, 32, 64, 1000, 420.8, 92.6), (8, 32, 8, 16, 2000, 320.0, 119.5),
            (4, 1, 1, 32, 4000, 13.1, 21.6)]


def test_the_faster_way_is_taken(tmp_path):
    src = tmp_path / "rule.cpp"
    calls = "\n".join(f"  printf(\"%d\\n\", way({g}, {kv}, {b}, {s}, {at}));" for g, kv, b, s, at, _, _ in MEASURED)
    src.write_text(r'''
#include "packed_cache.cuh"
#include <cstdio>
using namespace cake::pc;
int way(int g, int kv, int b, int s, int at, int hd = 128, int first = 0) {
  Attend a{};
  a.B = b; a.S = s; a.n_heads = g * kv; a.n_kv = kv; a.hd = hd; a.pos0 = at; a.first = first;
  return many_rows(a, 148);
}
int main() {
''' + calls + r'''
  // one token, other heads, and a window: its positions count, not those in front of it
  printf("%d\n", way(8, 8, 32, 1, 4000) + way(4, 8, 1, 64, 16000, 64) + way(4, 8, 1, 64, 16000, 256) + way(4, 8, 1, 16, 16000, 128, 15000));
}
''')
    exe = tmp_path / "rule"
    subprocess.check_call(["g++", "-std=c++17", "-x", "c++", str(src), "-I", os.path.join(ROOT, "cake_b200", "csrc"), "-I", "/usr/local/cuda/include", "-o", str(exe)])
    *ways, rest = [int(x) for x in subprocess.check_output([str(exe)], text=True).split()]
    assert rest == 0
    for case, way in zip(MEASURED, ways):
        codes, expanded = case[-2:]
        assert (expanded if way else codes) <= 1.1 * min(codes, expanded), case
