"""Caches in four bits: which way a call of many rows goes (no GPU)."""
import os
import subprocess

from tests.test_packed_cache import ROOT

# query heads a key head, key heads, batch rows, rows a call, position, device microseconds on codes and expanded
MEASURED = [(4, 8, 1, 5, 0, 4.1, 7.2), (4, 8, 1, 16, 16000, 39.7, 64.3), (4, 8, 1, 64, 16000, 121.8, 75.7), (4, 8, 1, 64, 4000, 37.8, 34.4),
            (8, 1, 1, 16, 4000, 12.3, 21.6), (8, 1, 8, 32, 16000, 121.6, 76.3), (4, 32, 1, 5, 16000, 69.2, 155.4), (4, 32, 1, 64, 1000, 55.2, 30.4),
            (4, 8, 8, 5, 4000, 37.6, 66.4), (8, 8, 8, 3, 16000, 122.3, 230.3), (4, 8, 8, 32, 4000, 139.6, 72.4), (4, 8, 8, 32, 0, 25.9, 10.0),
            (4, 8, 32, 5, 4000, 139.0, 217.2), (4, 8, 32, 5, 16000, 455.8, 849.1), (4, 8, 32, 5, 0, 22.8, 9.1), (4, 8, 32, 16, 4000, 259.5, 218.2),
            (1, 8, 32, 17, 16000, 456.5, 856.2), (4, 32, 32, 5, 16000, 1780.5, 3577.6), (4, 32, 32, 8, 250, 113.0, 80.0), (4, 32, 32, 16, 1000, 394.0, 235.3),
            (4, 32, 32, 64, 16000, 14236.0, 5374.5), (4, 8, 1, 16, 2000, 12.5, 16.5), (4, 8, 32, 64, 1000, 392.4, 92.2), (8, 32, 8, 16, 2000, 300.1, 119.5),
            (4, 1, 1, 32, 4000, 12.3, 21.6)]


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
