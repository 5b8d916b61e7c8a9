"""The C entries of caches in pages without a GPU: csrc/paged_host.cuh compiled with g++ in front of CUDA calls that are host memory and copies, of which any one, or any
allocation of the host's, can be made to fail."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cake_b200", "csrc")

FRONT = r'''
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cmath>
#include <mutex>
#include <new>
#include <set>
#include "cake_b200.h"
#include "paged_cache.cuh"
using namespace cake;

// ---- failures on demand: the n-th CUDA call, or the n-th allocation, from now
static long cuda_left = -1, new_left = -1, live = 0;
static bool cuda_fails() { return cuda_left >= 0 && cuda_left-- == 0; }
void *operator new(size_t n) {
  if (new_left >= 0 && new_left-- == 0) throw std::bad_alloc();
  void *p = malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void *operator new(size_t n, const std::nothrow_t &) noexcept { return new_left >= 0 && new_left-- == 0 ? nullptr : malloc(n ? n : 1); }
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, const std::nothrow_t &) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }
#define FAKE if (cuda_fails()) return cudaErrorUnknown
static cudaError_t take(void **p, size_t n) { FAKE; *p = malloc(n); live++; return cudaSuccess; }
static cudaError_t give(void *p) { if (p) live--; free(p); return cudaSuccess; }
extern "C" {
cudaError_t cudaMalloc(void **p, size_t n) { return take(p, n); }
cudaError_t cudaMallocHost(void **p, size_t n) { return take(p, n); }
cudaError_t cudaHostAlloc(void **p, size_t n, unsigned) { return take(p, n); }
cudaError_t cudaMallocFromPoolAsync(void **p, size_t n, cudaMemPool_t, cudaStream_t) { return take(p, n); }
cudaError_t cudaFree(void *p) { return give(p); }
cudaError_t cudaFreeHost(void *p) { return give(p); }
cudaError_t cudaFreeAsync(void *p, cudaStream_t) { return give(p); }
cudaError_t cudaMemcpyAsync(void *d, const void *s, size_t n, cudaMemcpyKind, cudaStream_t) { FAKE; memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void *d, int v, size_t n, cudaStream_t) { FAKE; memset(d, v, n); return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *e, unsigned) { FAKE; *e = (cudaEvent_t)1; return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { FAKE; return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { FAKE; return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemPoolTrimTo(cudaMemPool_t, size_t) { return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t) { return "made to fail"; }
}
static const cudaStream_t OWN = (cudaStream_t)16, CAPTURING = (cudaStream_t)48;
extern "C" cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus *st) {
  *st = s == CAPTURING ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}

// ---- what the entries find around them
static char g_err[512];
static int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
  return code;
}
#define CU(call) do { cudaError_t e_ = (call); if (e_ != cudaSuccess) return fail(CAKE_B200_ECUDA, "%s", #call); } while (0)
#define RC(call) do { int rc_ = (call); if (rc_ != CAKE_B200_OK) return rc_; } while (0)
struct cake_b200_block { int window = -1; bool use_rope = true; };
struct cake_b200_ctx {
  cake_b200_config cfg{};
  int device = 0, sm_count = 148, rot = 0, nqkv = 0;
  size_t es = 2;
  cudaStream_t stream = OWN;
  cudaMemPool_t pc_pool = nullptr;
  unsigned wait_failures = 0;
  int *wait_err = nullptr;
  void *cos_t = nullptr, *sin_t = nullptr;
  unsigned long long launches = 0;
  bool pc_behind = true;
  struct Staging { void *p = nullptr; size_t cap = 0; cudaEvent_t done = nullptr; bool busy = false; } pg_stage[4];
  unsigned pg_next = 0;
  float *pg_cos = nullptr, *pg_sin = nullptr;
  pg::Clusters pg_clusters{};
};
constexpr unsigned long long PC_POOL_KEEPS = 1ull << 30;
static std::mutex g_live_mu;
static std::set<cake_b200_ctx *> g_live_ctx;
struct OnDevice { explicit OnDevice(int) {} };
static int check_waits(cake_b200_ctx *) { return 0; }
static int settle(cake_b200_ctx *) { return cuda_fails() ? fail(CAKE_B200_ECUDA, "settle") : 0; }
static int ops_ready(cake_b200_ctx *) { return 0; }
static bool unaligned(const void *p, size_t s = 0) { return ((uintptr_t)p & 15) || s % 8; }
static uint64_t counted;
static uint64_t *launch_counter(cake_b200_ctx *) { return &counted; }
static int no_capture(cudaStream_t s, const char *) { return s == CAPTURING ? fail(CAKE_B200_ESTATE, "capturing") : 0; }
template <typename F> static int on_stream(cake_b200_ctx *c, void *stream, F &&call) {
  if (cuda_fails()) return fail(CAKE_B200_ECUDA, "events in front of the call");
  const cudaStream_t own = c->stream;
  if (stream) c->stream = (cudaStream_t)stream;
  const int rc = call();
  c->stream = own;
  if (cuda_fails()) return rc ? rc : fail(CAKE_B200_ECUDA, "the event behind the call");
  return rc;
}
template <typename F> static int dispatch(F &&f) { struct Tag { typedef unsigned short type; }; return f(Tag{}); }
#define DISPATCH_T(dtype, ...) dispatch(__VA_ARGS__)
#define T_LAMBDA [&](auto tag_) -> int

namespace cake { namespace pg {   // kernels that do what the host can see of them
int few_ctas(int hd, int sms) { return (hd == 256 ? 1 : 2) * sms; }
int room(int hd, int sms, int n_kv) { return std::max(1, (hd == 256 ? 1 : 2) * sms / n_kv); }
size_t few_floats(int, int) { return 64; }
size_t tiles_floats(int, int, int) { return 64; }
int prepare(int, int, Clusters *c) { FAKE; c->most[0][0] = 1; return 0; }
int spread(cudaStream_t, const StepHead *h, int n_seqs, int, int, int *table, int2 *rows, uint64_t *) {
  FAKE;
  const SeqRow *s = (const SeqRow *)(h + 1);
  const int2 *u = (const int2 *)(s + n_seqs);
  for (int i = 0; i < h->n_updates; i++) table[u[i].x] = u[i].y;
  for (int i = 0; i < n_seqs; i++)
    for (int r = 0; r < s[i].count; r++) rows[s[i].row0 + r] = int2{s[i].slot, s[i].pos0 + r};
  return 0;
}
static int appended, attended, been_read;
int append(cudaStream_t, int, const Pool &, const Append &, int, uint64_t *) { FAKE; appended++; return 0; }
int read(cudaStream_t, const Pool &, const Read &, int, uint64_t *) { FAKE; been_read++; return 0; }
int attend(cudaStream_t, int, const Pool &, const Attend &, const Scratch &, uint64_t *) { FAKE; attended++; return 0; }
} }
#define IS(x) do { if (!(x)) { printf("line %d: %s   (%s)\n", __LINE__, #x, g_err); exit(1); } } while (0)
static cake_b200_ctx *context(int heads, int kv, int hd) {
  auto *c = new cake_b200_ctx;
  c->cfg.n_heads = heads; c->cfg.n_kv_heads = kv; c->cfg.head_dim = hd; c->cfg.n_layers = 2; c->cfg.max_seq = 4096;
  g_live_ctx.insert(c);
  return c;
}
static void gone(cake_b200_ctx *c) {
  for (auto &t : c->pg_stage) if (t.p) cudaFreeHost(t.p);
  g_live_ctx.erase(c);
  delete c;
}
alignas(16) static char mem[1 << 20];
'''


def run(tmp_path, main):
    text = open(os.path.join(CSRC, "paged_host.cuh")).read()
    text = re.sub(r"template <typename T> __global__ void widen_kernel.*?\n}\n", "", text, flags=re.S)   # (no rotation here: nothing to widen)
    text = re.sub(r"widen_kernel<T><<<.*?>>>\([^;]*\);", "(void)n;", text)
    src = tmp_path / "host.cpp"
    src.write_text(FRONT + text + "int main() {\n" + main + "\nreturn 0; }\n")
    exe = tmp_path / "host"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-w", "-x", "c++", str(src), "-I", CSRC, "-I", os.path.join(ROOT, "include"),
                           "-I", "/usr/local/cuda/include", "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr[-3000:]


@pytest.mark.parametrize("what", ["cuda_left", "new_left"])
def test_a_step_that_fails_takes_nothing(tmp_path, what):
    """Whichever call or allocation fails on a step's way: lengths and pages are those in front of it, no step stands, nothing that was refused is attended over, and
    the next step is like any other."""
    run(tmp_path, r'''
  for (int kept = 0; kept < 2; kept++) {   // without and with a plan that a captured call reads
    long tries = 0;
    for (long n = 0;; n++) {
      cake_b200_ctx *c = context(8, 2, 64);
      cake_b200_pages *g = nullptr;
      IS(cake_b200_pages_create(c, 40, 16, 4, 300, nullptr, nullptr, 0, &g) == 0);
      int s[3], few[3] = {1, 40, 2}, more[3] = {20, 1, 70};
      for (int &x : s) IS(cake_b200_pages_add(g, &x) == 0);
      char *q = mem, *k = mem + (1 << 18), *v = k + (1 << 17), *out = mem + (1 << 19);
      auto pass = [&](void *stream) {
        RC(cake_b200_pages_append(g, 0, nullptr, 0, k, 128, v, 128, nullptr, 0, stream));
        return cake_b200_pages_attend(g, 0, q, 512, out, 7, 0.f, stream);
      };
      IS(cake_b200_pages_step(g, s, few, 3, nullptr) == 0 && pass(nullptr) == 0);
      if (kept) IS(pass(CAPTURING) == 0);
      const int free_pages = cake_b200_pages_available(g);
      WHAT = n;
      const int rc = cake_b200_pages_step(g, s, more, 3, (void *)32);
      const bool hit = WHAT < 0;
      WHAT = -1;
      IS(c->stream == OWN);
      if (!hit) {   // nothing more to fail
        IS(rc == 0 && tries >= 2);
        cake_b200_pages_free(g);
        gone(c);
        break;
      }
      tries++;
      if (rc) {
        for (int i = 0; i < 3; i++) IS(cake_b200_pages_len(g, s[i]) == few[i]);
        IS(cake_b200_pages_available(g) == free_pages);
        const int before = pg::attended;
        if (g->book.step.empty()) IS(pass(nullptr) == CAKE_B200_ESTATE);
        else IS(g->book.n_rows == 43);   // the one before still stands, whole
        IS(cake_b200_pages_read(g, 0, -1, 0, 93, k, v, nullptr) != 0);
        IS(pg::attended == before);
      } else IS(cake_b200_pages_len(g, s[0]) == 21);
      for (int i = 0; i < 3; i++) IS(cake_b200_pages_truncate(g, s[i], few[i]) == 0);
      IS(cake_b200_pages_step(g, s, more, 3, nullptr) == 0 && pass(nullptr) == 0);
      for (int i = 0; i < 3; i++) {
        IS(cake_b200_pages_len(g, s[i]) == few[i] + more[i]);
        for (size_t j = 0; j < g->book.seqs[s[i]].pages.size(); j++) IS(g->table[s[i] * g->book.per_seq + j] == g->book.seqs[s[i]].pages[j]);
      }
      IS(g->step->shape == g->book.shape);
      for (int i = 0; i < 3; i++) IS(cake_b200_pages_drop(g, s[i]) == 0);
      IS(cake_b200_pages_available(g) == 40);
      cake_b200_pages_free(g);
      gone(c);
    }
    IS(live == 0);
  }
'''.replace("WHAT", what))


def test_positions_of_one_sequence_are_read_outside_captures(tmp_path):
    """A graph would read whatever sequence, or none, has that row of the table by then."""
    run(tmp_path, r'''
  cake_b200_ctx *c = context(8, 2, 64);
  cake_b200_pages *g = nullptr;
  IS(cake_b200_pages_create(c, 40, 16, 4, 300, nullptr, nullptr, 0, &g) == 0);
  int s, n = 20;
  IS(cake_b200_pages_add(g, &s) == 0 && cake_b200_pages_step(g, &s, &n, 1, nullptr) == 0);
  IS(cake_b200_pages_append(g, 0, nullptr, 0, mem, 128, mem, 128, nullptr, 0, nullptr) == 0);
  IS(cake_b200_pages_read(g, 0, s, 3, 5, mem, mem + 65536, (void *)32) == 0 && pg::been_read == 1);
  IS(cake_b200_pages_read(g, 0, s, 3, 5, mem, mem + 65536, CAPTURING) == CAKE_B200_ESTATE && pg::been_read == 1);
  IS(cake_b200_pages_read(g, 0, -1, 0, 20, mem, mem + 65536, CAPTURING) == 0 && pg::been_read == 2);
  cake_b200_pages_free(g);
  gone(c);
''')
