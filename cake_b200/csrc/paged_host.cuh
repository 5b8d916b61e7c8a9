// paged_host.cuh — the C ABI of caches in pages (include/cake_b200.h, cake_b200_pages_*), part of cake_b200.cu
#pragma once

struct cake_b200_pages {
  cake_b200_ctx *ctx;
  int device = 0;
  pg::Book book;
  std::vector<char> blob;            // a step on its way to the device
  // device memory, one piece of the ctx's pool: the step, the page table, the rows' places
  char *arena = nullptr;
  pg::StepHead *step = nullptr;
  int *table = nullptr;
  int2 *rows = nullptr;
  std::vector<void *> pool;          // of each block: the pages and, behind them, their marks
  std::vector<std::vector<int>> len; // positions written, of each block and sequence
  std::vector<char> in_graph;        // a captured call writes this block's rows: how far, only its user knows
  // how a step's attention is cut, for each window that calls have asked for
  struct Plan {
    pg::Window win;
    unsigned long long step = 0, used = 0;   // made for this step; last used in this call
    bool kept = false;                       // captured calls read it: it is made anew with every step
    int longest = 0, tiles = 0, n_cuts = 0, n_items = 0, most_items = 0;   // tiles of the longest run of few rows, of all; cut runs; items of the many-row kernel, now and for any lengths of this shape
    int n_cut_tiles = 0, most_cut_tiles = 0;               // tiles that are cut, now and for any lengths
    char *dev = nullptr;
  } plans[8];
  unsigned long long steps = 0, calls = 0;
  float *few_ws = nullptr, *tiles_ws = nullptr;
  const float *cos_t = nullptr, *sin_t = nullptr;
  int rot = 0;
  int *bad = nullptr;                // pinned: a replayed call met a step of another shape
  unsigned wait_failures = 0;        // the context's count when there was no sequence last: another one, and the rows may be no results
  size_t page_bytes() const { return (size_t)2 * book.page * ctx->cfg.n_kv_heads * ctx->cfg.head_dim * 2; }
};

static int pages_call(const cake_b200_pages *g, const char *what) {
  if (!g) return fail(CAKE_B200_EINVAL, "null argument");
  RC(check_waits(g->ctx));
  if (g->wait_failures != g->ctx->wait_failures)
    return fail(CAKE_B200_ESTATE, "%s: a kernel gave up a wait while these sequences were there and their rows may be no results: drop them all", what);
  if (*(volatile int *)g->bad) {
    *(volatile int *)g->bad = 0;
    return fail(CAKE_B200_ESTATE, "%s: a replayed graph's calls were made for steps of other counts than the present one and did nothing", what);
  }
  return CAKE_B200_OK;
}
// No exception leaves a C entry: what of them makes host memory runs in here (inside on_stream, which gives the ctx its stream back when the call returns)
template <typename F> static int with_memory(F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return fail(CAKE_B200_ENOMEM, "out of host memory");
  }
}
static bool is_capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st;
  const cudaError_t e = cudaStreamIsCapturing(s, &st);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e != cudaSuccess || st != cudaStreamCaptureStatusNone;
}
// host data on its way to the device: pinned buffers in turn.  pages_room: the next upload has the room for so much.
static int pages_room(cake_b200_ctx *c, size_t bytes) {
  cake_b200_ctx::Staging &t = c->pg_stage[c->pg_next % (sizeof c->pg_stage / sizeof c->pg_stage[0])];
  if (!t.done) CU(cudaEventCreateWithFlags(&t.done, cudaEventDisableTiming));
  if (t.busy) CU(cudaEventSynchronize(t.done));
  t.busy = false;
  if (bytes > t.cap) {
    if (t.p) cudaFreeHost(t.p);
    t.p = nullptr; t.cap = 0;
    const size_t cap = std::max<size_t>(bytes, 1 << 16);
    CU(cudaMallocHost(&t.p, cap));
    t.cap = cap;
  }
  return CAKE_B200_OK;
}
static int pages_upload(cake_b200_ctx *c, void *dst, const void *src, size_t bytes) {
  RC(pages_room(c, bytes));
  cake_b200_ctx::Staging &t = c->pg_stage[c->pg_next++ % (sizeof c->pg_stage / sizeof c->pg_stage[0])];
  memcpy(t.p, src, bytes);
  CU(cudaMemcpyAsync(dst, t.p, bytes, cudaMemcpyHostToDevice, c->stream));
  CU(cudaEventRecord(t.done, c->stream));
  t.busy = true;
  return CAKE_B200_OK;
}
template <typename T> __global__ void widen_kernel(const T *x, float *y, size_t n) {
  for (size_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) y[i] = DT<T>::to_f(x[i]);
}

extern "C" int cake_b200_pages_create(cake_b200_ctx *c, int n_pages, int page_size, int max_seqs, int max_seq, const float *cos_dev, const float *sin_dev,
                                      int rot, cake_b200_pages **out) {
  if (!c || !out) return fail(CAKE_B200_EINVAL, "null argument");
  const cake_b200_config &f = c->cfg;
  if (f.layer_list) return fail(CAKE_B200_EINVAL, "caches in pages are for the Llama-family blocks");
  if (!pg::head_dim_ok(f.head_dim)) return fail(CAKE_B200_EINVAL, "caches in pages hold heads of 64, 128 or 256 entries, not %d", f.head_dim);
  if (!pg::page_ok(page_size)) return fail(CAKE_B200_EINVAL, "a page holds 16, 32, .. 1024 positions (a power of two), not %d", page_size);
  if (n_pages < 1 || max_seqs < 1 || max_seq < 1) return fail(CAKE_B200_EINVAL, "pages, max_seqs and max_seq are 1 or more");
  if ((long long)n_pages * page_size > (1ll << 30) || max_seq > 1 << 30 || max_seqs > 1 << 16 || (long long)max_seqs * ((max_seq + page_size - 1) / page_size) > (1ll << 28))
    return fail(CAKE_B200_EINVAL, "%d pages of %d positions, %d sequences of %d: more than a cache in pages counts", n_pages, page_size, max_seqs, max_seq);
  const bool own = !cos_dev && !sin_dev;
  if (!own && (!cos_dev || !sin_dev)) return fail(CAKE_B200_EINVAL, "cos without sin");
  if (own) {
    rot = c->rot;
    if (max_seq > f.max_seq) return fail(CAKE_B200_EINVAL, "max_seq %d exceeds config max_seq %d (RoPE table rows)", max_seq, f.max_seq);
  }
  if (rot < 0 || rot > f.head_dim || rot % 16) return fail(CAKE_B200_EINVAL, "caches in pages rotate multiples of 16 entries of a head, not %d", rot);
  if (!own && (((uintptr_t)cos_dev | (uintptr_t)sin_dev) & 15)) return fail(CAKE_B200_EINVAL, "rotation tables start on 16-byte boundaries");
  const OnDevice dev(c->device);
  RC(ops_ready(c));
  RC(settle(c));
  if (own && rot && !c->pg_cos) {
    const size_t n = (size_t)f.max_seq * (c->rot / 2);
    float *both = nullptr;
    CU(cudaMalloc(&both, 2 * n * sizeof(float)));
    const int rc = DISPATCH_T(f.dtype, T_LAMBDA {
      typedef typename decltype(tag_)::type T;
      widen_kernel<T><<<592, 256, 0, c->stream>>>((const T *)c->cos_t, both, n);
      widen_kernel<T><<<592, 256, 0, c->stream>>>((const T *)c->sin_t, both + n, n);
      CU(cudaGetLastError());
      return CAKE_B200_OK;
    });
    if (rc != CAKE_B200_OK) { cudaFree(both); return rc; }
    c->launches += 2;
    c->pg_cos = both; c->pg_sin = both + n;
    c->pc_behind = true;
  }
  return with_memory([&]() -> int {
    auto *g = new cake_b200_pages{c, c->device};
    struct Guard { cake_b200_pages *g; ~Guard() { if (g) cake_b200_pages_free(g); } } guard{g};
    g->book.init(n_pages, page_size, max_seqs, max_seq);
    g->pool.assign((size_t)f.n_layers, nullptr);
    g->len.assign((size_t)f.n_layers, std::vector<int>((size_t)max_seqs, 0));
    g->in_graph.assign((size_t)f.n_layers, 0);
    g->rot = rot;
    g->wait_failures = c->wait_failures;
    if (rot) { g->cos_t = own ? c->pg_cos : cos_dev; g->sin_t = own ? c->pg_sin : sin_dev; }
    CU(cudaMallocHost(&g->bad, 4));
    *g->bad = 0;
    if (!c->pg_clusters.most[0][0]) CU((cudaError_t)pg::prepare(f.dtype, f.head_dim, &c->pg_clusters));
    const size_t s_step = sizeof(pg::StepHead) + (size_t)max_seqs * sizeof(pg::SeqRow) + (size_t)n_pages * 8, s_table = (size_t)max_seqs * g->book.per_seq * 4,
                 s_rows = (size_t)n_pages * page_size * 8, s_ws = pg::few_floats(f.head_dim, c->sm_count) * 4;
    g->blob.reserve(s_step);
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    void *arena = nullptr;
    CU(cudaMallocFromPoolAsync(&arena, up(s_step) + up(s_table) + up(s_ws) + s_rows, c->pc_pool, c->stream));
    g->arena = (char *)arena;
    g->step = (pg::StepHead *)g->arena;
    g->table = (int *)(g->arena + up(s_step));
    g->few_ws = (float *)(g->arena + up(s_step) + up(s_table));
    g->rows = (int2 *)(g->arena + up(s_step) + up(s_table) + up(s_ws));
    CU(cudaMemsetAsync(arena, 0, up(s_step) + up(s_table), c->stream));
    c->pc_behind = true;
    guard.g = nullptr;
    *out = g;
    return CAKE_B200_OK;
  });
}
extern "C" void cake_b200_pages_free(cake_b200_pages *g) {
  if (!g) return;
  const OnDevice dev(g->device);
  {
    std::lock_guard<std::mutex> lk(g_live_mu);
    const bool live = g_live_ctx.count(g->ctx) != 0;
    if (live) {
      (void)settle(g->ctx);
      cudaStreamSynchronize(g->ctx->stream);
    }
    for (void *p : g->pool)
      if (p) (void)(live ? cudaFreeAsync(p, g->ctx->stream) : cudaFree(p));
    for (auto &p : g->plans)
      if (p.dev) (void)(live ? cudaFreeAsync(p.dev, g->ctx->stream) : cudaFree(p.dev));
    if (g->tiles_ws) (void)(live ? cudaFreeAsync(g->tiles_ws, g->ctx->stream) : cudaFree(g->tiles_ws));
    if (g->arena) (void)(live ? cudaFreeAsync(g->arena, g->ctx->stream) : cudaFree(g->arena));
    if (live && cudaStreamSynchronize(g->ctx->stream) == cudaSuccess) (void)cudaMemPoolTrimTo(g->ctx->pc_pool, PC_POOL_KEEPS);
  }
  if (g->bad) cudaFreeHost(g->bad);
  (void)cudaGetLastError();
  delete g;
}

extern "C" int cake_b200_pages_add(cake_b200_pages *g, int *seq) {
  if (!g || !seq) return fail(CAKE_B200_EINVAL, "null argument");
  if (!g->book.any()) g->wait_failures = g->ctx->wait_failures;
  const int s = g->book.add();
  if (s < 0) return fail(CAKE_B200_ESTATE, "all %d sequences are taken", g->book.max_seqs);
  for (auto &l : g->len) l[(size_t)s] = 0;
  *seq = s;
  return CAKE_B200_OK;
}
extern "C" int cake_b200_pages_truncate(cake_b200_pages *g, int seq, int len) {
  if (!g) return fail(CAKE_B200_EINVAL, "null argument");
  if (!g->book.has(seq)) return fail(CAKE_B200_EINVAL, "there is no sequence %d", seq);
  if (len < 0 || len > g->book.seqs[(size_t)seq].len) return fail(CAKE_B200_ESTATE, "sequence %d has %d positions, not %d", seq, g->book.seqs[(size_t)seq].len, len);
  g->book.cut(seq, len);
  for (auto &l : g->len) l[(size_t)seq] = std::min(l[(size_t)seq], len);
  return CAKE_B200_OK;
}
extern "C" int cake_b200_pages_drop(cake_b200_pages *g, int seq) {
  if (!g) return fail(CAKE_B200_EINVAL, "null argument");
  if (!g->book.has(seq)) return fail(CAKE_B200_EINVAL, "there is no sequence %d", seq);
  g->book.drop(seq);
  return CAKE_B200_OK;
}
extern "C" int cake_b200_pages_len(const cake_b200_pages *g, int seq) { return !g || !g->book.has(seq) ? -1 : g->book.seqs[(size_t)seq].len; }
extern "C" int cake_b200_pages_available(const cake_b200_pages *g) { return g ? (int)g->book.free_pages.size() : -1; }

static size_t pages_plan_bytes(const cake_b200_pages *g) {
  const cake_b200_config &f = g->ctx->cfg;
  const int sms = g->ctx->sm_count;
  return sizeof(pg::PlanHead) + (size_t)pg::few_ctas(f.head_dim, sms) * (sizeof(pg::Worker) + sizeof(pg::Cut)) +
         pg::Book::most_items((long long)g->book.n_pages * g->book.page, g->book.max_seqs, f.n_heads / f.n_kv_heads, pg::room(f.head_dim, sms, f.n_kv_heads)) * sizeof(pg::Item) + (size_t)pg::room(f.head_dim, sms, f.n_kv_heads) * 4;
}
static int pages_plan_make(cake_b200_pages *g, cake_b200_pages::Plan *p) {   // on the ctx's stream of the moment
  cake_b200_ctx *c = g->ctx;
  const int n_kv = c->cfg.n_kv_heads, hd = c->cfg.head_dim, G = c->cfg.n_heads / n_kv, room = pg::room(hd, c->sm_count, n_kv);
  const size_t most = (size_t)pg::few_ctas(hd, c->sm_count);
  std::vector<pg::Worker> few;
  std::vector<pg::Cut> cuts;
  std::vector<pg::Item> many;
  pg::PlanHead h{};
  g->book.cut_few(p->win, n_kv, (int)most, &few, &cuts);
  h.W = (int)few.size();
  h.n_cuts = (int)cuts.size();
  h.parts = g->book.cut_many(p->win, G, room, &many);
  h.n_items = (int)many.size();
  if (h.n_items && !g->tiles_ws) {
    void *m = nullptr;
    CU(cudaMallocFromPoolAsync(&m, pg::tiles_floats(hd, c->sm_count, n_kv) * 4, c->pc_pool, c->stream));
    g->tiles_ws = (float *)m;
  }
  const size_t at_cuts = sizeof h + most * sizeof(pg::Worker), at_many = at_cuts + most * sizeof(pg::Cut);
  std::vector<int> heads;
  int tiles = 0;
  for (size_t i = 0; i < many.size(); i++) {
    tiles += many[i].part == 0;
    if (many[i].part == 0 && many[i].parts > 1) heads.push_back((int)i);
  }
  h.n_cut_tiles = (int)heads.size();
  p->most_items = tiles ? tiles + 2 * room : 0;   // (of any lengths, as cut_many has it; their heads begin behind that many)
  p->most_cut_tiles = tiles ? std::min(tiles, room) : 0;
  const size_t at_heads = at_many + (size_t)p->most_items * sizeof(pg::Item);
  std::vector<char> blob(!many.empty() ? at_heads + heads.size() * 4 : at_cuts + cuts.size() * sizeof(pg::Cut));
  memcpy(blob.data(), &h, sizeof h);
  if (!few.empty()) memcpy(blob.data() + sizeof h, few.data(), few.size() * sizeof(pg::Worker));
  if (!cuts.empty()) memcpy(blob.data() + at_cuts, cuts.data(), cuts.size() * sizeof(pg::Cut));
  if (!many.empty()) memcpy(blob.data() + at_many, many.data(), many.size() * sizeof(pg::Item));
  if (!heads.empty()) memcpy(blob.data() + at_heads, heads.data(), heads.size() * 4);
  RC(pages_upload(c, p->dev, blob.data(), blob.size()));
  p->longest = p->tiles = 0;
  for (int i = 0; i < g->book.n_few; i++) {
    const int t = pg::tiles_of(g->book.step[(size_t)i], p->win);
    p->longest = std::max(p->longest, t);
    p->tiles += t * n_kv;
  }
  p->n_cuts = h.n_cuts;
  p->n_items = h.n_items;
  p->n_cut_tiles = h.n_cut_tiles;
  p->step = g->steps;
  return CAKE_B200_OK;
}
static int pages_plan(cake_b200_pages *g, const pg::Window &win, bool capturing, const cake_b200_pages::Plan **out) {
  cake_b200_ctx *c = g->ctx;
  cake_b200_pages::Plan *p = nullptr;
  for (auto &x : g->plans)
    if (x.dev && x.win.w == win.w && x.win.by_call == win.by_call) p = &x;
  if (!p) {
    RC(no_capture(c->stream, "the plan of attention with this window"));
    for (auto &x : g->plans)
      if (!x.kept && (!p || x.used < p->used)) p = &x;
    if (!p) return fail(CAKE_B200_EINVAL, "captured calls have used %d windows: there is room for no other", (int)(sizeof g->plans / sizeof g->plans[0]));
    if (!p->dev) {
      void *m = nullptr;
      CU(cudaMallocFromPoolAsync(&m, pages_plan_bytes(g), c->pc_pool, c->stream));
      p->dev = (char *)m;
    }
    p->win = win;
    p->step = 0;
  }
  p->used = ++g->calls;
  if (p->step != g->steps) {
    RC(no_capture(c->stream, "this step's plan of attention"));
    RC(with_memory([&]() -> int { return pages_plan_make(g, p); }));
  }
  p->kept = p->kept || capturing;
  *out = p;
  return CAKE_B200_OK;
}

extern "C" int cake_b200_pages_step(cake_b200_pages *g, const int *seqs, const int *counts, int n, void *stream) {
  RC(pages_call(g, "pages_step"));
  if (!seqs || !counts || n < 1) return fail(CAKE_B200_EINVAL, "null/empty argument");
  if (n > g->book.max_seqs) return fail(CAKE_B200_EINVAL, "a step of %d sequences, the cache has %d", n, g->book.max_seqs);
  cake_b200_ctx *c = g->ctx;
  const OnDevice dev(g->device);
  if (is_capturing(stream ? (cudaStream_t)stream : c->stream)) return fail(CAKE_B200_ESTATE, "a step is planned outside captures; its calls may be captured");
  long long pages = 0;   // that the step may take, at most
  for (int i = 0; i < n; i++) pages += std::max(counts[i], 0) / g->book.page + 1;
  RC(pages_room(c, sizeof(pg::StepHead) + (size_t)n * sizeof(pg::SeqRow) + (size_t)std::min<long long>(pages, (long long)g->book.free_pages.size()) * 8));
  return with_memory([&]() -> int {
    pg::Book &k = g->book;
    int i = 0;
    switch (k.plan(seqs, counts, n, c->cfg.n_heads / c->cfg.n_kv_heads, &i)) {
      case pg::Book::OK: break;
      case pg::Book::NOT_LIVE: return fail(CAKE_B200_EINVAL, "there is no sequence %d", seqs[i]);
      case pg::Book::TWICE: return fail(CAKE_B200_EINVAL, "sequence %d is twice in the step", seqs[i]);
      case pg::Book::COUNT: return fail(CAKE_B200_EINVAL, "sequence %d brings %d rows", seqs[i], counts[i]);
      case pg::Book::TOO_LONG: return fail(CAKE_B200_ESTATE, "sequence %d: %d + %d positions exceed max_seq %d", seqs[i], k.seqs[(size_t)seqs[i]].len, counts[i], k.max_seq);
      case pg::Book::NO_PAGES: return fail(CAKE_B200_ENOMEM, "the step needs more pages than the %d that are free", (int)k.free_pages.size());
    }
    auto send = [&]() -> int {
      const size_t at = sizeof(pg::StepHead) + (size_t)n * sizeof(pg::SeqRow), bytes = at + k.updates.size() * 4;
      std::vector<char> &blob = g->blob;   // (has the room)
      blob.assign(bytes, 0);
      pg::StepHead h{};
      h.shape = k.shape; h.n_seqs = n; h.n_rows = k.n_rows; h.n_updates = (int)k.updates.size() / 2;
      memcpy(blob.data(), &h, sizeof h);
      memcpy(blob.data() + sizeof h, k.step.data(), k.step.size() * sizeof(pg::SeqRow));
      if (!k.updates.empty()) memcpy(blob.data() + at, k.updates.data(), k.updates.size() * 4);
      RC(pages_upload(c, g->step, blob.data(), bytes));
      int most = 1;
      for (int j = 0; j < n; j++) most = std::max(most, counts[j]);
      CU((cudaError_t)pg::spread(c->stream, g->step, n, h.n_updates, most, g->table, g->rows, launch_counter(c)));
      g->steps++;
      for (auto &p : g->plans)
        if (p.kept) RC(with_memory([&]() -> int { return pages_plan_make(g, &p); }));
      return CAKE_B200_OK;
    };
    const int rc = on_stream(c, stream, [&]() -> int {
      const int rc = send();
      if (rc != CAKE_B200_OK) (void)cudaMemsetAsync(g->step, 0, sizeof(pg::StepHead), c->stream);   // none for a replayed graph either: its calls would follow an older one's plan
      return rc;
    });
    if (rc != CAKE_B200_OK)   // no step, and its sequences are as they were
      for (int j = 0; j < n; j++) k.cut(seqs[j], k.seqs[(size_t)seqs[j]].len - counts[j]);
    return rc;
  });
}

static int pages_block(cake_b200_pages *g, int block_idx, const char *what, bool wants_step) {
  RC(pages_call(g, what));
  if (block_idx < 0 || block_idx >= (int)g->pool.size()) return fail(CAKE_B200_EINVAL, "block_idx %d out of range", block_idx);
  if (wants_step && g->book.step.empty()) return fail(CAKE_B200_ESTATE, "%s: there is no step (or one of its sequences was cut or dropped)", what);
  return CAKE_B200_OK;
}
static int pages_ensure(cake_b200_pages *g, int l) {
  if (g->pool[(size_t)l]) return CAKE_B200_OK;
  cake_b200_ctx *c = g->ctx;
  RC(no_capture(c->stream, "a block's pages"));
  const size_t bytes = (size_t)g->book.n_pages * (g->page_bytes() + (size_t)c->cfg.n_kv_heads * 4);
  void *p = nullptr;
  CU(cudaMallocFromPoolAsync(&p, bytes, c->pc_pool, c->stream));
  const cudaError_t e = cudaMemsetAsync(p, 0, bytes, c->stream);
  if (e != cudaSuccess) { (void)cudaFreeAsync(p, c->stream); return fail(CAKE_B200_ECUDA, "pages: %s", cudaGetErrorString(e)); }
  g->pool[(size_t)l] = p;
  return CAKE_B200_OK;
}
static pg::Pool pages_pool(const cake_b200_pages *g, int l) {
  const cake_b200_config &f = g->ctx->cfg;
  int log2 = 0;
  while (1 << log2 < g->book.page) log2++;
  char *p = (char *)g->pool[(size_t)l];
  return pg::Pool{p, (uint32_t *)(p + (size_t)g->book.n_pages * g->page_bytes()), g->table, g->step, g->book.shape, g->bad, f.n_kv_heads, f.head_dim, log2, g->book.per_seq};
}
// the rows that the step's follow are there (append), and its own (attend, read)
static int pages_written(const cake_b200_pages *g, int l, bool own) {
  if (g->in_graph[(size_t)l]) return CAKE_B200_OK;
  for (const pg::SeqRow &s : g->book.step) {
    const int have = g->len[(size_t)l][(size_t)s.slot], need = own ? s.pos0 + s.count : s.pos0;
    if (have < need) return fail(CAKE_B200_ESTATE, "block %d has %d positions of sequence %d, not %d", l, have, s.slot, need);
  }
  return CAKE_B200_OK;
}
static int pages_append_on(cake_b200_pages *g, int l, const pg::Append &a) {   // on the ctx's stream of the moment
  cake_b200_ctx *c = g->ctx;
  CU((cudaError_t)pg::append(c->stream, c->cfg.dtype, pages_pool(g, l), a, c->sm_count, launch_counter(c)));
  if (is_capturing(c->stream)) g->in_graph[(size_t)l] = 1;
  for (const pg::SeqRow &s : g->book.step) g->len[(size_t)l][(size_t)s.slot] = s.pos0 + s.count;
  return CAKE_B200_OK;
}
static int pages_attend_on(cake_b200_pages *g, int l, const void *q, size_t q_tok, void *out, const pg::Window &win, float scale) {
  cake_b200_ctx *c = g->ctx;
  const cake_b200_pages::Plan *plan = nullptr;
  const bool capturing = is_capturing(c->stream);
  RC(pages_plan(g, win, capturing, &plan));
  int cols = 0;
  // a captured call's lengths may become any: up to what the cache and the window allow
  const int most_seen = win.w > 0 && !win.by_call ? (int)std::min<long long>(g->book.max_seq, (long long)win.w + pg::TOKEN_COLS + pg::TILE) : g->book.max_seq;
  const int longest = capturing ? (most_seen + pg::TILE - 1) / pg::TILE + 1 : plan->longest;
  const int most_cuts = std::min(g->book.n_few * c->cfg.n_kv_heads, pg::few_ctas(c->cfg.head_dim, c->sm_count));
  for (int i = 0; i < g->book.n_few; i++) cols = std::max(cols, g->book.step[(size_t)i].count * (c->cfg.n_heads / c->cfg.n_kv_heads));
  const pg::Attend a{q, (long long)q_tok, out, (const pg::SeqRow *)(g->step + 1), c->cfg.n_heads, scale, win, (const pg::PlanHead *)plan->dev, g->book.n_few, cols,
                     longest, capturing ? 0 : plan->tiles, capturing ? most_cuts : plan->n_cuts, capturing ? plan->most_items : plan->n_items, plan->most_items, capturing ? plan->most_cut_tiles : plan->n_cut_tiles, c->wait_err};
  CU((cudaError_t)pg::attend(c->stream, c->cfg.dtype, pages_pool(g, l), a, pg::Scratch{g->few_ws, g->tiles_ws, c->sm_count, &c->pg_clusters}, launch_counter(c)));
  return CAKE_B200_OK;
}
// rows of `row` entries of `es` bytes, `tok` entries from one to the next: whether two sets of them, from their first byte to their last, share any
struct RowsAt { const void *at; size_t rows, tok, row; };
static bool on_another(const RowsAt &a, const RowsAt &b, size_t es) {
  const char *pa = (const char *)a.at, *pb = (const char *)b.at;
  return pa < pb + ((b.rows - 1) * b.tok + b.row) * es && pb < pa + ((a.rows - 1) * a.tok + a.row) * es;
}
extern "C" int cake_b200_pages_append(cake_b200_pages *g, int block_idx, const void *q_dev, size_t q_tok, const void *k_dev, size_t k_tok, const void *v_dev,
                                      size_t v_tok, void *q_out, int rotate, void *stream) {
  RC(pages_block(g, block_idx, "pages_append", true));
  const OnDevice dev(g->device);
  if (!k_dev || !v_dev || !q_dev != !q_out) return fail(CAKE_B200_EINVAL, "null argument");
  if (unaligned(k_dev, k_tok) || unaligned(v_dev, v_tok) || unaligned(q_dev, q_tok) || unaligned(q_out))
    return fail(CAKE_B200_EINVAL, "pages_append takes rows on 16-byte boundaries (strides of a multiple of 8 entries)");
  cake_b200_ctx *c = g->ctx;
  const cake_b200_config &f = c->cfg;
  if (q_out) {   // a warp has one row: another row's may not have been read yet
    const size_t rows = (size_t)g->book.n_rows, row = (size_t)f.n_heads * f.head_dim, kv = (size_t)f.n_kv_heads * f.head_dim;
    const RowsAt out{q_out, rows, row, row};
    const bool in_place = q_out == q_dev && (q_tok == row || rows == 1);
    if ((!in_place && on_another(out, RowsAt{q_dev, rows, q_tok, row}, c->es)) || on_another(out, RowsAt{k_dev, rows, k_tok, kv}, c->es) ||
        on_another(out, RowsAt{v_dev, rows, v_tok, kv}, c->es))
      return fail(CAKE_B200_EINVAL, "pages_append's q_out lies beside q, k and v, or on a contiguous q");
  }
  RC(pages_written(g, block_idx, false));
  if (!g->pool[(size_t)block_idx] && stream) RC(no_capture((cudaStream_t)stream, "a block's pages"));
  return on_stream(c, stream, [&]() -> int {
    RC(pages_ensure(g, block_idx));
    pg::Append a{};
    a.rows = g->rows; a.q = q_dev; a.k = k_dev; a.v = v_dev; a.q_out = q_out; a.q_tok = (long long)q_tok; a.k_tok = (long long)k_tok; a.v_tok = (long long)v_tok;
    a.out_tok = (long long)f.n_heads * f.head_dim;
    if (rotate) { a.cos_t = g->cos_t; a.sin_t = g->sin_t; a.rot = g->rot; }
    a.n_rows = g->book.n_rows; a.n_q = q_dev ? f.n_heads : 0;
    return pages_append_on(g, block_idx, a);
  });
}
extern "C" int cake_b200_pages_attend(cake_b200_pages *g, int block_idx, const void *q_dev, size_t q_tok, void *out_dev, int window, float scale, void *stream) {
  RC(pages_block(g, block_idx, "pages_attend", true));
  const OnDevice dev(g->device);
  if (!q_dev || !out_dev) return fail(CAKE_B200_EINVAL, "null argument");
  if (unaligned(q_dev, q_tok) || unaligned(out_dev)) return fail(CAKE_B200_EINVAL, "pages_attend takes rows on 16-byte boundaries (strides of a multiple of 8 entries)");
  const cake_b200_config &f = g->ctx->cfg;
  const size_t row = (size_t)f.n_heads * f.head_dim, rows = (size_t)g->book.n_rows;
  if (on_another(RowsAt{out_dev, rows, row, row}, RowsAt{q_dev, rows, q_tok, row}, g->ctx->es))
    return fail(CAKE_B200_EINVAL, "pages_attend's out lies beside q, not on it");
  if (window < 0 || !(scale >= 0.f && scale <= 2e38f)) return fail(CAKE_B200_EINVAL, "window %d or scale %g out of range", window, (double)scale);
  if (!g->pool[(size_t)block_idx]) return fail(CAKE_B200_ESTATE, "block %d has no rows", block_idx);
  RC(pages_written(g, block_idx, true));
  return on_stream(g->ctx, stream, [&]() -> int {
    return pages_attend_on(g, block_idx, q_dev, q_tok, out_dev, pg::Window{window, false}, scale > 0.f ? scale : (float)(1.0 / sqrt((double)g->ctx->cfg.head_dim)));
  });
}
extern "C" int cake_b200_pages_read(cake_b200_pages *g, int block_idx, int seq, int first, int n, void *k_dev, void *v_dev, void *stream) {
  RC(pages_block(g, block_idx, "pages_read", seq < 0));
  const OnDevice dev(g->device);
  if (!k_dev && !v_dev) return fail(CAKE_B200_EINVAL, "null argument");
  if (unaligned(k_dev) || unaligned(v_dev)) return fail(CAKE_B200_EINVAL, "pages_read writes to 16-byte boundaries");
  if (!g->pool[(size_t)block_idx]) return fail(CAKE_B200_ESTATE, "block %d has no rows", block_idx);
  pg::Read a{nullptr, seq, first, n, k_dev, v_dev};
  if (seq < 0) {
    if (n != 0 && n != g->book.n_rows) return fail(CAKE_B200_EINVAL, "pages_read: room for %d rows, the step has %d", n, g->book.n_rows);
    RC(pages_written(g, block_idx, true));
    a = pg::Read{g->rows, 0, 0, g->book.n_rows, k_dev, v_dev};
  } else {
    if (!g->book.has(seq)) return fail(CAKE_B200_EINVAL, "there is no sequence %d", seq);
    if (is_capturing(stream ? (cudaStream_t)stream : g->ctx->stream))   // (when it is replayed, nothing says whose pages the table names in that row)
      return fail(CAKE_B200_ESTATE, "positions of one sequence are read outside captures");
    const int have = g->in_graph[(size_t)block_idx] ? g->book.seqs[(size_t)seq].len : g->len[(size_t)block_idx][(size_t)seq];
    if (first < 0 || n < 1 || (long long)first + n > have)
      return fail(CAKE_B200_ESTATE, "block %d, sequence %d: positions %d .. + %d are not within %d", block_idx, seq, first, n, have);
  }
  return on_stream(g->ctx, stream, [&]() -> int {
    CU((cudaError_t)pg::read(g->ctx->stream, pages_pool(g, block_idx), a, g->ctx->sm_count, launch_counter(g->ctx)));
    return CAKE_B200_OK;
  });
}
// a layer's attention in a step of rows in pages: qkv [rows, heads + 2 kv heads, hd] as the projection left them (q is normed and rotated in place) -> y
static int pages_layer(cake_b200_ctx *c, const cake_b200_block *b, cake_b200_pages *g, int l, void *qkv, const void *qn, const void *kn, void *y) {
  const cake_b200_config &f = c->cfg;
  RC(pages_ensure(g, l));
  char *p = (char *)qkv;
  pg::Append a{};
  a.rows = g->rows; a.q = p; a.q_out = p;
  a.k = p + (size_t)f.n_heads * f.head_dim * c->es;
  a.v = p + (size_t)(f.n_heads + f.n_kv_heads) * f.head_dim * c->es;
  a.q_tok = a.k_tok = a.v_tok = a.out_tok = c->nqkv;
  a.q_norm = qn; a.k_norm = kn; a.eps = f.rms_eps;
  if (b->use_rope) { a.cos_t = g->cos_t; a.sin_t = g->sin_t; a.rot = g->rot; }
  a.n_rows = g->book.n_rows; a.n_q = f.n_heads; a.as_blocks = true;
  RC(pages_append_on(g, l, a));
  return pages_attend_on(g, l, qkv, c->nqkv, y, pg::Window{b->window >= 0 ? b->window : f.sliding_window, true}, (float)(1.0 / sqrt((double)f.head_dim)));
}
