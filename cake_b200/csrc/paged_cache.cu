// paged_cache.cu — kernels of the cache in pages (format and interface: paged_cache.cuh)
#include "paged_cache.cuh"
#include "paged_few.cuh"
#include "paged_tiles.cuh"

#include <algorithm>
#include <type_traits>

namespace cake {
namespace pg {

template <typename... KArgs, typename... Args>
static int launch(cudaStream_t s, uint64_t *launches, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
  if (e == cudaSuccess) ++*launches;
  return (int)e;
}
template <typename T> struct Tag { typedef T type; };
template <typename F> static int by_type(int dtype, F &&f) { return dtype == 1 ? f(Tag<__half>{}) : f(Tag<__nv_bfloat16>{}); }

// ------------------------------------------------------------------------------------------ a step's sequences and rows
__global__ void __launch_bounds__(256) spread_kernel(const StepHead *step, int n_seqs, int *table, int2 *rows) {
  const SeqRow *seqs = reinterpret_cast<const SeqRow *>(step + 1);
  const int at = blockIdx.y * 256 + threadIdx.x, by = gridDim.y * 256;
  if ((int)blockIdx.x == n_seqs) {
    const int2 *u = reinterpret_cast<const int2 *>(seqs + n_seqs);
    for (int i = at; i < step->n_updates; i += by) table[u[i].x] = u[i].y;
    return;
  }
  const SeqRow s = seqs[blockIdx.x];
  for (int i = at; i < s.count; i += by) rows[s.row0 + i] = make_int2(s.slot, s.pos0 + i);
}
int spread(cudaStream_t s, const StepHead *step, int n_seqs, int n_updates, int most_rows, int *table, int2 *rows, uint64_t *launches) {
  const int most = std::max(most_rows, n_updates);
  // Attention reads the step, its plan and the table in front of its wait for the launch before it.  Between this kernel and the first attention over a step with any
  // window lies the copy of that window's plan (made by that call, or with the step where captured calls read it), and no launch behind a copy starts early: all
  // that is in front of the copy is there for it and for what starts behind it.  Appends and reads look behind their wait.
  spread_kernel<<<dim3((unsigned)n_seqs + 1, (unsigned)std::min(64, (most + 255) / 256)), 256, 0, s>>>(step, n_seqs, table, rows);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) ++*launches;
  return (int)e;
}

// ------------------------------------------------------------------------------------------ rows into the pages
// Bound by memory: what comes in goes out.  A lane has two 16-byte chunks of a head, those of a rotation's pairs (entries e .. e + 7 and e + rot / 2 ..) or, behind the
// rotated entries, two neighbours: no exchange between lanes.  hd / 16 lanes a head, 512 / hd heads of a token a warp at once, several times that asked for
// before the first is worked on; where the tokens alone do not fill the chip, a warp has a part of a token's heads.  The row of the tables is read once a warp.
// 12314 rows of 48 heads of 128: a chunk a lane, its pair's other one by 8 exchanges, 73 us with 2 loads in flight and 66 with 4; so 50.
// Norm and rotation in fp32 and one rounding; in a block's step (BLOCKS) they are rounded where the blocks' other paths round them (the normed entries, the
// products), so that its rows are those that any other cache would hold: logits of three layers within 4 units in the last place of the oracle, else up to 6.
template <typename T> __device__ __forceinline__ bool not_finite(uint32_t w) {
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w >> 16 & e) == e;
}
template <typename T> __device__ __forceinline__ bool not_finite(const uint4 &w) { return not_finite<T>(w.x) || not_finite<T>(w.y) || not_finite<T>(w.z) || not_finite<T>(w.w); }
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2x<T>(x[0], x[1]), pack2x<T>(x[2], x[3]), pack2x<T>(x[4], x[5]), pack2x<T>(x[6], x[7]));
}
template <typename T, int HD, bool BLOCKS>
__global__ void __launch_bounds__(128) append_kernel(const Pool p, const Append a, int parts) {
  pdl_launch_dependents();
  constexpr int LPH = HD / 16, AT_ONCE = 32 / LPH, U = 4;   // lanes of a head; heads of a warp at once; such groups asked for at once
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pair = lane % LPH, sub = lane / LPH;
  const int row = blockIdx.x * 4 + warp, heads = a.n_q + 2 * p.n_kv;
  const int h8 = a.cos_t ? a.rot >> 4 : 0;   // chunks of the pairs' first entries
  const bool turns = pair < h8;
  const int c0 = turns ? pair : 2 * h8 + 2 * (pair - h8), c1 = turns ? pair + h8 : c0 + 1;
  pdl_wait();
  if (!same_step(p) || row >= a.n_rows) return;
  const int2 at = __ldg(a.rows + row);
  const int page = page_of(p, at.x, at.y), r = at.y & ((1 << p.page_log2) - 1);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const size_t o = (size_t)at.y * (8 * h8) + 8 * pair + i;
    const float4 x = turns ? __ldg(reinterpret_cast<const float4 *>(a.cos_t + o)) : make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 y = turns ? __ldg(reinterpret_cast<const float4 *>(a.sin_t + o)) : make_float4(0.f, 0.f, 0.f, 0.f);
    cs[i] = x.x; cs[i + 1] = x.y; cs[i + 2] = x.z; cs[i + 3] = x.w;
    sn[i] = y.x; sn[i + 1] = y.y; sn[i + 2] = y.z; sn[i + 3] = y.w;
  }
  const T *q = reinterpret_cast<const T *>(a.q) + (size_t)row * a.q_tok, *k = reinterpret_cast<const T *>(a.k) + (size_t)row * a.k_tok,
          *v = reinterpret_cast<const T *>(a.v) + (size_t)row * a.v_tok;
  for (int g0 = blockIdx.y; g0 * AT_ONCE < heads; g0 += U * parts) {
    uint4 in[U][2];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int head = (g0 + u * parts) * AT_ONCE + sub;
      if (head < heads) {
        const T *src = head < a.n_q ? q + (size_t)head * HD : head < a.n_q + p.n_kv ? k + (size_t)(head - a.n_q) * HD : v + (size_t)(head - a.n_q - p.n_kv) * HD;
        in[u][0] = *reinterpret_cast<const uint4 *>(src + 8 * c0);
        in[u][1] = *reinterpret_cast<const uint4 *>(src + 8 * c1);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int head = (g0 + u * parts) * AT_ONCE + sub;
      const bool there = head < heads, is_q = head < a.n_q, is_v = head >= a.n_q + p.n_kv;
      const T *nw = reinterpret_cast<const T *>(is_q ? a.q_norm : a.k_norm);
      float inv = 0.f;
      if (BLOCKS && (a.q_norm || a.k_norm)) {   // (the same for all lanes, as the exchanges have to be)
        float x[8], y[8], ss = 0.f;
        unpack8<T>(in[u][0], x);
        unpack8<T>(in[u][1], y);
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
      }
      if (!there) continue;
      if (is_v) {
        const int h = head - a.n_q - p.n_kv;
        char *to = rows_of(p, page, h, 1);
        *reinterpret_cast<uint4 *>(to + chunk_at(HD, r, c0)) = in[u][0];
        *reinterpret_cast<uint4 *>(to + chunk_at(HD, r, c1)) = in[u][1];
        if (not_finite<T>(in[u][0]) || not_finite<T>(in[u][1])) p.marks[(size_t)page * p.n_kv + h] = 1u;
        continue;
      }
      if (turns || (BLOCKS && nw)) {
        float x[8], y[8];
        unpack8<T>(in[u][0], x);
        unpack8<T>(in[u][1], y);
        if (BLOCKS && nw) {
          float g[8];
          unpack8<T>(*reinterpret_cast<const uint4 *>(nw + 8 * c0), g);
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = rnd<T>(x[i] * inv * g[i]);
          unpack8<T>(*reinterpret_cast<const uint4 *>(nw + 8 * c1), g);
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = rnd<T>(y[i] * inv * g[i]);
        }
        if (turns)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float s = x[i], t = y[i];
            x[i] = BLOCKS ? rnd<T>(s * cs[i]) - rnd<T>(t * sn[i]) : s * cs[i] - t * sn[i];
            y[i] = BLOCKS ? rnd<T>(t * cs[i]) + rnd<T>(s * sn[i]) : t * cs[i] + s * sn[i];
          }
        in[u][0] = pack8<T>(x);
        in[u][1] = pack8<T>(y);
      }
      if (is_q) {
        T *to = reinterpret_cast<T *>(a.q_out) + (size_t)row * a.out_tok + (size_t)head * HD;
        *reinterpret_cast<uint4 *>(to + 8 * c0) = in[u][0];
        *reinterpret_cast<uint4 *>(to + 8 * c1) = in[u][1];
      } else {
        char *to = rows_of(p, page, head - a.n_q, 0);
        *reinterpret_cast<uint4 *>(to + chunk_at(HD, r, c0)) = in[u][0];
        *reinterpret_cast<uint4 *>(to + chunk_at(HD, r, c1)) = in[u][1];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ rows out of the pages
__global__ void __launch_bounds__(256) read_kernel(const Pool p, const Read a) {
  pdl_launch_dependents();
  const int cph = p.hd >> 3;
  const size_t n = (size_t)a.n * p.n_kv * cph;
  pdl_wait();
  if (a.rows && !same_step(p)) return;
  for (size_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
    const int c = (int)(i % cph), h = (int)(i / cph % p.n_kv), row = (int)(i / cph / p.n_kv);
    const int2 at = a.rows ? __ldg(a.rows + row) : make_int2(a.slot, a.first + row);
    const int page = page_of(p, at.x, at.y), r = at.y & ((1 << p.page_log2) - 1);
    if (a.k) reinterpret_cast<uint4 *>(a.k)[i] = *reinterpret_cast<const uint4 *>(rows_of(p, page, h, 0) + chunk_at(p.hd, r, c));
    if (a.v) reinterpret_cast<uint4 *>(a.v)[i] = *reinterpret_cast<const uint4 *>(rows_of(p, page, h, 1) + chunk_at(p.hd, r, c));
  }
}
int read(cudaStream_t s, const Pool &p, const Read &a, int sms, uint64_t *launches) {
  const size_t n = (size_t)a.n * p.n_kv * (p.hd >> 3);
  return launch(s, launches, read_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, (size_t)sms * 32)), dim3(256), 0, 1, p, a);
}

// ------------------------------------------------------------------------------------------ attention
int few_ctas(int hd, int sms) { return (hd == 256 ? 1 : 2) * sms; }
int room(int hd, int sms, int n_kv) { return std::max(1, (hd == 256 ? 1 : 2) * sms / n_kv); }
size_t tiles_floats(int hd, int sms, int n_kv) { return (size_t)2 * room(hd, sms, n_kv) * n_kv * TILE_ROWS * (hd + 2); }
size_t few_floats(int hd, int sms) { return (size_t)2 * few_ctas(hd, sms) * TOKEN_COLS * (hd + 2); }
// f(T, HD): the instances of a kind of cache
template <typename F> static int by_kind(int dtype, int hd, F &&f) {
  return by_type(dtype, [&](auto t) {
    switch (hd) {
      case 64: return f(t, std::integral_constant<int, 64>{});
      case 128: return f(t, std::integral_constant<int, 128>{});
      default: return f(t, std::integral_constant<int, 256>{});
    }
  });
}
int append(cudaStream_t s, int dtype, const Pool &p, const Append &a, int sms, uint64_t *launches) {
  const int at_once = 512 / p.hd, groups = (a.n_q + 2 * p.n_kv + at_once - 1) / at_once;
  int parts = 1;
  while (parts < groups && (long)a.n_rows * parts < 16l * sms) parts++;
  return by_kind(dtype, p.hd, [&](auto t, auto h) {
    typedef typename decltype(t)::type T;
    constexpr int HD = decltype(h)::value;
    return launch(s, launches, a.as_blocks ? append_kernel<T, HD, true> : append_kernel<T, HD, false>, dim3((unsigned)((a.n_rows + 3) / 4), (unsigned)parts), dim3(128), 0, 1, p, a, parts);
  });
}
int prepare(int dtype, int hd, Clusters *out) {
  return by_kind(dtype, hd, [&](auto t, auto h) {
    typedef typename decltype(t)::type T;
    constexpr int HD = decltype(h)::value;
    cudaError_t e = cudaSuccess;
    auto few = [&](auto n) {
      constexpr int NT = decltype(n)::value, SMEM = FewCfg<HD, NT>::SMEM;
      for (auto k : {few_kernel<T, HD, NT, false>, few_kernel<T, HD, NT, true>})
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
      for (int i = 0; i < 4 && e == cudaSuccess; i++) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 1u << i;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(1u << i);
        cfg.blockDim = dim3(FEW_THREADS);
        cfg.dynamicSmemBytes = SMEM;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&out->most[NT - 1][i], few_kernel<T, HD, NT, true>, &cfg);
      }
    };
    few(std::integral_constant<int, 1>{});
    few(std::integral_constant<int, 2>{});
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tiles_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<HD>::SMEM);
    return (int)e;
  });
}
// A cluster's CTAs for each run, or 0: shares.  One launch without a list, whose sums meet in shared memory, is the faster way where all clusters are on the chip
// at once and no CTA has many more tiles than an equal share.  Clusters / shares in us (shares in a graph; alone their second launch costs 2 more of the
// host's), sequences x positions:  8 key heads of 128, 1 x 500 7.1 (the host's) / 5.7, 1 x 4000 9.7 / 12.1, 4 x 1000 7.1 / 9.8, 9 x 500 7.4 / 8.8, 9 x 2000 (16 tiles a CTA,
// an equal share 8) 15.0 / 13.9, 16 x 1000 10.7 / 11.7, 32 x 1000 23.5 / 27.3, 32 x 4000 81 / 84;  2 of 64, 1 x 4000 8.4 / 7.1, 32 x 1000 7.1 / 8.2, 64 x 4000 25 / 28;  4 of 256,
// 2 x 2000 8.0 / 12.4, 4 x 4000 (16 tiles, 7) 15.9 / 14.8, 16 x 1000 11.1 / 12.6.  A captured call follows the same rule by the longest run that the cache allows: in a
// graph 1 x 4000 of 2 x 64 takes 7.5 in clusters and 7.1 in shares, and 1 x 998 (8 of 128) 4.4 in a cache of up to some 4000 positions and 6.0, in shares, in larger ones.
constexpr int CLUSTER_TILES = 8;
static int cluster_of(int runs, int longest, int tiles, int ctas, const int (&most)[4]) {
  int best = 0;
  for (int k = 0; k < 4 && 1 << k < 2 * longest; k++) {
    const int mine = (longest + (1 << k) - 1) >> k;
    if (runs <= most[k] && (mine <= CLUSTER_TILES || mine <= 1.5 * tiles / ctas)) best = 1 << k;
  }
  return best;
}
int attend(cudaStream_t s, int dtype, const Pool &p, const Attend &a, const Scratch &w, uint64_t *launches) {
  const int G = a.n_heads / p.n_kv;
  const float scale_log2 = a.scale * 1.4426950408889634f;
  if (a.n_few) {
    const Few f{p, a.plan, a.seqs, a.q, a.q_tok, a.out, w.few_ws, a.n_heads, G, a.win, scale_log2, a.err, a.n_items ? 1 : 0};
    const Cut *cuts = reinterpret_cast<const Cut *>(reinterpret_cast<const Worker *>(a.plan + 1) + few_ctas(p.hd, w.sms));
    const int cluster = cluster_of(a.n_few * p.n_kv, a.longest, a.tiles, few_ctas(p.hd, w.sms), w.clusters->most[a.few_cols <= 8 ? 0 : 1]);
    const int e = by_kind(dtype, p.hd, [&](auto t, auto h) {
      typedef typename decltype(t)::type T;
      constexpr int HD = decltype(h)::value;
      auto both = [&](auto n) {
        constexpr int NT = decltype(n)::value;
        if (cluster)
          return launch(s, launches, few_kernel<T, HD, NT, true>, dim3((unsigned)(a.n_few * p.n_kv * cluster)), dim3(FEW_THREADS), FewCfg<HD, NT>::SMEM, cluster, f);
        const int rc = launch(s, launches, few_kernel<T, HD, NT, false>, dim3((unsigned)few_ctas(HD, w.sms)), dim3(FEW_THREADS), FewCfg<HD, NT>::SMEM, 1, f);
        if (rc || !a.n_cuts) return rc;
        return launch(s, launches, few_join_kernel<T, HD, NT>, dim3((unsigned)a.n_cuts, (unsigned)a.few_cols), dim3(128), 0, 1, f, cuts);
      };
      return a.few_cols <= 8 ? both(std::integral_constant<int, 1>{}) : both(std::integral_constant<int, 2>{});
    });
    if (e) return e;
  }
  if (!a.n_items) return 0;
  const Item *items = reinterpret_cast<const Item *>(reinterpret_cast<const char *>(a.plan + 1) + (size_t)few_ctas(p.hd, w.sms) * (sizeof(Worker) + sizeof(Cut)));
  const Tiles t8{p, a.plan, items, a.q, a.q_tok, a.out, w.tiles_ws, a.n_heads, G, TILE_ROWS / G, a.win, scale_log2, 8.f, a.err, a.n_few ? 1 : 0};
  return by_kind(dtype, p.hd, [&](auto t, auto h) {
    typedef typename decltype(t)::type T;
    constexpr int HD = decltype(h)::value;
    const int e = launch(s, launches, tiles_kernel<T, HD>, dim3((unsigned)(a.n_items * p.n_kv)), dim3(FT_THREADS), TileCfg<HD>::SMEM, 1, t8);
    if (e || !a.n_cut_tiles) return e;
    return launch(s, launches, join_kernel<T, HD>, dim3((unsigned)(a.n_cut_tiles * p.n_kv), HD / 8), dim3(128), 0, 1, t8, reinterpret_cast<const int *>(items + a.most_items));
  });
}

}  // namespace pg
}  // namespace cake
