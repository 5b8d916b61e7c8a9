// paged_few.cuh — attention of a few rows a sequence over a cache in pages (tokens of a decode step; up to 16 query rows a key head)
//
// Bound by memory: every key and value is read once, 4 hd bytes a position and key head, for 4 operations an entry and query head.  The line of all
// (sequence, key head, tile of 64 positions) is cut into equal shares, one a CTA (paged_plan.hpp, cut_few), so that sequences of any lengths fill the chip
// evenly; the parts of a run (a sequence's key head) that is cut are joined by a kernel of its own (the CTA that comes last, behind a fence, a ticket and a loop over
// the parts, took 4 to 9 us, others waiting for it).  Where the runs are few or alike, a cluster of CTAs has one and joins its parts itself (paged_cache.cu,
// cluster_of).  In a CTA a warp copies tiles into a ring of shared memory by bulk copies of whole pages (or of 64 rows of one), looking up the pages of
// up to 32 copies at once and ahead; four warps take 16 positions of a tile each and never wait for one another before the run's end.  One token at 131071
// positions, 8 key heads of 128: 89 us, 6.0 TB/s; 32 tokens to 8191: 60 us, 5.6 TB/s, of 6.55.
//
// A warp's products are S^T [16 positions, 8 query rows] = K Q^T and O^T [hd, 8 query rows] += V^T P^T on mma.sync m16n8k16: the positions take the operand's
// 16 rows, the query rows its 8 columns (twice 8 for more), so that a group of 4 or 8 heads wastes little, and the weights turn from S^T's layout to
// P^T's by movmatrix.  A tensor core of the fifth generation would take 128 rows; 8 are used, and memory is the bound.  Weights are two operands of D, hi + lo: 16 bits and more.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "paged_cache.cuh"

namespace cake {
namespace pg {

constexpr int FEW_WARPS = 4, FEW_THREADS = 32 * FEW_WARPS + 32;
template <int HD, int NT> struct FewCfg {
  static constexpr int STAGES = HD == 64 ? 6 : NT == 1 ? 3 : 2;   // (two CTAs an SM; the four warps' sums of 16 rows take the third one's room)
  static constexpr int ROWS_BYTES = TILE * HD * 2;          // keys, or values, of a tile
  static constexpr int COLS = 8 * NT;
  static constexpr int RED_BYTES = FEW_WARPS * COLS * HD * 4, ML_BYTES = FEW_WARPS * COLS * 8;
  static constexpr int SMEM = STAGES * 2 * ROWS_BYTES + RED_BYTES + ML_BYTES + STAGES * (16 + 4) + 16;
  static constexpr int CTAS = HD == 256 ? 1 : 2;
  static_assert(SMEM <= 227 * 1024 && CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory");
};
// whether this call is the present step's; a replayed call of another one does nothing
__device__ __forceinline__ bool same_step(const Pool &p) {
  if (__ldg(&p.step->shape) == p.shape) return true;
  if (threadIdx.x == 0) *p.bad = 1;
  return false;
}
__device__ __forceinline__ char *rows_of(const Pool &p, int page, int kvh, int which) {
  return p.pages + ((size_t)page * p.n_kv + kvh) * (rows_bytes(p.hd, 2) << p.page_log2) + (which ? rows_bytes(p.hd, 1) << p.page_log2 : (size_t)0);
}
__device__ __forceinline__ int page_of(const Pool &p, int slot, int pos) { return __ldg(p.table + (size_t)slot * p.per_seq + (pos >> p.page_log2)); }

// Weights of D = f16 are lifted by a power of two, so that those 2^-24 of the largest and below still count: 100000 of them may be a hundredth of the sum
template <typename T> constexpr float lift(int log2) { return std::is_same<T, __half>::value ? (float)log2 : 0.f; }
struct Few {
  Pool pool;
  const PlanHead *plan;
  const SeqRow *seqs;
  const void *q;
  long long q_tok;
  void *out;
  float *ws;            // [2 CTAs][COLS][HD + 2]
  int n_heads, G;
  Window win;
  float scale_log2;
  int *err;
  int beside;           // the many-row kernel runs beside this one: it may start when this one has waited for what both read
};

__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {   // an 8 x 8 matrix of D, a row a lane group
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int dev_first(const SeqRow &s, const Window &w) {   // first_seen
  if (w.w <= 0) return 0;
  if (w.by_call) return s.pos0 > 0 ? max(0, s.pos0 + s.count - w.w) : 0;
  return max(0, s.pos0 + 1 - w.w);
}
// a walk over a share: runs (sequence, key head) of tiles
struct Walk {
  int i, kvh, tile, left, t0, n;   // tile: in the run, of n; the run's first tile is t0 of its sequence
  SeqRow s;
  __device__ __forceinline__ void run(const Window &w) {
    t0 = dev_first(s, w) / TILE;
    n = (s.pos0 + s.count - 1) / TILE - t0 + 1;
  }
  __device__ __forceinline__ void start(const Worker &x, const Window &w) {
    i = x.i; kvh = x.kvh; tile = x.tile; left = x.left; s = x.s;
    run(w);
  }
  __device__ __forceinline__ int here() const { return min(left, n - tile); }   // tiles of this run in the share
  __device__ __forceinline__ void next(const Few &a, int by) {                  // `by` of them on
    left -= by;
    tile += by;
    if (tile < n || left <= 0) return;
    tile = 0;
    if (++kvh == a.pool.n_kv) {
      kvh = 0;
      const int4 v = __ldg(reinterpret_cast<const int4 *>(a.seqs + ++i));
      s = SeqRow{v.x, v.y, v.z, v.w};
      run(a.win);
    }
  }
};

// CLUSTER: no list of shares; a cluster of CTAs has a run, whose tiles they cut between them, and joins their sums over its shared memory
template <typename T, int HD, int NT, bool CLUSTER>
__global__ void __launch_bounds__(FEW_THREADS, FewCfg<HD, NT>::CTAS) few_kernel(const Few a) {
  typedef FewCfg<HD, NT> C;
  extern __shared__ __align__(128) unsigned char few_smem[];
  unsigned char *ring = few_smem;
  float *red = reinterpret_cast<float *>(ring + C::STAGES * 2 * C::ROWS_BYTES);
  float2 *ml = reinterpret_cast<float2 *>(red + FEW_WARPS * C::COLS * HD);
  uint64_t *full = reinterpret_cast<uint64_t *>(ml + FEW_WARPS * C::COLS), *empty = full + C::STAGES;
  uint32_t *marked = reinterpret_cast<uint32_t *>(empty + C::STAGES);
  int *gave_up = reinterpret_cast<int *>(marked + C::STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], FEW_WARPS);
    }
    *gave_up = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (a.beside) {
    pdl_wait();
    __syncthreads();
  }
  pdl_launch_dependents();
  if (!same_step(a.pool) || (!CLUSTER && (int)blockIdx.x >= a.plan->W)) {   // (nothing in flight, no barrier ahead of anybody)
    pdl_wait();
    return;
  }
  Walk w;
  const int size = CLUSTER ? (int)cluster_size() : 1, rank = CLUSTER ? (int)cluster_rank() : 0;
  if (CLUSTER) {
    const int run = (int)blockIdx.x / size;
    w.i = run / a.pool.n_kv;
    w.kvh = run - w.i * a.pool.n_kv;
    const int4 v = __ldg(reinterpret_cast<const int4 *>(a.seqs + w.i));
    w.s = SeqRow{v.x, v.y, v.z, v.w};
    w.run(a.win);
    w.tile = w.n * rank / size;
    w.left = w.n * (rank + 1) / size - w.tile;
  } else {
    const int4 *x = reinterpret_cast<const int4 *>(reinterpret_cast<const Worker *>(a.plan + 1) + blockIdx.x);
    const int4 u = __ldg(x), v = __ldg(x + 1);
    w.start(Worker{u.x, u.y, u.z, u.w, SeqRow{v.x, v.y, v.z, v.w}}, a.win);
  }
  // (a cluster's sums of this CTA, where its tiles were)
  float *sums = reinterpret_cast<float *>(ring);
  float2 *tops = reinterpret_cast<float2 *>(ring + C::COLS * HD * 4);
  const int all_cols = w.s.count * a.G;
  int left = MBAR_TRIES, in_ring = 0;
  if (warp == FEW_WARPS) {
    // ---- copies.  A lane has one piece (a page, or 64 rows of one) of a batch of tiles; the next batch's pages are looked up ahead
    const int P = 1 << a.pool.page_log2, pr = min(P, TILE), ppt = TILE / pr, most = 32 / ppt;   // rows of a piece; pieces of a tile; tiles of a batch
    const size_t head_bytes = rows_bytes(HD, 2 * P);
    const int piece = lane % ppt;
    int issued = 0;
    auto look = [&](const Walk &x, int n) -> int {
      return lane < n * ppt && x.left > 0 ? page_of(a.pool, x.s.slot, min(((x.t0 + x.tile + lane / ppt) * TILE) + piece * pr, x.s.pos0 + x.s.count - 1)) : 0;
    };
    Walk b = w;
    int n = min(b.here(), most), page = look(b, n);
    pdl_wait();
    while (b.left > 0) {
      const uint32_t mark = lane < n * ppt ? __ldcg(a.pool.marks + (size_t)page * a.pool.n_kv + b.kvh) : 0u;
      Walk nb = b;
      nb.next(a, n);
      const int nn = nb.left > 0 ? min(nb.here(), most) : 0, npage = look(nb, nn);
      const int end = b.s.pos0 + b.s.count;
      const char *src = a.pool.pages + ((size_t)page * a.pool.n_kv + b.kvh) * head_bytes;
      auto issue = [&](int t) {
        const int st = issued % C::STAGES, at = (b.t0 + b.tile + t) * TILE, mine = at + piece * pr;
        if (issued >= C::STAGES) {
          mbar_wait_lim(&empty[st], (uint32_t)(issued / C::STAGES - 1) & 1u, a.err, left);
          if (__any_sync(0xffffffffu, left == 0)) left = 0;
        }
        const int tile_rows = min(TILE, (end - at + 15) & ~15), rows = min(pr, max(0, (end - mine + 15) & ~15));
        if (left && lane == 0) mbar_expect_tx(&full[st], (uint32_t)rows_bytes(HD, 2 * tile_rows));
        __syncwarp();
        if (left && rows > 0 && lane / ppt == t) {
          unsigned char *k = ring + st * 2 * C::ROWS_BYTES + rows_bytes(HD, piece * pr);
          const char *from = src + rows_bytes(HD, mine & (P - 1));
          bulk_copy(k, from, (uint32_t)rows_bytes(HD, rows), &full[st]);
          bulk_copy(k + C::ROWS_BYTES, from + rows_bytes(HD, P), (uint32_t)rows_bytes(HD, rows), &full[st]);
        }
        issued++;
      };
      auto arrive = [&](int t, int nth) {
        const uint32_t any = __ballot_sync(0xffffffffu, mark != 0u && lane / ppt == t);
        if (lane == 0) {
          marked[nth % C::STAGES] = any;
          mbar_arrive(&full[nth % C::STAGES]);
        }
      };
      int t = 0;
      if (issued == 0) {   // the ring is empty: its copies first, what else a tile needs behind them
        for (; t < min(n, C::STAGES); t++) issue(t);
        for (int j = 0; j < t; j++) arrive(j, j);
      }
      for (; t < n; t++) {
        issue(t);
        arrive(t, issued - 1);
      }
      b = nb; n = nn; page = npage;
    }
    if (left == 0) *gave_up = 1;
    in_ring = issued;
  } else {
    // ---- products
    const int g = lane >> 2, t = lane & 3, r8 = lane & 7;
    // ldmatrix: lane's row of the 16 positions and its chunk's parity.  K: matrices (positions 0-7, 8-15) x (chunks c, c + 1); V transposed: chunks first
    const uint32_t k_row = (uint32_t)((2 * warp + (lane >> 3 & 1)) * (HD / 64) * 1024 + r8 * 128), v_row = (uint32_t)((2 * warp + (lane >> 4)) * (HD / 64) * 1024 + r8 * 128);
    const int k_odd = lane >> 4, v_odd = lane >> 3 & 1;
    pdl_wait();
    int taken = 0;
    while (w.left > 0) {
      const int n = w.here(), cols = w.s.count * a.G, end = w.s.pos0 + w.s.count;
      uint32_t qb[NT][HD / 16][2];
      int hi[NT][2], lo[NT][2];   // what columns 2t, 2t + 1 see
#pragma unroll
      for (int x = 0; x < NT; x++) {
        const int c = 8 * x + g, tok = c / a.G;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.q) + (size_t)(w.s.row0 + tok) * a.q_tok + (size_t)(w.kvh * a.G + c - tok * a.G) * HD);
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          qb[x][k][0] = c < cols ? __ldcg(src + 8 * k + t) : 0u;
          qb[x][k][1] = c < cols ? __ldcg(src + 8 * k + 4 + t) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int c2 = 8 * x + 2 * t + e, p = w.s.pos0 + c2 / a.G;
          hi[x][e] = c2 < cols ? p : -1;
          lo[x][e] = a.win.w <= 0 ? 0 : a.win.by_call ? dev_first(w.s, a.win) : max(0, p + 1 - a.win.w);
        }
      }
      const int late = a.win.w <= 0 ? 0 : a.win.by_call ? dev_first(w.s, a.win) : max(0, end - a.win.w);   // what the last row begins at
      float o[NT][HD / 16][4], m[NT][2], l[NT][2];
#pragma unroll
      for (int x = 0; x < NT; x++) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[x][i][e] = 0.f;
        m[x][0] = m[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.f;
      }
      for (int j = 0; j < n; j++, taken++) {
        const int st = taken % C::STAGES, at = (w.t0 + w.tile + j) * TILE + 16 * warp;   // this warp's positions: at .. at + 15
        mbar_wait_lim(&full[st], (uint32_t)(taken / C::STAGES) & 1u, a.err, left);
        __syncwarp();
        if (at < end && at + 15 >= dev_first(w.s, a.win)) {
          const uint32_t kt = smem_u32(ring + st * 2 * C::ROWS_BYTES), vt = kt + C::ROWS_BYTES;
          float s[NT][4];
#pragma unroll
          for (int x = 0; x < NT; x++) {
            float s2[4] = {0.f, 0.f, 0.f, 0.f};
            s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
              uint32_t f[4];
              const int c = 2 * k + k_odd;
              ldm4(kt + k_row + (uint32_t)((c >> 3) * 1024 + (((c & 7) ^ r8) << 4)), f);
              mma16816<T>(k & 1 ? s2 : s[x], f, qb[x][k][0], qb[x][k][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) s[x][e] += s2[e];
          }
          const bool edge = at + 15 > w.s.pos0 || at < late;
          if (edge)
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const int p = at + g + (e >> 1) * 8;
                if (p > hi[x][e & 1] || p < lo[x][e & 1]) s[x][e] = -INFINITY;
              }
          float f[NT][2];
          bool grew = false;
#pragma unroll
          for (int x = 0; x < NT; x++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float v = fmaxf(s[x][e], s[x][e + 2]);
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
              f[x][e] = 1.f;
              if (v > m[x][e]) {
                f[x][e] = ex2((m[x][e] - v) * a.scale_log2);   // (from -inf: 0)
                m[x][e] = v;
                grew = true;
              }
            }
          if (__any_sync(0xffffffffu, grew))
#pragma unroll
            for (int x = 0; x < NT; x++) {
#pragma unroll
              for (int e = 0; e < 2; e++) l[x][e] *= f[x][e];
#pragma unroll
              for (int i = 0; i < HD / 16; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[x][i][e] *= f[x][e & 1];
            }
          uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
          for (int x = 0; x < NT; x++) {
            constexpr float UP = lift<T>(15);   // (the largest is 1)
            const float c0 = m[x][0] == -INFINITY ? 0.f : m[x][0] * a.scale_log2 - UP, c1 = m[x][1] == -INFINITY ? 0.f : m[x][1] * a.scale_log2 - UP;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              s[x][e] = ex2(fmaf(s[x][e], a.scale_log2, -(e & 1 ? c1 : c0)));
              l[x][e & 1] += s[x][e];
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t h = pack2x<T>(s[x][2 * e], s[x][2 * e + 1]);
              const float2 hf = DT<T>::unpack2(h);
              bh[x][e] = transposed(h);
              bl[x][e] = transposed(pack2x<T>(s[x][2 * e] - hf.x, s[x][2 * e + 1] - hf.y));
            }
          }
          if (marked[st] == 0u) {
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
              uint32_t v[4];
              const int c = 2 * i + v_odd;
              ldm4t(vt + v_row + (uint32_t)((c >> 3) * 1024 + (((c & 7) ^ r8) << 4)), v);
#pragma unroll
              for (int x = 0; x < NT; x++) {
                mma16816<T>(o[x][i], v, bh[x][0], bh[x][1]);
                mma16816<T>(o[x][i], v, bl[x][0], bl[x][1]);
              }
            }
          } else {
            // an infinity or a NaN is somewhere in these pages: a row sums what it sees and nothing else
            for (int k = 0; k < 16; k++) {
              float pk[NT][2];
              bool sees[NT][2];
#pragma unroll
              for (int x = 0; x < NT; x++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const float lo8 = __shfl_sync(0xffffffffu, s[x][e], (k & 7) * 4 + t), hi8 = __shfl_sync(0xffffffffu, s[x][e + 2], (k & 7) * 4 + t);
                  pk[x][e] = k < 8 ? lo8 : hi8;
                  sees[x][e] = at + k <= hi[x][e] && at + k >= lo[x][e];
                }
              const unsigned char *row = ring + st * 2 * C::ROWS_BYTES + C::ROWS_BYTES + (size_t)(2 * warp + (k >> 3)) * (HD / 64) * 1024 + (k & 7) * 128;
#pragma unroll
              for (int i = 0; i < HD / 16; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const int d = 16 * i + g + (e >> 1) * 8;
                  const float v = DT<T>::to_f(*reinterpret_cast<const T *>(row + (d >> 6) * 1024 + (((d >> 3 & 7) ^ (k & 7)) << 4) + (d & 7) * 2));
#pragma unroll
                  for (int x = 0; x < NT; x++)
                    if (sees[x][e & 1]) o[x][i][e] = fmaf(pk[x][e & 1], v, o[x][i][e]);
                }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      // ---- the four warps' sums together
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float v = l[x][e];
          v += __shfl_xor_sync(0xffffffffu, v, 4);
          v += __shfl_xor_sync(0xffffffffu, v, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 16);
          if (g == 0) ml[warp * C::COLS + 8 * x + 2 * t + e] = make_float2(m[x][e], v);
        }
      auto in_red = [](int k, int c, int d) { return (k * C::COLS + c) * HD + (d ^ ((c >> 1 & 3) << 3)); };   // (a warp's 8 entries of 4 pairs of columns: 32 banks)
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) red[in_red(warp, 8 * x + 2 * t + (e & 1), 16 * i + g + (e >> 1) * 8)] = o[x][i][e];
      named_bar_sync(1, 32 * FEW_WARPS);
      const bool whole = CLUSTER ? size == 1 : w.tile == 0 && n == w.n;
      const int per = HD / 4;   // pieces of four entries of a column
      auto store = [&](int c, int d, float4 v, float inv) {
        const int tok = c / a.G;
        uint2 *to = reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + ((size_t)(w.s.row0 + tok) * a.n_heads + w.kvh * a.G + c - tok * a.G) * HD + d);
        *to = make_uint2(pack2x<T>(v.x * inv, v.y * inv), pack2x<T>(v.z * inv, v.w * inv));
      };
      auto place = [&](int k) { return a.ws + (size_t)k * C::COLS * (HD + 2); };
      const int mine = 2 * (int)blockIdx.x + (w.tile == 0 ? 1 : 0);   // a share's last run may begin in it (places 2 w + 1), its first one go on (2 w)
      for (int u = threadIdx.x; u < cols * per; u += 32 * FEW_WARPS) {
        const int c = u / per, d = 4 * (u - c * per);
        float M = -INFINITY, L = 0.f;
        float2 of[FEW_WARPS];
#pragma unroll
        for (int k = 0; k < FEW_WARPS; k++) {
          of[k] = ml[k * C::COLS + c];
          M = fmaxf(M, of[k].x);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < FEW_WARPS; k++) {   // (a warp that has seen nothing, or no number, has sums of 0 or NaN)
          const float f = of[k].x == -INFINITY ? 1.f : ex2((of[k].x - M) * a.scale_log2);
          const float4 y = *reinterpret_cast<const float4 *>(&red[in_red(k, c, d)]);
          L = fmaf(of[k].y, f, L);
          v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
        }
        if (whole) store(c, d, v, 1.0f / L);
        else if (CLUSTER) {
          *reinterpret_cast<float4 *>(sums + c * HD + d) = v;
          if (d == 0) tops[c] = make_float2(M, L);
        } else {
          __stcg(reinterpret_cast<float4 *>(place(mine) + c * HD + d), v);
          if (d == 0) __stcg(reinterpret_cast<float2 *>(place(mine) + C::COLS * HD) + c, make_float2(M, L));
        }
      }
      if (CLUSTER) break;
      named_bar_sync(1, 32 * FEW_WARPS);   // (red and ml are free again)
      w.next(a, n);
    }
    if (left == 0) *gave_up = 1;
  }
  if (CLUSTER && size > 1) {
    if (w.left == 0)   // fewer tiles than CTAs
      for (int c = threadIdx.x; c < all_cols; c += FEW_THREADS) tops[c] = make_float2(-INFINITY, 0.f);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    for (int u = rank * FEW_THREADS + (int)threadIdx.x; u < all_cols * (HD / 4); u += size * FEW_THREADS) {
      const int c = u / (HD / 4), d = 4 * (u - c * (HD / 4)), tok = c / a.G;
      const uint32_t of_sums = smem_u32(sums + c * HD + d), of_tops = smem_u32(tops + c);
      float M = -INFINITY, L = 0.f;
      float2 m[8];
      float4 y[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        m[k] = make_float2(-INFINITY, 0.f);
        y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < size) {
          m[k] = ld_cluster_f2(cluster_map(of_tops, (uint32_t)k));
          y[k] = ld_cluster_f4(cluster_map(of_sums, (uint32_t)k));
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) M = fmaxf(M, m[k].x);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const bool none = m[k].x == -INFINITY && m[k].y == 0.f;   // (a CTA without tiles, or one of rows that see none of them: its sums are not there, or 0)
        const float f = none ? 0.f : m[k].x == -INFINITY ? 1.f : ex2((m[k].x - M) * a.scale_log2);
        L = fmaf(m[k].y, f, L);
        if (!none) { v.x = fmaf(y[k].x, f, v.x); v.y = fmaf(y[k].y, f, v.y); v.z = fmaf(y[k].z, f, v.z); v.w = fmaf(y[k].w, f, v.w); }
      }
      const float inv = 1.0f / L;
      *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + ((size_t)(w.s.row0 + tok) * a.n_heads + w.kvh * a.G + c - tok * a.G) * HD + d) =
          make_uint2(pack2x<T>(v.x * inv, v.y * inv), pack2x<T>(v.z * inv, v.w * inv));
    }
    __syncwarp();
    cluster_arrive();   // (nobody leaves while another reads its sums)
    cluster_wait();
  }
  __syncthreads();
  if (*gave_up && threadIdx.x == 32 * FEW_WARPS)   // a wait was given up: copies in flight end before the CTA does
    for (int j = max(0, in_ring - C::STAGES); j < in_ring; j++) mbar_drain(&full[j % C::STAGES], (uint32_t)(j / C::STAGES) & 1u);
}

// The parts of a run: a CTA a query row, a thread four entries of every PG-th part, up to eight of them asked for at once
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(128) few_join_kernel(const Few a, const Cut *cuts) {
  pdl_launch_dependents();
  constexpr int PER = HD / 4, PG = 128 / PER, AT_ONCE = 8, COLS = 8 * NT;
  __shared__ float4 sums[128];
  __shared__ float2 tops[128];
  const int col = (int)blockIdx.y, d = 4 * (threadIdx.x % PER), pg = threadIdx.x / PER;
  const bool any = same_step(a.pool) && (int)blockIdx.x < a.plan->n_cuts;
  Cut cut{};
  if (any) {
    const int4 *x = reinterpret_cast<const int4 *>(cuts + blockIdx.x);
    const int4 u = __ldg(x), v = __ldg(x + 1);
    cut = Cut{SeqRow{u.x, u.y, u.z, u.w}, v.x, v.y, v.z, 0};
  }
  pdl_wait();
  if (!any || col >= cut.s.count * a.G) return;
  float M = -INFINITY, L = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = pg; k < cut.parts; k += PG * AT_ONCE) {
    float4 y[AT_ONCE];
    float2 m[AT_ONCE];
    float top = M;
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) {
      const int j = k + PG * i;
      const float *place = a.ws + (size_t)(j ? 2 * (cut.first + j) : 2 * cut.first + 1) * COLS * (HD + 2);
      m[i] = j < cut.parts ? __ldcg(reinterpret_cast<const float2 *>(place + COLS * HD) + col) : make_float2(-INFINITY, 0.f);
      y[i] = j < cut.parts ? __ldcg(reinterpret_cast<const float4 *>(place + col * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) top = fmaxf(top, m[i].x);
    const float old = M == -INFINITY ? 1.f : ex2((M - top) * a.scale_log2);   // (nothing, or no number, so far: sums of 0 or NaN)
    M = top;
    L *= old; v.x *= old; v.y *= old; v.z *= old; v.w *= old;
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) {
      const float f = m[i].x == -INFINITY ? 1.f : ex2((m[i].x - M) * a.scale_log2);
      L = fmaf(m[i].y, f, L);
      v.x = fmaf(y[i].x, f, v.x); v.y = fmaf(y[i].y, f, v.y); v.z = fmaf(y[i].z, f, v.z); v.w = fmaf(y[i].w, f, v.w);
    }
  }
  sums[threadIdx.x] = v;
  tops[threadIdx.x] = make_float2(M, L);
  __syncthreads();
  if (pg) return;
  float top = M;
#pragma unroll
  for (int k = 1; k < PG; k++) top = fmaxf(top, tops[k * PER + threadIdx.x].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  L = 0.f;
#pragma unroll
  for (int k = 0; k < PG; k++) {
    const float2 m = tops[k * PER + threadIdx.x];
    const float4 y = sums[k * PER + threadIdx.x];
    const float f = m.x == -INFINITY ? 1.f : ex2((m.x - top) * a.scale_log2);
    L = fmaf(m.y, f, L);
    o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y); o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
  }
  const float inv = 1.0f / L;
  const int tok = col / a.G;
  *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + ((size_t)(cut.s.row0 + tok) * a.n_heads + cut.kvh * a.G + col - tok * a.G) * HD + d) =
      make_uint2(pack2x<T>(o.x * inv, o.y * inv), pack2x<T>(o.z * inv, o.w * inv));
}

}  // namespace pg
}  // namespace cake
