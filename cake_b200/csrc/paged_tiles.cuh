// paged_tiles.cuh — attention of many rows a sequence over a cache in pages (portions of prompts, prompts), on tcgen05
//
// The same division of work as attn_prefill_tc.cuh: 128 query rows (the G heads of a key head x 128 / G tokens) a CTA, softmax in warps 0-3 with a thread a
// row, warp 4 copies, warp 5 multiplies; S in fp32 in TMEM, P as two operands of D (16 bits and more) over the S that it came from, O in TMEM, rescaled where a
// maximum grew by more than tau.  Bound by the softmax warps' chain beside the products (6 hd operations a pair instead of 4: P V twice) at the clock that the
// chip's power leaves: two CTAs an SM take 1950 cycles for a tile of 64 keys each, of which the products are 1540 and the exponentials 1020 (MUFU), at 1.55 GHz;
// 5 us a CTA go by before the first tile and behind the last.  A prompt of 4096, 32 / 8 heads of 128: 177 us (195 to 204 at the power cap),
// 0.48 of measured bf16, 0.72 counting P V twice.  Tiles of 128 keys: with one S buffer 256 us for 206 (a CTA's S, softmax and P V follow one another, and two CTAs fall in step),
// with two and one CTA an SM 263 (nothing beside a CTA's beginning and end).
// What is different:
//   - keys and values come page by page as they lie: a page's groups of eight rows are the operands' own layout, so that bulk copies without a tensor map fill
//     a tile from pages of any size, and Q is laid out by the softmax warps (no map to encode, any stride)
//   - a CTA's sequence, tokens and keys stand in a list (paged_plan.hpp, cut_many): sequences of any lengths side by side, the tiles with the most keys first, and
//     keys cut into parts where the tiles do not fill the chip; a kernel of its own joins them, in their order (the CTA that comes last would have 5 parts of 132 KB for a
//     tile of 256-entry heads)
//   - only whole sixteens of positions that hold a visible one are multiplied; where a page is marked (an infinity or a NaN in its values) a row sums what it sees by itself
#pragma once
#include "attn_prefill_tc.cuh"
#include "paged_few.cuh"

namespace cake {
namespace pg {

template <int HD> struct TileCfg {
  static constexpr int Q_BYTES = TILE_ROWS * HD * 2, KV_BYTES = TILE * HD * 2;
  static constexpr int BARS = 14, SMEM = Q_BYTES + 4 * KV_BYTES + 1024 + BARS * 8 + 32;
  static constexpr int TMEM = HD == 256 ? 512 : 256;   // S and P: columns 0 .. 63 and 64 .. 127; O from 128
  static constexpr int CTAS = HD == 256 ? 1 : 2;
  static constexpr size_t PART = (size_t)TILE_ROWS * (HD + 2);   // floats of a part: O as [HD / 4][row][4], then (m, l) of the rows
  static_assert(128 + HD <= TMEM && CTAS * TMEM <= 512 && CTAS * (SMEM + 1024) <= 228 * 1024, "TMEM columns, shared memory");
};
struct Tiles {
  Pool pool;
  const PlanHead *plan;
  const Item *items;
  const void *q;
  long long q_tok;
  void *out;
  float *ws;             // [key head][parts][PART]
  int n_heads, G, tpt;
  Window win;
  float scale_log2, tau_log2;
  int *err;
  int beside;            // the few-row kernel in front of this one waited for what both read: this one waits for it at its end
};

// two fp32 numbers in one operation
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 of_two(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 32 columns on their way; tc_wait_ld in front of their use
__device__ __forceinline__ void tc_ld32_go(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// (the registers pass through it, so that nothing that uses them is moved in front; an asm takes no more than 30 operands)
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
  asm volatile(""
               : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                 "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ float tc_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  return __uint_as_float(r);
}
// the product with P from TMEM, or nothing: a predicate and not a branch (behind one every product's operands make their own way to the uniform registers)
__device__ __forceinline__ void mma_ts_if(uint32_t yes, uint32_t tmem_c, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_c),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(yes)
      : "memory");
}
// an operand whose groups of eight rows lie `group` bytes apart and whose 64-entry ranges 1 KB: K-major (keys), and MN-major (values)
__device__ __forceinline__ uint64_t desc_keys(const void *tile, uint32_t group) {
  return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | (1ull << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_values(const void *tile, uint32_t group) {
  return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | ((uint64_t)(1024 >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <typename T, int HD>
__global__ void __launch_bounds__(FT_THREADS, TileCfg<HD>::CTAS) tiles_kernel(const Tiles a) {
  typedef TileCfg<HD> C;
  constexpr uint32_t GROUP = HD / 64 * 1024;
  extern __shared__ unsigned char tiles_smem[];
  unsigned char *q_s = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(tiles_smem) + 1023) & ~(uintptr_t)1023);
  unsigned char *k_s = q_s + C::Q_BYTES, *v_s = k_s + 2 * C::KV_BYTES;   // two stages each
  uint64_t *bars = reinterpret_cast<uint64_t *>(v_s + 2 * C::KV_BYTES);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7, *s_full = bars + 9, *p_full = bars + 11, *o_full = bars + 12;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(bars + C::BARS);
  int *gave_up = reinterpret_cast<int *>(tmem_ptr + 1);
  volatile uint32_t *marked = tmem_ptr + 4;   // of tiles j, j + 1 .. j + 3: a slot is written again when the tile two in front of it has been multiplied

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = (int)blockIdx.x % a.pool.n_kv, nth = (int)blockIdx.x / a.pool.n_kv;
  if (!same_step(a.pool) || nth >= a.plan->n_items) {
    pdl_wait();
    return;
  }
  Item it;
  {
    const int4 *x = reinterpret_cast<const int4 *>(a.items + nth);
    const int4 u = __ldg(x), v = __ldg(x + 1), w = __ldg(x + 2);
    it = Item{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w, SeqRow{w.x, w.y, w.z, w.w}};
  }
  const int G = a.G, n_tok = min(a.tpt, it.s.count - it.tok0), rows = G * n_tok, n_tiles = it.t1 - it.t0;
  const int p0 = it.s.pos0 + it.tok0, kv_end = p0 + n_tok;   // the first token's position; keys that the last one sees
  const uint32_t by_G = (65536u + (uint32_t)G - 1u) / (uint32_t)G;   // r / G = r by_G >> 16 for r < 128, G <= 128
  const int row = (warp & 3) * 32 + lane, tok = (int)((uint32_t)row * by_G >> 16);
  const int by_call = a.win.w > 0 && a.win.by_call ? dev_first(it.s, a.win) : 0;
  const int late = a.win.w <= 0 ? 0 : a.win.by_call ? by_call : max(0, kv_end - a.win.w);   // what the last token begins at

  // the queries are asked for while the rest is set up, up to sixteen 16-byte chunks a thread (one after the other, each in front of its store, they took 5 to 17 us)
  constexpr int CH = HD / 8, BY = 128 / CH, FEW = CH < 16 ? CH : 16;   // chunks of a row; rows of a pass
  const int qc = (int)threadIdx.x % CH, qr = (int)threadIdx.x / CH;
  struct Chunks { uint4 v[FEW]; } first;
  auto ask = [&](int i0) {
    const T *q = reinterpret_cast<const T *>(a.q) + (size_t)(it.s.row0 + it.tok0) * a.q_tok + (size_t)kvh * G * HD + 8 * qc;
    Chunks x;
#pragma unroll
    for (int i = 0; i < FEW; i++) {
      const int r = qr + (i0 + i) * BY, tk = (int)((uint32_t)r * by_G >> 16);
      x.v[i] = r < rows ? __ldcg(reinterpret_cast<const uint4 *>(q + (size_t)tk * a.q_tok + (size_t)(r - tk * G) * HD)) : make_uint4(0u, 0u, 0u, 0u);
    }
    return x;
  };
  auto lay = [&](int i0, const Chunks &x) {
#pragma unroll
    for (int i = 0; i < FEW; i++) {
      const int r = qr + (i0 + i) * BY;
      *reinterpret_cast<uint4 *>(q_s + (qc >> 3) * (TILE_ROWS * 128) + r * 128 + (((qc & 7) ^ (r & 7)) << 4)) = x.v[i];
    }
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::BARS; i++) mbar_init(&bars[i], i == 11 || i == 0 ? 128u : 1u);
    *gave_up = 0;
    mbar_fence_init();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_ptr)), "n"(C::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the copying warp's first pages likewise
  const int P = 1 << a.pool.page_log2, pr = min(P, TILE), ppt = TILE / pr, most = 32 / ppt, piece = lane % ppt;   // rows of a piece; pieces of a tile; tiles of a batch
  const size_t head_bytes = rows_bytes(HD, 2 * P);
  auto look = [&](int j, int n) -> int { return lane < n * ppt ? page_of(a.pool, it.s.slot, min((it.t0 + j + lane / ppt) * TILE + piece * pr, kv_end - 1)) : 0; };
  int n = min(n_tiles, most), page = 0;
  if (warp == 4) page = look(0, n);
  if (warp < 4) {
    if (!a.beside) pdl_wait();
    first = ask(0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem_base = *tmem_ptr, tmem_o = tmem_base + 128u, lane_addr = (uint32_t)((warp & 3) * 32) << 16;
  const bool busy = warp < 4 && warp * 32 < rows;
  float m_run = -INFINITY, l_run = 0.f;
  int left = MBAR_TRIES, k_loads = 0, v_loads = 0;

  if (warp == 4) {
    // ---- copies.  A lane has one piece (a page, or 64 rows of one) of a batch of tiles
    if (!a.beside) pdl_wait();
    for (int j0 = 0; j0 < n_tiles; j0 += most) {
      const uint32_t mark = lane < n * ppt ? __ldcg(a.pool.marks + (size_t)page * a.pool.n_kv + kvh) : 0u;
      const int nn = min(max(0, n_tiles - j0 - most), most), npage = look(j0 + most, nn);
      const char *src = a.pool.pages + ((size_t)page * a.pool.n_kv + kvh) * head_bytes;
      auto copy = [&](int t, bool values) {
        const int j = j0 + t, st = j & 1, at = (it.t0 + j) * TILE, mine = at + piece * pr;
        uint64_t *full = values ? &v_full[st] : &k_full[st];
        if (j >= 2) {
          mbar_wait_lim(values ? &v_empty[st] : &k_empty[st], (uint32_t)(j / 2 - 1) & 1u, a.err, left);
          if (__any_sync(0xffffffffu, left == 0)) left = 0;
        }
        const int of_tile = min(TILE, (kv_end - at + 15) & ~15), of_piece = min(pr, max(0, (kv_end - mine + 15) & ~15));
        if (left && lane == 0) mbar_expect_tx(full, (uint32_t)rows_bytes(HD, of_tile));
        __syncwarp();
        if (left && of_piece > 0 && lane / ppt == t)
          bulk_copy((values ? v_s : k_s) + st * C::KV_BYTES + rows_bytes(HD, piece * pr), src + rows_bytes(HD, (mine & (P - 1)) + (values ? P : 0)), (uint32_t)rows_bytes(HD, of_piece), full);
        (values ? v_loads : k_loads)++;
      };
      auto arrive = [&](int t) {
        const uint32_t any = __ballot_sync(0xffffffffu, mark != 0u && lane / ppt == t);
        if (lane == 0) {
          marked[(j0 + t) & 3] = any;
          mbar_arrive(&k_full[(j0 + t) & 1]);
        }
      };
      int t = 0;
      if (j0 == 0) {   // nothing in the stages yet: the copies first
        for (; t < min(n, 2); t++) {
          copy(t, false);
          copy(t, true);
        }
        for (int i = 0; i < t; i++) {
          arrive(i);
          if (lane == 0) mbar_arrive(&v_full[i]);
        }
      }
      for (; t < n; t++) {
        copy(t, false);
        arrive(t);
        copy(t, true);
        if (lane == 0) mbar_arrive(&v_full[(j0 + t) & 1]);
      }
      n = nn; page = npage;
    }
  } else if (warp == 5) {
    // ---- products (one thread issues them; the warp runs the loop with it)
    const uint32_t one = elect_one();
    const uint32_t idesc_s = tc_idesc<T>(TILE), idesc_o = tc_idesc<T>(HD) | (1u << 16);   // M128 N TILE, both K-major; M128 N hd, A from TMEM, B (V) MN-major
    uint32_t mark = 0u, next_mark = 0u;   // of tiles j and j + 1
    auto issue_s = [&](int j) {   // S_j = Q K_j^T into S buffer j & 1
      const int st = j & 1;
      mbar_wait_lim(&k_full[st], (uint32_t)(j / 2) & 1u, a.err, left);
      __syncwarp();
      tc_fence_after();
      mark = next_mark;
      next_mark = marked[j & 3];
      const uint64_t q0 = tc_smem_desc(q_s), kt = desc_keys(k_s, GROUP) + (uint64_t)(st * (C::KV_BYTES >> 4));
      if (one) {
#pragma unroll
        for (int k = 0; k < HD / 16; k++)
          tc_mma_f16(tmem_base + (uint32_t)(st * TILE), q0 + (uint64_t)((k >> 2) * (TILE_ROWS * 128 >> 4) + (k & 3) * 2), kt + (uint64_t)((k >> 2) * (1024 >> 4) + (k & 3) * 2), idesc_s,
                     k ? 1u : 0u);
        tc_commit(&k_empty[st], left);
        tc_commit(&s_full[st], left);
      }
      __syncwarp();
    };
    mbar_wait_lim(q_full, 0, a.err, left);
    __syncwarp();
    issue_s(0);
    for (int j = 0; j < n_tiles; j++) {
      const int st = j & 1;
      if (j + 1 < n_tiles) issue_s(j + 1);   // (its buffer held P of tile j - 1, whose P V is in front of it in the pipe)
      else mark = next_mark;
      mbar_wait_lim(p_full, (uint32_t)j & 1u, a.err, left);
      mbar_wait_lim(&v_full[st], (uint32_t)(j / 2) & 1u, a.err, left);
      __syncwarp();
      tc_fence_after();
      const uint64_t vt = desc_values(v_s, GROUP) + (uint64_t)(st * (C::KV_BYTES >> 4));
      const int steps = mark ? 0 : min(TILE, (kv_end - (it.t0 + j) * TILE + 15) & ~15) / 16;   // sixteens of positions; marked: the rows have summed by themselves
      if (one) {
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ks++)   // P of 32 keys: 16 columns of hi, 16 of lo
#pragma unroll
          for (int half = 0; half < 2; half++)
            mma_ts_if(ks < steps ? 1u : 0u, tmem_o, tmem_base + (uint32_t)(st * TILE + (ks >> 1) * 32 + half * 16 + (ks & 1) * 8), vt + (uint64_t)(ks * (2 * GROUP >> 4)), idesc_o,
                      (j | half | ks) ? 1u : 0u);
        tc_commit(&v_empty[st], left);
        tc_commit(o_full, left);
      }
      __syncwarp();
    }
  } else {
    // ---- queries into shared memory, in the operand's layout; rows that are not there are zero
    if (CH > 16) lay(16, ask(16));
    lay(0, first);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive(q_full);
    if (!busy) {
      for (int j = 0; j < n_tiles; j++) {   // (an arrival for tile j must not join the barrier's previous phase)
        if (j > 0) mbar_wait_lim(o_full, (uint32_t)(j - 1) & 1u, a.err, left);
        mbar_arrive(p_full);
      }
      mbar_wait_lim(o_full, (uint32_t)(n_tiles - 1) & 1u, a.err, left);
    } else {
      // ---- softmax (a thread a query row), 32 keys at a time: their maximum first, then weights over the scores that they come from
      const int qp = p0 + tok, lo = a.win.w <= 0 ? 0 : a.win.by_call ? by_call : max(0, qp + 1 - a.win.w);
      const uint64_t scale2 = two(a.scale_log2, a.scale_log2), minus1 = two(-1.f, -1.f);
      for (int j = 0; j < n_tiles; j++) {
        const uint32_t tmem_sp = tmem_base + lane_addr + (uint32_t)((j & 1) * 64);
        mbar_wait_lim(&s_full[j & 1], (uint32_t)(j / 2) & 1u, a.err, left);
        tc_fence_after();
        const uint32_t mark = marked[j & 3];
        const int k0 = (it.t0 + j) * TILE;
        const bool edge = k0 + TILE - 1 > p0 || k0 < late;   // a row of the tile does not see all of these
        auto hide = [&](uint32_t (&r)[32], int c) {
          if (edge)
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (k0 + 32 * c + i > qp || k0 + 32 * c + i < lo) r[i] = 0xff800000u;
        };
        uint32_t r[2][32];
        float mx[2] = {-INFINITY, -INFINITY};
        tc_ld32_go(tmem_sp, r[0]);
#pragma unroll
        for (int c = 0; c < TILE / 32; c++) {
          tc_wait_ld(r[c & 1]);
          tc_ld32_go(tmem_sp + (c + 1 < TILE / 32 ? 32u * (c + 1) : 0u), r[(c + 1) & 1]);   // (behind the last the first again, for its weights)
          hide(r[c & 1], c);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            mx[0] = max3(mx[0], __uint_as_float(r[c & 1][i]), __uint_as_float(r[c & 1][i + 1]));
            mx[1] = max3(mx[1], __uint_as_float(r[c & 1][i + 2]), __uint_as_float(r[c & 1][i + 3]));
          }
        }
        const float top = fmaxf(mx[0], mx[1]);
        float fac = 1.f;
        bool resc = false;
        if (j == 0) {
          m_run = top;
        } else if ((top - m_run) * a.scale_log2 > a.tau_log2) {   // (from -inf: factor 0)
          fac = ft_ex2((m_run - top) * a.scale_log2);
          m_run = top;
          resc = true;
        }
        const float mc = m_run == -INFINITY ? 0.f : m_run * a.scale_log2 - lift<T>(7);   // a row that has seen nothing yet counts from 0; the largest weight is 2^8
        const uint64_t mc2 = two(-mc, -mc);
        uint64_t rs[2] = {0ull, 0ull};
        auto weights = [&](auto clean) {   // two operands of D, or as they are
#pragma unroll
          for (int c = 0; c < TILE / 32; c++) {
            constexpr int B = TILE / 32 & 1;   // the buffer that the first chunk came into again
            uint32_t (&x)[32] = r[(c + B) & 1];
            tc_wait_ld(x);
            if (c + 1 < TILE / 32) tc_ld32_go(tmem_sp + 32u * (c + 1), r[(c + 1 + B) & 1]);
            hide(x, c);
            uint32_t lw[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float2 z = of_two(fma_two(two(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, mc2));
              const float e0 = ft_ex2(z.x), e1 = ft_ex2(z.y);
              const uint64_t e = two(e0, e1);
              rs[i & 1] = add_two(rs[i & 1], e);
              if (decltype(clean)::value) {
                x[i] = pack2x<T>(e0, e1);
                const float2 h = DT<T>::unpack2(x[i]);
                const float2 d = of_two(fma_two(two(h.x, h.y), minus1, e));
                lw[i] = pack2x<T>(d.x, d.y);
              } else {
                x[2 * i] = __float_as_uint(e0);
                x[2 * i + 1] = __float_as_uint(e1);
              }
            }
            if (decltype(clean)::value) {
#pragma unroll
              for (int i = 0; i < 16; i++) x[16 + i] = lw[i];
            }
            tc_st32(tmem_sp + 32u * c, x);
          }
        };
        if (mark == 0u) weights(std::true_type{});
        else weights(std::false_type{});
        const float2 s0 = of_two(add_two(rs[0], rs[1]));
        l_run = l_run * fac + (s0.x + s0.y);
        if (j > 0) {   // P V of the previous tile is there, O at rest (waited for in front of the weights: 300 to 600 of 2200 cycles a tile)
          mbar_wait_lim(o_full, (uint32_t)(j - 1) & 1u, a.err, left);
          tc_fence_after();
          if (__any_sync(0xffffffffu, resc)) {
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
              uint32_t x[32];
              tc_ld32(tmem_o + lane_addr + (uint32_t)c0, x);
#pragma unroll
              for (int i = 0; i < 32; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * fac);
              tc_st32(tmem_o + lane_addr + (uint32_t)c0, x);
            }
          }
        }
        if (mark) {
          // the tile's values hold an infinity or a NaN: the row sums those that it sees, weights by way of TMEM
          tc_wait_st();
          mbar_wait_lim(&v_full[j & 1], (uint32_t)(j / 2) & 1u, a.err, left);
          __syncwarp();
          const unsigned char *vt = v_s + (j & 1) * C::KV_BYTES;
          const int n = min(TILE, kv_end - k0);
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 32) {
            uint32_t x[32];
            tc_ld32(tmem_o + lane_addr + (uint32_t)c0, x);
            float o[32];
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = j > 0 ? __uint_as_float(x[i]) : 0.f;
#pragma unroll 1
            for (int k = 0; k < n; k++) {
              const float p = tc_ld1(tmem_sp + (uint32_t)k);
              if (k0 + k <= qp && k0 + k >= lo) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  const int c = (c0 >> 3) + i;
                  float v[8];
                  unpack8<T>(*reinterpret_cast<const uint4 *>(vt + (k >> 3) * GROUP + (c >> 3) * 1024 + (k & 7) * 128 + (((c & 7) ^ (k & 7)) << 4)), v);
#pragma unroll
                  for (int e = 0; e < 8; e++) o[8 * i + e] = fmaf(p, v[e], o[8 * i + e]);
                }
              }
              __syncwarp();
            }
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = __float_as_uint(o[i]);
            tc_st32(tmem_o + lane_addr + (uint32_t)c0, x);
          }
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(p_full);
      }
      mbar_wait_lim(o_full, (uint32_t)(n_tiles - 1) & 1u, a.err, left);   // every product of this CTA is there
      tc_fence_after();
    }
  }
  // ---- O / l, one rounding to D; or a part's sums for the one that joins them
  auto store = [&](int c0, const float (&v)[32], float inv) {
    T *dst = reinterpret_cast<T *>(a.out) + ((size_t)(it.s.row0 + it.tok0 + tok) * a.n_heads + kvh * G + row - tok * G) * HD + c0;
#pragma unroll
    for (int i = 0; i < 4; i++)
      reinterpret_cast<uint4 *>(dst)[i] = make_uint4(pack2x<T>(v[8 * i] * inv, v[8 * i + 1] * inv), pack2x<T>(v[8 * i + 2] * inv, v[8 * i + 3] * inv),
                                                     pack2x<T>(v[8 * i + 4] * inv, v[8 * i + 5] * inv), pack2x<T>(v[8 * i + 6] * inv, v[8 * i + 7] * inv));
  };
  auto place = [&](int part) { return a.ws + ((size_t)kvh * a.plan->parts + it.part0 + part) * C::PART; };
  if (busy) {
    const float inv_l = 1.0f / l_run;
    float4 *to = reinterpret_cast<float4 *>(place(it.part));
#pragma unroll 1
    for (int c0 = 0; c0 < HD; c0 += 32) {
      uint32_t r[32];
      tc_ld32(tmem_o + lane_addr + (uint32_t)c0, r);
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
      if (row < rows) {
        if (it.parts == 1) store(c0, v, inv_l);
        else
#pragma unroll
          for (int i = 0; i < 8; i++) __stcg(to + (c0 / 4 + i) * TILE_ROWS + row, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
      }
    }
    if (it.parts > 1 && row < rows) __stcg(reinterpret_cast<float2 *>(place(it.part) + TILE_ROWS * HD) + row, make_float2(m_run, l_run));
  }
  if (!left) *gave_up = 1;
  tc_fence_before();
  __syncthreads();
  if (*gave_up) ft_drain(bars, warp, lane, k_loads, v_loads);
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(C::TMEM) : "memory");
  }
  if (a.beside) pdl_wait();
}

// The parts of a tile: a CTA for eight entries of its rows, a thread a row; threads that few rows leave take every second, third .. part.  Up to eight parts are
// asked for at once (two at a time by one thread a row: 33 parts of 20 rows 45 us, so 7; 32 rows, 8 parts 22 and 8)
template <typename T, int HD>
__global__ void __launch_bounds__(128) join_kernel(const Tiles a, const int *cuts) {
  pdl_launch_dependents();
  constexpr int AT_ONCE = 8;
  __shared__ float4 sums[2][128];
  __shared__ float2 tops[128];
  const int kvh = (int)blockIdx.x % a.pool.n_kv, nth = (int)blockIdx.x / a.pool.n_kv;
  const bool any = same_step(a.pool) && nth < a.plan->n_cut_tiles;
  Item it{};
  if (any) it = a.items[cuts[nth]];
  const int rows = a.G * min(a.tpt, it.s.count - it.tok0), wide = rows <= 32 ? 32 : rows <= 64 ? 64 : 128, groups = 128 / wide;
  const int row = (int)threadIdx.x % wide, pg = (int)threadIdx.x / wide;
  pdl_wait();
  if (!any) return;
  const float *place = a.ws + ((size_t)kvh * a.plan->parts + it.part0) * TileCfg<HD>::PART;
  float M = -INFINITY, L = 0.f;
  float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  if (row < rows)
    for (int k = pg; k < it.parts; k += groups * AT_ONCE) {
      float4 y[AT_ONCE][2];
      float2 m[AT_ONCE];
      float top = M;
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) {
        const int j = k + groups * i;
        const float *from = place + (size_t)j * TileCfg<HD>::PART;
        m[i] = make_float2(-INFINITY, 0.f);
        if (j < it.parts) {
          m[i] = __ldcg(reinterpret_cast<const float2 *>(from + TILE_ROWS * HD) + row);
#pragma unroll
          for (int c = 0; c < 2; c++) y[i][c] = __ldcg(reinterpret_cast<const float4 *>(from) + (2 * blockIdx.y + c) * TILE_ROWS + row);
        }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) top = fmaxf(top, m[i].x);
      const float old = M == -INFINITY ? 1.f : ft_ex2((M - top) * a.scale_log2);   // (nothing, or no number, so far: sums of 0 or NaN)
      M = top;
      L *= old;
#pragma unroll
      for (int c = 0; c < 2; c++) { v[c].x *= old; v[c].y *= old; v[c].z *= old; v[c].w *= old; }
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++)
        if (k + groups * i < it.parts) {
          const float f = m[i].x == -INFINITY ? 1.f : ft_ex2((m[i].x - M) * a.scale_log2);
          L = fmaf(m[i].y, f, L);
#pragma unroll
          for (int c = 0; c < 2; c++) {
            v[c].x = fmaf(y[i][c].x, f, v[c].x); v[c].y = fmaf(y[i][c].y, f, v[c].y); v[c].z = fmaf(y[i][c].z, f, v[c].z); v[c].w = fmaf(y[i][c].w, f, v[c].w);
          }
        }
    }
  sums[0][threadIdx.x] = v[0];
  sums[1][threadIdx.x] = v[1];
  tops[threadIdx.x] = make_float2(M, L);
  __syncthreads();
  if (pg || row >= rows) return;
  for (int k = 1; k < groups; k++) M = fmaxf(M, tops[k * wide + row].x);
  L = 0.f;
  v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < groups; k++) {
    const float2 m = tops[k * wide + row];
    const float f = m.x == -INFINITY ? 1.f : ft_ex2((m.x - M) * a.scale_log2);
    L = fmaf(m.y, f, L);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const float4 y = sums[c][k * wide + row];
      v[c].x = fmaf(y.x, f, v[c].x); v[c].y = fmaf(y.y, f, v[c].y); v[c].z = fmaf(y.z, f, v[c].z); v[c].w = fmaf(y.w, f, v[c].w);
    }
  }
  const float inv = 1.0f / L;
  const int tok = row / a.G;
  T *dst = reinterpret_cast<T *>(a.out) + ((size_t)(it.s.row0 + it.tok0 + tok) * a.n_heads + kvh * a.G + row - tok * a.G) * HD + 8 * blockIdx.y;
  *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2x<T>(v[0].x * inv, v[0].y * inv), pack2x<T>(v[0].z * inv, v[0].w * inv), pack2x<T>(v[1].x * inv, v[1].y * inv),
                                               pack2x<T>(v[1].z * inv, v[1].w * inv));
}

}  // namespace pg
}  // namespace cake
