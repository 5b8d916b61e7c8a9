// packed_cache.cu — kernels of the cache in four bits (format and interface: packed_cache.cuh)
#include "packed_cache.cuh"
#include "common.cuh"

#include <algorithm>
#include <type_traits>

namespace cake {
namespace pc {

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

template <typename T> __device__ __forceinline__ T round_up(float f);
template <> __device__ __forceinline__ __nv_bfloat16 round_up<__nv_bfloat16>(float f) { return __float2bfloat16_ru(f); }
template <> __device__ __forceinline__ __half round_up<__half>(float f) { return __float2half_ru(f); }
template <typename T> __device__ __forceinline__ uint32_t bits(T v) { return *reinterpret_cast<const uint16_t *>(&v); }

// 8 entries of a group of four neighbouring lanes -> this lane's codes, entry i in nibble i, and the group's pair
// t inv + 1/2 is exact but for 2^-22 relative, and (x - lo) / step is k + 1/2 or at least the last place of x, lo or step away from it (in
// steps): 2^-19 decides the former and leaves the latter, where x's last place is above step 2^-19.
template <typename T> __device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t *pair) {
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad = bad || x[i] != x[i];
  }
  if (bad) hi = INFINITY;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float span = hi - lo;   // NaN or infinite: the group has no code
  const bool fine = span <= 3.402823466e38f;
  T st = round_up<T>(fine ? span / 15.f : 0.f);
  if (sizeof(T) == 2 && DT<T>::to_f(st) < 1.17549435e-38f && span > 0.f) st = DT<T>::from_f(1.17549435e-38f);
  const float step = DT<T>::to_f(st), inv = step > 0.f ? 1.f / step : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float n = fmaf(x[i] - lo, inv, 0.5f + 1.9073486328125e-6f);
    w |= (fine ? min(15u, (uint32_t)n) : 0u) << (4 * i);
  }
  *pair = fine ? bits(st) | bits(DT<T>::from_f(lo)) << 16 : 0x7fff7fffu;
  return w;
}

// a warp takes 256 / HD rows, a lane 8 neighbouring entries
template <typename T, int HD>
__global__ void __launch_bounds__(128) write_kernel(const Write a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LPR = HD / 8;
  const int lane = threadIdx.x & 31, u = lane % LPR;
  const int heads = a.n_q + 2 * a.n_kv;
  const long long rows = (long long)a.B * a.S * heads;
  const long long row = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * (32 / LPR) + lane / LPR;
  const bool in = row < rows;
  const long long at = in ? row : rows - 1;
  const int head = (int)(at % heads), t = (int)(at / heads % a.S), b = (int)(at / heads / a.S);
  const int pos = (a.d_pos ? *a.d_pos : a.pos0) + t;
  const bool is_q = head < a.n_q, is_v = head >= a.n_q + a.n_kv;
  const int h = is_q ? head : is_v ? head - a.n_q - a.n_kv : head - a.n_q;
  const T *src = is_q ? reinterpret_cast<const T *>(a.q) + b * a.k_batch + t * a.k_tok
                 : is_v ? reinterpret_cast<const T *>(a.v) + b * a.v_batch + t * a.v_tok : reinterpret_cast<const T *>(a.k) + b * a.k_batch + t * a.k_tok;
  uint4 raw = *reinterpret_cast<const uint4 *>(src + (size_t)h * HD + 8 * u);
  float x[8];
  unpack8<T>(raw, x);
  const T *nw = is_v ? nullptr : reinterpret_cast<const T *>(is_q ? a.q_norm : a.k_norm);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) ss += x[i] * x[i];
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (nw) {
    const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
    float w[8];
    unpack8<T>(*reinterpret_cast<const uint4 *>(nw + 8 * u), w);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = rnd<T>(x[i] * inv * w[i]);
  }
  if (a.cos_t) {   // pairs (i, i + rot / 2); rot is a multiple of 16: a lane's entries are all of one half
    const int half = a.rot / 2, at8 = 8 * u;
    const bool turned = !is_v && at8 < a.rot, low = at8 < half;
    const int other = (lane & ~(LPR - 1)) + (turned ? (low ? u + half / 8 : u - half / 8) : u);
    float y[8], c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], other);
    if (turned) {
      const size_t o = (size_t)pos * half + (low ? at8 : at8 - half);
      unpack8<T>(*reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.cos_t) + o), c);
      unpack8<T>(*reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.sin_t) + o), s);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = low ? rnd<T>(rnd<T>(x[i] * c[i]) - rnd<T>(y[i] * s[i])) : rnd<T>(rnd<T>(x[i] * c[i]) + rnd<T>(y[i] * s[i]));
    }
  }
  uint32_t pair, w = encode8<T>(x, &pair);
  if (is_q) {
    if (in)
      *reinterpret_cast<uint4 *>(const_cast<T *>(src) + (size_t)h * HD + 8 * u) =
          make_uint4(pack2x<T>(x[0], x[1]), pack2x<T>(x[2], x[3]), pack2x<T>(x[4], x[5]), pack2x<T>(x[6], x[7]));
  }
  if (is_q || !in) return;
  char *blk = reinterpret_cast<char *>(a.cache) + ((size_t)(b * a.n_kv + h) * a.blocks + (pos >> 4)) * block_bytes(HD);
  const int r = pos & 15, j = u >> 2, q = u & 3;
  if (!is_v) {
    // entry 2i to nibble i, entry 2i + 1 to nibble 4 + i
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) k |= (w >> (8 * i) & 15u) << (4 * i) | (w >> (8 * i + 4) & 15u) << (16 + 4 * i);
    reinterpret_cast<uint32_t *>(blk)[k_word(HD, r, u)] = k;
    if (q == 0) reinterpret_cast<uint32_t *>(blk + k_pairs(HD))[pair_word(HD, r, j)] = pair;
  } else {
    uint16_t *v = reinterpret_cast<uint16_t *>(blk + v_codes(HD));
    v[v_half(HD, r, 2 * q, j)] = (uint16_t)w;
    v[v_half(HD, r, 2 * q + 1, j)] = (uint16_t)(w >> 16);
    if (q == 0) reinterpret_cast<uint32_t *>(blk + v_pairs(HD))[pair_word(HD, r, j)] = pair;
  }
}

template <typename T> __device__ __forceinline__ float2 open_pair(uint32_t p) { return DT<T>::unpack2(p); }   // (step, lo)

// entry i's code in nibble i of what is returned: entries 8u .. 8u + 7 of position r
template <int HD> __device__ __forceinline__ uint32_t codes8(const char *blk, int which, int r, int u) {
  if (!which) {
    const uint32_t k = reinterpret_cast<const uint32_t *>(blk)[k_word(HD, r, u)];
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= (k >> (4 * i) & 15u) << (8 * i) | (k >> (16 + 4 * i) & 15u) << (8 * i + 4);
    return w;
  }
  const uint16_t *v = reinterpret_cast<const uint16_t *>(blk + v_codes(HD));
  return v[v_half(HD, r, 2 * (u & 3), u >> 2)] | (uint32_t)v[v_half(HD, r, 2 * (u & 3) + 1, u >> 2)] << 16;
}

template <typename T, int HD>
__global__ void __launch_bounds__(128) read_kernel(const Read a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LPR = HD / 8;
  const int lane = threadIdx.x & 31, u = lane % LPR;
  const long long row = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * (32 / LPR) + lane / LPR;
  if (row >= (long long)a.B * a.n_kv * a.n) return;
  const int i = (int)(row % a.n), slab = (int)(row / a.n), pos = a.first + i, r = pos & 15;
  const char *blk = reinterpret_cast<const char *>(a.cache) + ((size_t)slab * a.blocks + (pos >> 4)) * block_bytes(HD);
  const uint32_t w = codes8<HD>(blk, a.which, r, u);
  const float2 p = open_pair<T>(reinterpret_cast<const uint32_t *>(blk + (a.which ? v_pairs(HD) : k_pairs(HD)))[pair_word(HD, r, u >> 2)]);
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    o[e] = pack2x<T>(fmaf(p.x, (float)(w >> (8 * e) & 15u), p.y), fmaf(p.x, (float)(w >> (8 * e + 4) & 15u), p.y));
  *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + ((size_t)slab * a.out_rows + i) * HD + 8 * u) = make_uint4(o[0], o[1], o[2], o[3]);
}

// ------------------------------------------------------------------------------------------ attention of a few rows, keys split
// A CTA serves up to 8 NT / PK query rows (row = token G + head of one key head) and a range of blocks; its warps take the blocks in turn, each through
// a ring of its own (cp.async, 16 bytes a lane; a bulk copy and an mbarrier a block took a fifth of the loop), so that no warp waits for another
// until the end.  Per block, with m16n8k16 products in fp16:
//   S^T = K Q^T   A: 16 keys' codes, B: the rows' queries, kept in registers.  A group's sum is taken apart from the others', then
//                 s += step sum + lo (sum of the group's q): the codes go in exactly, and no entry is formed.  Queries are scaled by a power of two
//                 that puts a row's largest below 2^15: an entry down to 2^-29 of it keeps its bits.
//   O^T += V^T P  A: 16 entries' codes, B: weights times steps in fp16 (11 bits), one operand per group; what is left of the value, lo + 8
//                 step, is a number per key and group and is summed in fp32.  P^T turns into an operand by movmatrix.
// Four bits become fp16 by one logic operation a pair: n under the exponent of 1024 is 1024 + n in the lowest four bits, 1024 + 16 n in the next.
// The 16 stays in: K's queries are divided by it, V's sums at the end.  K's 1024 is what the accumulators start from (-1024 sum of q), a sum that
// cancels to 2^-24 of 1024 sum |q|; from V's codes 1024 + 8 (1024 + 128) is subtracted, which also centres them: a weight's rounding counts for 8
// steps at most.  (The codes are what binds the kernel: ALU operations at half rate, 130 of 340 a block.)
// PK = 2, up to 4 rows: columns 0 .. 3 of an operand belong to a group and columns 4 .. 7 to its neighbour (the queries of the other are zero there),
// so that no lane works for columns without a row; a row's two halves join by a shuffle.
// A row's reference m moves when a score exceeds it by 2^6 (TAU), and 2^ce is kept so that steps times 2^ce are at most 512, the first ones about 8:
// weights times steps then use fp16's range whatever the size of V's entries.
//
// Who takes which blocks: a unit is 8 NT / PK rows of a (batch row, key head).  Short caches: the CTAs of a cluster cut a unit's blocks between them and
// join over the cluster's shared memory.  Else all units' blocks lie in one line that the grid, two CTAs per SM, cuts into equal parts; a CTA's part of
// a unit that others have parts of goes to ws, and the last one to come joins them, in the order of the line.
constexpr int SP_STAGES = 4, SP_WARPS = 8, SP_CLUSTER = 8;
constexpr int sp_per_sm(int hd, int nt) { return hd * nt <= 128 ? 2 : 1; }   // CTAs that 128 or 255 registers a thread leave room for
struct Split {
  Attend a;
  int cols, units, n_blk;        // rows of a (batch row, key head); blocks of a unit (0: the device knows)
  int cluster;                   // CTAs of a cluster, 0: the line
  float *ws;                     // [2 CTA + (part that begins behind the CTA's first block)] of {O [col][hd], m [col], l [col]}
  unsigned *tickets;             // [first CTA of a cut unit], zero between launches
};
template <int HD, int NT> __host__ __device__ constexpr int sp_smem() {
  const int w = SP_WARPS, ring = w * SP_STAGES * block_bytes(HD), out = w * 8 * NT * (HD * 4 + 16) + w * 8 * NT * 8;
  return (ring > out ? ring : out) + 8 * NT * (HD + 4) * 4 + 16;
}
// a block into a stage, by the whole warp
template <int HD> __device__ __forceinline__ void copy_block(uint32_t dst, const char *src, int lane) {
  constexpr int N = block_bytes(HD) / 16;
#pragma unroll
  for (int c = 0; c < N; c += 32)
    if (c + 32 <= N || c + lane < N)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c * 16), "l"(src + c * 16) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {   // 8 x 8 of 16 bits, rows on lanes / 4: transposed
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t m, uint32_t c) {   // (as two constants the compiler takes two operations)
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(m), "r"(c));
  return r;
}
// nibbles i and 4 + i of w as a pair of fp16: 1024 + n for even i, 1024 + 16 n for odd i
__device__ __forceinline__ void open_codes(uint32_t w, uint32_t (&r)[4]) {
  const uint32_t v = w >> 8;
  r[0] = and_or(w, 0x000f000fu, 0x64006400u);
  r[1] = and_or(w, 0x00f000f0u, 0x64006400u);
  r[2] = and_or(v, 0x000f000fu, 0x64006400u);
  r[3] = and_or(v, 0x00f000f0u, 0x64006400u);
}
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t c) {   // pairs of fp16; exact here
  const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <int N> __device__ __forceinline__ void lds_words(const void *p, uint32_t (&w)[N]) {   // in pieces of up to 16 bytes
  if (N == 1) w[0] = *reinterpret_cast<const uint32_t *>(p);
  else if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x; w[1 % N] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[(4 * i) % N] = v.x; w[(4 * i + 1) % N] = v.y; w[(4 * i + 2) % N] = v.z; w[(4 * i + 3) % N] = v.w;
    }
  }
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ld_cluster4(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}

template <typename T, int HD, int NT, int PK>
__global__ void __launch_bounds__(SP_WARPS * 32, sp_per_sm(HD, NT)) attend_split_kernel(const Split p) {
  // a lane's groups: all (PK 1), or those of its half of the columns (PK 2); its heads: columns 2 t and 2 t + 1, of the half
  constexpr int WARPS = SP_WARPS, NG = HD / 32, MG = NG / PK, COLS = 8 * NT / PK, OUT_LD = HD + 4;
  const Attend &a = p.a;
  extern __shared__ __align__(128) unsigned char sp_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int half = PK == 2 ? t >> 1 : 0, tc = PK == 2 ? t & 1 : t;
  unsigned char *ring = sp_raw + warp * SP_STAGES * block_bytes(HD);
  int *last = reinterpret_cast<int *>(sp_raw + sp_smem<HD, NT>() - 16);
  float *sr = reinterpret_cast<float *>(last) - 8 * NT * (HD + 4);   // the CTA's sums [col][hd], m, l and 1 / l [col]
  pdl_launch_dependents();
  pdl_wait();
  const int G = a.n_heads / a.n_kv, col_blocks = (p.cols + COLS - 1) / COLS;
  const int pos0 = a.d_pos ? *a.d_pos : a.pos0;
  const int first = a.d_pos ? (a.window > 0 ? max(0, pos0 + 1 - a.window) : 0) : a.first;
  const int blk0 = first >> 4, n_blk = max(0, ((pos0 + a.S - 1) >> 4) - blk0 + 1);   // of a unit (its own rows may see fewer)
  const long long line = (long long)p.units * n_blk;
  // this CTA's blocks of the line, or of its unit
  const int rank = p.cluster ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
  const long long ctas = min((long long)gridDim.x, (line + WARPS - 1) / WARPS);   // that the line is cut between: none of them without a block
  if (!p.cluster && blockIdx.x >= ctas) return;
  // first block of a CTA, CTA of a block (whole CTAs for a unit where their number divides: a part of its own costs a CTA some 3 us)
  auto start_of = [&](int cta) {
    return line * ctas >> 32 ? line * cta / ctas : (long long)((unsigned)line * (unsigned)cta / (unsigned)ctas);
  };
  auto cta_of = [&](long long x) {
    return line * ctas >> 32 ? (int)(((x + 1) * ctas - 1) / line) : (int)(((unsigned)(x + 1) * (unsigned)ctas - 1u) / (unsigned)line);
  };
  const long long unit_at = (long long)(blockIdx.x / (unsigned)max(1, p.cluster)) * n_blk;
  long long at = p.cluster ? unit_at + n_blk * rank / p.cluster : start_of(blockIdx.x);
  const long long end = p.cluster ? unit_at + n_blk * (rank + 1) / p.cluster : start_of(blockIdx.x + 1);
  // ---- one unit's blocks
#pragma unroll 1
  for (bool again = true; again;) {
  const int unit = p.cluster ? (int)(blockIdx.x / (unsigned)p.cluster) : n_blk ? (int)(at / n_blk) : 0;
  const long long unit0 = (long long)unit * n_blk, stop = min(end, unit0 + n_blk);
  const int c0 = unit % col_blocks * COLS, kvh = unit / col_blocks % a.n_kv, b = unit / col_blocks / a.n_kv;
  const int n_cols = min(COLS, p.cols - c0), pos_lo = pos0 + c0 / G, pos_hi = pos0 + (c0 + n_cols - 1) / G;   // the rows' first and last position
  const int mine0 = blk0 + (int)(at - unit0), n_here = (int)(stop - at);
  const int n_mine = max(0, (n_here - warp + WARPS - 1) / WARPS);   // this warp's blocks: mine0 + warp, + WARPS, ...
  const char *src = reinterpret_cast<const char *>(a.cache) + ((size_t)(b * a.n_kv + kvh) * a.blocks + mine0 + warp) * block_bytes(HD) + lane * 16;
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
#pragma unroll
  for (int i = 0; i < SP_STAGES - 1; i++) {
    if (i < n_mine) copy_block<HD>(ring_at + i * block_bytes(HD), src, lane);
    copies_commit();
    src += WARPS * block_bytes(HD);
  }
  // the rows' queries as operands: column g of n-tile nt, entries 32 j + 8 t .. (PK 2: column g & 3, group j's where g / 4 is j's half and else 0)
  uint32_t qf[NT][NG][4];
  float qs[NT][MG][2], qn[NT][MG][2], sc[NT][2];   // a group's sums of q, and what the products start from; scale log2(e) and the power of two back
  int cpos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int c = c0 + (PK == 2 ? g & 3 : nt * 8 + g), tok = c / G;
    const bool in = c < p.cols;
    const T *q = reinterpret_cast<const T *>(a.q) + b * a.q_batch + (long long)tok * a.q_tok + (size_t)(kvh * G + c - tok * G) * HD + 8 * t;
    uint4 raw[NG];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NG; j++) raw[j] = in ? *reinterpret_cast<const uint4 *>(q + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < NG; j++) {
      float f[8];
      unpack8<T>(raw[j], f);
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(f[i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(141 - (int)(__float_as_uint(top) >> 23), 100);   // 2^14 <= top 2^e < 2^15
    const float up = ldexpf(1.f, e), down = ldexpf(a.scale * 1.4426950408889634f, -e);
    sc[nt][0] = __shfl_sync(0xffffffffu, down, 8 * tc);
    sc[nt][1] = __shfl_sync(0xffffffffu, down, 8 * tc + 4);
#pragma unroll
    for (int j = 0; j < NG; j++) {
      float f[8], sum = 0.f, off = 0.f;
      unpack8<T>(raw[j], f);
#pragma unroll
      for (int i = 0; i < 8; i++) sum += f[i] *= up;
      const bool here = PK == 1 || (j & 1) == g >> 2;
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const uint32_t x = pack2x<__half>(f[2 * h] * (h & 1 ? 0.0625f : 1.f), f[2 * h + 1] * (h & 1 ? 0.0625f : 1.f));
        const float2 y = DT<__half>::unpack2(x);
        off += y.x + y.y;
        qf[nt][j][h] = here ? x : 0u;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      off += __shfl_xor_sync(0xffffffffu, off, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      off += __shfl_xor_sync(0xffffffffu, off, 2);
#pragma unroll
      for (int e2 = 0; e2 < 2; e2++) {
        const float s2 = __shfl_sync(0xffffffffu, sum, 8 * tc + 4 * e2), o2 = -1024.f * __shfl_sync(0xffffffffu, off, 8 * tc + 4 * e2);
        if (PK == 1 || (j & 1) == half) {
          qs[nt][j / PK][e2] = s2;
          qn[nt][j / PK][e2] = o2;
        }
      }
    }
#pragma unroll
    for (int e2 = 0; e2 < 2; e2++) cpos[nt][e2] = pos0 + min(c0 + nt * 8 + 2 * tc + e2, p.cols - 1) / G;
  }
  float o[NT][2 * NG][4] = {}, mid[NT][MG][2] = {}, m[NT][2], l[NT][2] = {};
  float ce = 0.f, step_lim = 0.f;
  constexpr float TAU = 6.f;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -3.402823466e38f;

  auto body = [&](auto edge_, const unsigned char *blk, int key0) {
    constexpr bool EDGE = decltype(edge_)::value;
    float s[NT][4] = {};
    {
      uint32_t kw[2][NG], kp[2][MG];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        lds_words<NG>(blk + ((g + 8 * r) * 4 + t) * NG * 4, kw[r]);
        lds_words<MG>(blk + k_pairs(HD) + ((g + 8 * r) * NG + half * MG) * 4, kp[r]);
      }
#pragma unroll
      for (int w = 0; w < NG / 2; w++) {   // groups 2 w and 2 w + 1
        uint32_t x[2][4], y[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          open_codes(kw[0][2 * w + h], x[h]);
          open_codes(kw[1][2 * w + h], y[h]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint32_t(&q0)[4] = qf[nt][2 * w], (&q1)[4] = qf[nt][2 * w + 1];
          auto join = [&](int i, float(&d)[4]) {   // d: sums of the group that is the lane's i-th word of pairs
            const float2 p0 = open_pair<T>(kp[0][i]), p1 = open_pair<T>(kp[1][i]);
            const int jj = PK == 1 ? 2 * (i % (NG / 2)) + i / (NG / 2) : i;
            s[nt][0] = fmaf(p0.x, d[0], fmaf(p0.y, qs[nt][jj][0], s[nt][0]));
            s[nt][1] = fmaf(p0.x, d[1], fmaf(p0.y, qs[nt][jj][1], s[nt][1]));
            s[nt][2] = fmaf(p1.x, d[2], fmaf(p1.y, qs[nt][jj][0], s[nt][2]));
            s[nt][3] = fmaf(p1.x, d[3], fmaf(p1.y, qs[nt][jj][1], s[nt][3]));
          };
          if constexpr (PK == 2) {   // 8 entries of either group a product
            float d[4] = {qn[nt][w][0], qn[nt][w][1], qn[nt][w][0], qn[nt][w][1]};
#pragma unroll
            for (int h = 0; h < 4; h++) mma16(d, x[0][h], y[0][h], x[1][h], y[1][h], q0[h], q1[h]);
            join(w, d);
          } else {
            float d[4] = {qn[nt][2 * w][0], qn[nt][2 * w][1], qn[nt][2 * w][0], qn[nt][2 * w][1]};
            mma16(d, x[0][0], y[0][0], x[0][1], y[0][1], q0[0], q0[1]);
            mma16(d, x[0][2], y[0][2], x[0][3], y[0][3], q0[2], q0[3]);
            join(w, d);
            float f[4] = {qn[nt][2 * w + 1][0], qn[nt][2 * w + 1][1], qn[nt][2 * w + 1][0], qn[nt][2 * w + 1][1]};
            mma16(f, x[1][0], y[1][0], x[1][1], y[1][1], q1[0], q1[1]);
            mma16(f, x[1][2], y[1][2], x[1][3], y[1][3], q1[2], q1[3]);
            join(NG / 2 + w, f);
          }
        }
      }
      if (PK == 2)
#pragma unroll
        for (int i = 0; i < 4; i++) s[0][i] += __shfl_xor_sync(0xffffffffu, s[0][i], 2);
    }
    uint32_t vp[2][MG];
    uint32_t step_bits = 0;
#pragma unroll
    for (int r = 0; r < 2; r++) {
      lds_words<MG>(blk + v_pairs(HD) + ((g + 8 * r) * NG + half * MG) * 4, vp[r]);
      const bool seen = !EDGE || (key0 + g + 8 * r >= first && key0 + g + 8 * r <= pos_hi);   // by any row: the others' steps say nothing
#pragma unroll
      for (int i = 0; i < MG; i++) vp[r][i] = seen ? vp[r][i] : 0u;
#pragma unroll
      for (int i = 0; i < MG; i++) step_bits = max(step_bits, __float_as_uint(open_pair<T>(vp[r][i]).x));   // no step is negative; NaN is the largest
    }
    // scores less their reference, in powers of two
    float far = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (EDGE) {
          const int key = key0 + g + 8 * (i >> 1);
          if (key < first || key > cpos[nt][i & 1]) s[nt][i] = -INFINITY;
        }
        far = fmaxf(far, fmaf(s[nt][i], sc[nt][i & 1], -m[nt][i & 1]));
      }
    if (__any_sync(0xffffffffu, far > TAU || step_bits > __float_as_uint(step_lim))) {
      uint32_t top = 0;
#pragma unroll
      for (int r = 0; r < 2; r++)
#pragma unroll
        for (int i = 0; i < MG; i++) {
          const uint32_t st = __float_as_uint(open_pair<T>(vp[r][i]).x);
          if (st < 0x7f800000u) top = max(top, st);
        }
      top = __reduce_max_sync(0xffffffffu, top);
      float up = 0.f;   // change of ce
      if (top > __float_as_uint(step_lim)) {
        const float e = fminf(fmaxf(130.f - (float)(top >> 23), -100.f), 100.f);   // 8 <= top 2^e < 16
        up = e - ce;
        ce = e;
        step_lim = ex2(9.f - e);
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = fmaxf(s[nt][e], s[nt][2 + e]) * sc[nt][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float mn = fmaxf(m[nt][e], mx), f = ex2(m[nt][e] - mn + up);
          m[nt][e] = mn;
          l[nt][e] *= f;
#pragma unroll
          for (int j = 0; j < MG; j++) mid[nt][j][e] *= f;
#pragma unroll
          for (int j = 0; j < 2 * NG; j++) {
            o[nt][j][e] *= f;
            o[nt][j][2 + e] *= f;
          }
        }
      }
    }
    uint32_t vw[2 * NG];
#pragma unroll
    for (int i = 0; i < NG / 2; i++) {
      const uint4 v = reinterpret_cast<const uint4 *>(blk + v_codes(HD))[i * 32 + lane];
      vw[4 * i] = v.x; vw[4 * i + 1] = v.y; vw[4 * i + 2] = v.z; vw[4 * i + 3] = v.w;
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[nt][i] = ex2(fmaf(s[nt][i], sc[nt][i & 1], ce - m[nt][i & 1]));
        l[nt][i & 1] += s[nt][i];
      }
    auto times = [](float w, float x) { return EDGE && w == 0.f ? 0.f : w * x; };   // a key that a row does not see may be anything
#pragma unroll
    for (int w = 0; w < NG / 2; w++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        uint32_t b0[2], b1[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (PK == 2 && h) {
            b0[1] = b0[0];
            b1[1] = b1[0];
            continue;
          }
          const int i = PK == 2 ? w : h * (NG / 2) + w;   // the pair's word; its sums' place
          const int jj = PK == 2 ? w : 2 * w + h;
          const float2 p0 = open_pair<T>(vp[0][i]), p1 = open_pair<T>(vp[1][i]);
          const float m0 = fmaf(8.f, p0.x, p0.y), m1 = fmaf(8.f, p1.x, p1.y);
          b0[h] = turn8x8(pack2x<__half>(times(s[nt][0], p0.x), times(s[nt][1], p0.x)));
          b1[h] = turn8x8(pack2x<__half>(times(s[nt][2], p1.x), times(s[nt][3], p1.x)));
          mid[nt][jj][0] += times(s[nt][0], m0);
          mid[nt][jj][0] += times(s[nt][2], m1);
          mid[nt][jj][1] += times(s[nt][1], m0);
          mid[nt][jj][1] += times(s[nt][3], m1);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t x[4], y[4];
          open_codes(vw[2 * w + h], x);
          open_codes(vw[NG + 2 * w + h], y);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            x[e] = add2(x[e], e & 1 ? 0xe480e480u : 0xe408e408u);   // -(1024 + 16 * 8), -(1024 + 8)
            y[e] = add2(y[e], e & 1 ? 0xe480e480u : 0xe408e408u);
          }
          float(&u)[4] = o[nt][2 * (2 * w + h)], (&v)[4] = o[nt][2 * (2 * w + h) + 1];
          mma16(u, x[0], x[1], y[0], y[1], b0[h], b1[h]);
          mma16(v, x[2], x[3], y[2], y[3], b0[h], b1[h]);
        }
      }
  };
  for (int i = 0, st = 0; i < n_mine; i++) {
    copies_wait<SP_STAGES - 2>();
    __syncwarp();   // block i is there; every lane has read the block in front of it, whose stage takes the next copy
    if (i + SP_STAGES - 1 < n_mine) copy_block<HD>(ring_at + (st == 0 ? SP_STAGES - 1 : st - 1) * block_bytes(HD), src, lane);
    copies_commit();
    src += WARPS * block_bytes(HD);
    const unsigned char *blk = ring + st * block_bytes(HD);
    st = st == SP_STAGES - 1 ? 0 : st + 1;
    const int key0 = (mine0 + warp + i * WARPS) * 16;
    if (key0 > pos_hi) ;   // only later rows of the call see it
    else if (key0 < first || key0 + 15 > pos_lo) body(std::true_type{}, blk, key0);
    else body(std::false_type{}, blk, key0);
  }
  copies_wait<0>();

  // ---- the warp's sums, then the CTA's -------------------------------------------------------------------------------
#pragma unroll
  for (int x = 4; x < 32; x <<= 1)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
#pragma unroll
        for (int j = 0; j < MG; j++) mid[nt][j][e] += __shfl_xor_sync(0xffffffffu, mid[nt][j][e], x);
      }
  __syncthreads();   // every ring is free
  constexpr int PART = COLS * (HD + 2);
  float *so = reinterpret_cast<float *>(sp_raw);                       // [warp][col][OUT_LD]
  float *sm = so + WARPS * COLS * OUT_LD, *sl = sm + WARPS * COLS;     // [warp][col]
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = nt * 8 + 2 * tc + e;
      if (g == 0 && half == 0) {
        sm[warp * COLS + col] = l[nt][e] == 0.f ? -INFINITY : m[nt][e] - ce;
        sl[warp * COLS + col] = l[nt][e];
      }
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const float z = mid[nt][j / PK][e];
        if (PK == 1 || (j & 1) == half)
          *reinterpret_cast<float4 *>(&so[(warp * COLS + col) * OUT_LD + 32 * j + 4 * g]) =
              make_float4(o[nt][2 * j][e] + z, fmaf(0.0625f, o[nt][2 * j][2 + e], z), o[nt][2 * j + 1][e] + z, fmaf(0.0625f, o[nt][2 * j + 1][2 + e], z));
      }
    }
  __syncthreads();
  const bool whole = p.cluster ? p.cluster == 1 : n_here == n_blk;   // nobody else has a part
  if (threadIdx.x < COLS) {
    const int col = threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm[w * COLS + col]);
    for (int w = 0; w < WARPS; w++) {
      const float f = sm[w * COLS + col] == -INFINITY ? 0.f : ex2(sm[w * COLS + col] - M);
      L += f * sl[w * COLS + col];
      sm[w * COLS + col] = f;
    }
    sr[COLS * HD + col] = M;
    sr[COLS * HD + COLS + col] = L;
    sr[COLS * HD + 2 * COLS + col] = L == 0.f ? 0.f : 1.f / L;
  }
  __syncthreads();
  auto put = [&](int col, int d, const float (&v)[4], float f) {
    const int c = c0 + col, tok = c / G;
    T *y = reinterpret_cast<T *>(a.out) + ((size_t)(b * (long long)a.S + tok) * a.n_heads + kvh * G + c - tok * G) * HD + d;
    *reinterpret_cast<uint2 *>(y) = make_uint2(pack2x<T>(v[0] * f, v[1] * f), pack2x<T>(v[2] * f, v[3] * f));
  };
  // parts of this unit, where there are several: CTAs first_cta .., in the line
  const int first_cta = whole || p.cluster ? 0 : cta_of(unit0), parts = whole || p.cluster ? 1 : cta_of(unit0 + n_blk - 1) - first_cta + 1;
  const bool behind = !whole && start_of(first_cta) < unit0;   // the first CTA has blocks of another unit in front
  auto slot_of = [&](int cta) { return p.ws + (size_t)(2 * cta + (cta == first_cta && behind ? 1 : 0)) * PART; };
  float *part = whole || p.cluster ? sr : slot_of(blockIdx.x);
  const int items = n_cols * (HD / 4);
  for (int i = threadIdx.x; i < items; i += WARPS * 32) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float v[4] = {};
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = sm[w * COLS + col];
      const float4 x = *reinterpret_cast<const float4 *>(&so[(w * COLS + col) * OUT_LD + d]);
      if (f != 0.f) {
        v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
      }
    }
    if (whole) put(col, d, v, sr[COLS * HD + 2 * COLS + col]);
    else *reinterpret_cast<float4 *>(&part[col * HD + d]) = make_float4(v[0], v[1], v[2], v[3]);
  }
  if (p.cluster > 1) {
    // ---- the cluster's CTAs take an equal share of the results each; neighbouring lanes read the parts of one ---------------
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const int P = p.cluster, who = lane & (P - 1);
    const uint32_t theirs = cluster_map(smem_u32(sr), (uint32_t)who);
    for (int i0 = 0; i0 < items; i0 += WARPS * 32) {   // (the same trips for every lane)
      const int i = i0 + (int)threadIdx.x / P * P + rank, at_col = min(i, items - 1) / (HD / 4), d = min(i, items - 1) % (HD / 4) * 4;
      const float mm = ld_cluster(theirs + (COLS * HD + at_col) * 4);
      float L = ld_cluster(theirs + (COLS * HD + COLS + at_col) * 4), v[4];
      ld_cluster4(theirs + (at_col * HD + d) * 4, v);
      float M = mm;
      for (int o2 = 1; o2 < P; o2 <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o2));
      const float f = mm == -INFINITY ? 0.f : ex2(mm - M);
      L *= f;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = f == 0.f ? 0.f : v[e] * f;
      for (int o2 = 1; o2 < P; o2 <<= 1) {
        L += __shfl_xor_sync(0xffffffffu, L, o2);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += __shfl_xor_sync(0xffffffffu, v[e], o2);
      }
      if (who == 0 && i < items) put(at_col, d, v, L == 0.f ? 0.f : 1.f / L);
    }
    __syncwarp();
    cluster_arrive();   // nobody leaves while its parts are read
    cluster_wait();
  } else if (!whole) {
    // ---- the last CTA of a unit joins its parts, in their order -----------------------------------------------------------
    if (threadIdx.x < 2 * COLS) part[COLS * HD + threadIdx.x] = sr[COLS * HD + threadIdx.x];
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *last = atomicAdd(&p.tickets[first_cta], 1u) == (unsigned)parts - 1;
    __syncthreads();
    if (*last) {
      __threadfence();
      // a share of the parts for each of `teams` threads of a result
      int teams = 1;
      while (2 * teams * items <= WARPS * 32 && 2 * teams <= parts) teams *= 2;
      const int i = threadIdx.x % items, team = threadIdx.x / items;
      for (int i1 = i; i1 < items && team < teams; i1 += teams == 1 ? WARPS * 32 : items) {
        const int col = i1 / (HD / 4), d = i1 % (HD / 4) * 4, p0 = parts * team / teams, p1 = parts * (team + 1) / teams;
        float M = -INFINITY, L = 0.f, v[4] = {};
#pragma unroll 4
        for (int s = p0; s < p1; s++) {   // (the running maximum keeps the loads of four parts on their way together)
          const float *x = slot_of(first_cta + s);
          const float mm = __ldcg(x + COLS * HD + col), ll = __ldcg(x + COLS * HD + COLS + col);
          const float4 y = __ldcg(reinterpret_cast<const float4 *>(x + col * HD + d));
          const float mn = fmaxf(M, mm), f0 = M == -INFINITY ? 0.f : ex2(M - mn), f1 = mm == -INFINITY ? 0.f : ex2(mm - mn);
          M = mn;
          L = L * f0 + ll * f1;
          if (f1 != 0.f) {
            v[0] = v[0] * f0 + y.x * f1; v[1] = v[1] * f0 + y.y * f1; v[2] = v[2] * f0 + y.z * f1; v[3] = v[3] * f0 + y.w * f1;
          }
        }
        if (teams == 1) put(col, d, v, L == 0.f ? 0.f : 1.f / L);
        else {
          float *x = so + (size_t)(team * items + i1) * 8;
          *reinterpret_cast<float4 *>(x) = make_float4(v[0], v[1], v[2], v[3]);
          x[4] = M;
          x[5] = L;
        }
      }
      if (teams > 1) {
        __syncthreads();
        if ((int)threadIdx.x < items) {
          const int col = threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4) * 4;
          float M = -INFINITY, L = 0.f, v[4] = {};
          for (int s = 0; s < teams; s++) M = fmaxf(M, so[(size_t)(s * items + threadIdx.x) * 8 + 4]);
          for (int s = 0; s < teams; s++) {
            const float *x = so + (size_t)(s * items + threadIdx.x) * 8;
            if (x[4] == -INFINITY) continue;
            const float f = ex2(x[4] - M);
            L = fmaf(f, x[5], L);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = fmaf(f, x[e], v[e]);
          }
          put(col, d, v, L == 0.f ? 0.f : 1.f / L);
        }
      }
      if (threadIdx.x == 0) p.tickets[first_cta] = 0;   // for the next launch
    }
  }
  at = stop;
  again = !p.cluster && at < end;
  if (again) __syncthreads();   // the ring takes copies again
  }
}

template <typename F> static int by_type(int dtype, int hd, F &&f) {
  if (dtype) {
    if (hd == 64) return f(__half{}, std::integral_constant<int, 64>{});
    if (hd == 128) return f(__half{}, std::integral_constant<int, 128>{});
    return f(__half{}, std::integral_constant<int, 256>{});
  }
  if (hd == 64) return f(__nv_bfloat16{}, std::integral_constant<int, 64>{});
  if (hd == 128) return f(__nv_bfloat16{}, std::integral_constant<int, 128>{});
  return f(__nv_bfloat16{}, std::integral_constant<int, 256>{});
}

int write(cudaStream_t s, int dtype, const Write &a, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    const long long warps = ((long long)a.B * a.S * (a.n_q + 2 * a.n_kv) * (a.hd / 8) + 31) / 32;
    return launch(s, launches, write_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, 1, a);
  });
}
int read(cudaStream_t s, int dtype, const Read &a, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    const long long warps = ((long long)a.B * a.n_kv * a.n * (a.hd / 8) + 31) / 32;
    return launch(s, launches, read_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, 1, a);
  });
}
// The form of a call: 4, 8 or 16 rows a CTA (heads of 256 entries: 4 or 8, whose sums fill the registers), and as many CTAs per (batch row, key head,
// rows) as are resident together, with a block for every warp.
template <typename T, int HD, int NT, int PK> static int attend_split(cudaStream_t s, const Attend &a, const Scratch &x, uint64_t *launches) {
  constexpr int COLS = 8 * NT / PK;
  Split p{a};
  p.cols = a.S * (a.n_heads / a.n_kv);
  p.ws = x.ws; p.tickets = x.tickets;
  const long long units = (long long)a.B * a.n_kv * ((p.cols + COLS - 1) / COLS), slots = (long long)x.sms * sp_per_sm(HD, NT);
  const int n_blk = a.d_pos ? a.blocks : std::max(1, (a.pos0 + a.S - 1) / BLOCK - a.first / BLOCK + 1);
  p.units = (int)units;
  int cluster = 1;
  while (cluster < SP_CLUSTER && cluster * SP_WARPS < n_blk && units * 2 * cluster <= slots) cluster *= 2;
  // Microseconds of either way behind what both cost: a block takes a quarter of an SM 0.3 (hd 128, 8 columns), a CTA alone twice as long a warp; parts
  // in the line cost 8, or 5 where no CTA has parts of two units (one token, 32 / 8 heads, 128 entries, cluster and line: batch 1 at 4096 positions 8.8,
  // 11.2 us, at 16384 16.3, 14.4; batch 4 at 16384 24.9, 27.9; batch 16 at 4096 24.1, 28.6, at 16384 75, 73)
  const double each = 0.3 * std::max(1.0, HD * NT / 128.0), ctas = (double)((units * cluster + x.sms - 1) / x.sms);
  const bool line = each * units * n_blk / (4.0 * x.sms) + (slots % units ? 8 : 5) < 2 * each * ctas * n_blk / (SP_WARPS * cluster);
  if (!line) p.cluster = cluster;
  const long long grid = line ? std::min<long long>(slots, (units * n_blk + SP_WARPS - 1) / SP_WARPS) : units * cluster;
  return launch(s, launches, attend_split_kernel<T, HD, NT, PK>, dim3((unsigned)grid), dim3(SP_WARPS * 32),
                // (few clusters: so much shared memory that their CTAs come to lie on an SM each; 16384 positions 20.2 -> 16.8 us)
                !line && 2 * grid <= x.sms ? (size_t)std::max(sp_smem<HD, NT>(), 120 * 1024) : (size_t)sp_smem<HD, NT>(), line ? 1 : cluster, p);
}
int attend(cudaStream_t s, int dtype, const Attend &a, const Scratch &x, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    constexpr int HD = hd.value;
    const long long cols = (long long)a.S * (a.n_heads / a.n_kv);
    if (cols <= 4) return attend_split<T, HD, 1, 2>(s, a, x, launches);
    if (HD == 256 || cols <= 8) return attend_split<T, HD, 1, 1>(s, a, x, launches);
    return attend_split<T, HD, HD == 256 ? 1 : 2, 1>(s, a, x, launches);
  });
}
// two parts a CTA, two CTAs per SM
size_t scratch_floats(int sms) { return (size_t)sms * 4 * 16 * (256 + 2); }
size_t scratch_tickets(int sms) { return (size_t)sms * 2; }
template <typename T, int HD, int NT, int PK> static int big_smem() {
  cudaError_t e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT, PK>, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(sp_smem<HD, NT>(), 120 * 1024));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT, PK>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT, PK>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return (int)e;
}
int prepare(int dtype, int hd) {
  return by_type(dtype, hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    constexpr int HD = hd.value;
    int e = big_smem<T, HD, 1, 2>();
    if (!e) e = big_smem<T, HD, 1, 1>();
    if (!e) e = big_smem<T, HD, HD == 256 ? 1 : 2, 1>();
    return e;
  });
}

}  // namespace pc
}  // namespace cake
