// packed_cache.cu — kernels of the cache in four bits (format and interface: packed_cache.cuh)
#include "packed_cache.cuh"
#include "common.cuh"

#include <algorithm>
#include <type_traits>

namespace cake {
namespace pc {

template <typename... KArgs, typename... Args>
static int launch(cudaStream_t s, uint64_t *launches, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
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
  constexpr int LPR = HD / 8, NG = HD / 32;
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
  const uint32_t theirs = __shfl_xor_sync(0xffffffffu, w, 4);   // V: the neighbouring group's codes of the same quarter
  if (is_q || !in) return;
  char *blk = reinterpret_cast<char *>(a.cache) + ((size_t)(b * a.n_kv + h) * a.blocks + (pos >> 4)) * block_bytes(HD);
  const int r = pos & 15, j = u >> 2, q = u & 3;
  if (!is_v) {
    // entry 2i to nibble i, entry 2i + 1 to nibble 4 + i
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) k |= (w >> (8 * i) & 15u) << (4 * i) | (w >> (8 * i + 4) & 15u) << (16 + 4 * i);
    reinterpret_cast<uint32_t *>(blk)[k_word(HD, r, u)] = k;
    if (q == 0) reinterpret_cast<uint32_t *>(blk + k_pairs(HD))[r * NG + j] = pair;
  } else {
    const uint32_t o = (j & 1) ? (theirs >> 16) | (w & 0xffff0000u) : (w & 0xffffu) | (theirs << 16);
    reinterpret_cast<uint32_t *>(blk + v_codes(HD))[v_word(HD, r, 2 * q + (j & 1), j >> 1)] = o;
    if (q == 0) reinterpret_cast<uint32_t *>(blk + v_pairs(HD))[r * NG + j] = pair;
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
  const int j = u >> 2, q = u & 3, sh = 16 * (j & 1);
  const uint32_t *v = reinterpret_cast<const uint32_t *>(blk + v_codes(HD));
  return (v[v_word(HD, r, 2 * q, j >> 1)] >> sh & 0xffffu) | (v[v_word(HD, r, 2 * q + 1, j >> 1)] >> sh) << 16;
}

template <typename T, int HD>
__global__ void __launch_bounds__(128) read_kernel(const Read a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LPR = HD / 8, NG = HD / 32;
  const int lane = threadIdx.x & 31, u = lane % LPR;
  const long long row = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * (32 / LPR) + lane / LPR;
  if (row >= (long long)a.B * a.n_kv * a.n) return;
  const int i = (int)(row % a.n), slab = (int)(row / a.n), pos = a.first + i, r = pos & 15;
  const char *blk = reinterpret_cast<const char *>(a.cache) + ((size_t)slab * a.blocks + (pos >> 4)) * block_bytes(HD);
  const uint32_t w = codes8<HD>(blk, a.which, r, u);
  const float2 p = open_pair<T>(reinterpret_cast<const uint32_t *>(blk + (a.which ? v_pairs(HD) : k_pairs(HD)))[r * NG + (u >> 2)]);
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    o[e] = pack2x<T>(fmaf(p.x, (float)(w >> (8 * e) & 15u), p.y), fmaf(p.x, (float)(w >> (8 * e + 4) & 15u), p.y));
  *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + ((size_t)slab * a.out_rows + i) * HD + 8 * u) = make_uint4(o[0], o[1], o[2], o[3]);
}

// ------------------------------------------------------------------------------------------ attention of a few rows, keys split
// A CTA serves 8 NT query rows (row = token G + head of one key head) and a range of blocks; its warps take the blocks in turn, each through a ring of
// its own (one bulk copy a block: codes and pairs of K and V), so that no warp waits for another until the end.  Per block, with m16n8k16 products:
//   S^T = K Q^T   A: 16 keys' codes as D numbers, B: the rows' queries, kept in registers.  A group's sum is taken apart from the others', then
//                 s += step sum + lo (sum of the group's q): the codes go in exactly, and no entry is formed.  bf16 holds 128 + n without an
//                 instruction for the 128: the accumulator starts at -128 (sum of q).
//   O^T += V^T P  A: 16 entries' codes n - 8 in fp16, B: weights times steps in fp16 (11 bits), one operand per group; what is left of
//                 the value, lo + 8 step, is a number per key and group and is summed in fp32.  P^T turns into an operand by movmatrix.
// A row's reference m moves when a score exceeds it by 2^6 (tau), and 2^ce is kept so that steps times 2^ce are at most 512, the first ones about 8:
// weights times steps then use fp16's range whatever the size of V's entries.
constexpr int SP_WARPS = 8, SP_STAGES = 4;
struct Split {
  Attend a;
  int cols, splits;              // rows of a (batch row, key head), CTAs that cut their keys
  float *ws;                     // splits > 1: [unit][split] of {O [col][hd], m [col], l [col]}
  unsigned *tickets;             // [unit], zero between launches
  int *err;
};
template <int HD, int NT> __host__ __device__ constexpr int sp_smem() {
  const int ring = SP_WARPS * SP_STAGES * block_bytes(HD), out = SP_WARPS * 8 * NT * (HD * 4 + 16) + SP_WARPS * 8 * NT * 8;
  return (ring > out ? ring : out) + 64 * NT + SP_WARPS * SP_STAGES * 8 + 16;
}
__device__ __forceinline__ void bulk_in(void *dst, const void *src, uint32_t bytes, uint64_t *bar, uint32_t yes) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t@p cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar)), "r"(yes)
               : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                                            float c1, float c2, float c3);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                                     float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2,
                                              float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {   // 8 x 8 of 16 bits, rows on lanes / 4: transposed
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t add2(uint32_t a, float c) {   // fp16: a + c, exact here
  const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&a), __float2half2_rn(c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, float m, float c) {   // fp16: a m + c, exact here
  const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), __float2half2_rn(m), __float2half2_rn(c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
// nibbles i and 4 + i of w as a pair of fp16, n + c each (1024 + n, or 1024 + 16 n, by their bits)
__device__ __forceinline__ void pairs_f16(uint32_t w, float c, uint32_t (&r)[4]) {
  const uint32_t v = w >> 8;
  r[0] = add2((w & 0x000f000fu) | 0x64006400u, c - 1024.f);
  r[1] = fma2((w & 0x00f000f0u) | 0x64006400u, 0.0625f, c - 64.f);
  r[2] = add2((v & 0x000f000fu) | 0x64006400u, c - 1024.f);
  r[3] = fma2((v & 0x00f000f0u) | 0x64006400u, 0.0625f, c - 64.f);
}
// K's codes as numbers of D: fp16 n, bf16 128 + n
template <typename T> struct KCode;
template <> struct KCode<__half> {
  static constexpr float off = 0.f;
  static __device__ __forceinline__ void open(uint32_t w, uint32_t (&r)[4]) { pairs_f16(w, 0.f, r); }
};
template <> struct KCode<__nv_bfloat16> {
  static constexpr float off = 128.f;
  static __device__ __forceinline__ void open(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  }
};
template <int N> __device__ __forceinline__ void lds_words(const void *p, uint32_t (&w)[N]) {   // N = 2: 8 bytes, else pieces of 16
  if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(SP_WARPS * 32, HD * NT <= 128 ? 2 : 1) attend_split_kernel(const Split p) {
  constexpr int NG = HD / 32, COLS = 8 * NT, OUT_LD = HD + 4;
  const Attend &a = p.a;
  extern __shared__ __align__(128) unsigned char sp_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned char *ring = sp_raw + warp * SP_STAGES * block_bytes(HD);
  uint64_t *bars = reinterpret_cast<uint64_t *>(sp_raw + sp_smem<HD, NT>() - SP_WARPS * SP_STAGES * 8 - 16);
  int *last = reinterpret_cast<int *>(bars + SP_WARPS * SP_STAGES);
  uint64_t *bar = bars + warp * SP_STAGES;
  if (lane == 0) {
    for (int i = 0; i < SP_STAGES; i++) mbar_init(&bar[i], 1);
    mbar_fence_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  const int G = a.n_heads / a.n_kv, col_blocks = (p.cols + COLS - 1) / COLS;
  const int split = (int)(blockIdx.x % (unsigned)p.splits), unit = (int)(blockIdx.x / (unsigned)p.splits);
  const int c0 = unit % col_blocks * COLS, kvh = unit / col_blocks % a.n_kv, b = unit / col_blocks / a.n_kv;
  const int pos0 = a.d_pos ? *a.d_pos : a.pos0;
  const int first = a.d_pos ? (a.window > 0 ? max(0, pos0 + 1 - a.window) : 0) : a.first;
  const int n_cols = min(COLS, p.cols - c0), pos_lo = pos0 + c0 / G, pos_hi = pos0 + (c0 + n_cols - 1) / G;   // the rows' first and last position
  const int blk0 = first >> 4, n_blk = first <= pos_hi ? (pos_hi >> 4) - blk0 + 1 : 0;
  const int mine0 = blk0 + (int)((long long)n_blk * split / p.splits), mine1 = blk0 + (int)((long long)n_blk * (split + 1) / p.splits);
  const int n_mine = max(0, (mine1 - mine0 - warp + SP_WARPS - 1) / SP_WARPS);   // this warp's blocks: mine0 + warp, + SP_WARPS, ...
  const char *src = reinterpret_cast<const char *>(a.cache) + ((size_t)(b * a.n_kv + kvh) * a.blocks + mine0 + warp) * block_bytes(HD);
  int left = MBAR_TRIES;
  if (lane == 0)
    for (int i = 0; i < min(SP_STAGES, n_mine); i++) {
      mbar_arrive_expect_tx(&bar[i], block_bytes(HD));
      bulk_in(ring + i * block_bytes(HD), src + (size_t)i * SP_WARPS * block_bytes(HD), block_bytes(HD), &bar[i], 1u);
    }
  // the rows' queries: column g of n-tile nt, entries 32 j + 8 t ..; sums of a group for columns 2t and 2t + 1
  uint4 qf[NT][NG];
  float qs[NT][NG][2];
  int cpos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int c = c0 + nt * 8 + g, tok = c / G;
    const bool in = c < p.cols;
    const T *q = reinterpret_cast<const T *>(a.q) + b * a.q_batch + (long long)tok * a.q_tok + (size_t)(kvh * G + c - tok * G) * HD + 8 * t;
#pragma unroll
    for (int j = 0; j < NG; j++) {
      qf[nt][j] = in ? *reinterpret_cast<const uint4 *>(q + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
      float f[8], sum = 0.f;
      unpack8<T>(qf[nt][j], f);
#pragma unroll
      for (int i = 0; i < 8; i++) sum += f[i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qs[nt][j][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
      qs[nt][j][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
    }
#pragma unroll
    for (int e = 0; e < 2; e++) cpos[nt][e] = pos0 + min(c0 + nt * 8 + 2 * t + e, p.cols - 1) / G;
  }
  float o[NT][2 * NG][4] = {}, mid[NT][NG][2] = {}, m[NT][2], l[NT][2] = {};
  float ce = 0.f, step_lim = 0.f;
  constexpr float TAU = 6.f;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -3.402823466e38f;
  const float sc = a.scale * 1.4426950408889634f;

  auto body = [&](auto edge_, const unsigned char *blk, int key0) {
    constexpr bool EDGE = decltype(edge_)::value;
    float s[NT][4] = {};
    {
      uint32_t kw[2][NG], kp[2][NG];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        lds_words<NG>(blk + ((g + 8 * r) * 4 + t) * NG * 4, kw[r]);
        lds_words<NG>(blk + k_pairs(HD) + (g + 8 * r) * NG * 4, kp[r]);
      }
#pragma unroll
      for (int j = 0; j < NG; j++) {
        uint32_t x[4], y[4];
        KCode<T>::open(kw[0][j], x);
        KCode<T>::open(kw[1][j], y);
        const float2 p0 = open_pair<T>(kp[0][j]), p1 = open_pair<T>(kp[1][j]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float d[4];
          const float n0 = -KCode<T>::off * qs[nt][j][0], n1 = -KCode<T>::off * qs[nt][j][1];
          mma16<T>(d, x[0], y[0], x[1], y[1], qf[nt][j].x, qf[nt][j].y, n0, n1, n0, n1);
          mma16<T>(d, x[2], y[2], x[3], y[3], qf[nt][j].z, qf[nt][j].w, d[0], d[1], d[2], d[3]);
          s[nt][0] = fmaf(p0.x, d[0], fmaf(p0.y, qs[nt][j][0], s[nt][0]));
          s[nt][1] = fmaf(p0.x, d[1], fmaf(p0.y, qs[nt][j][1], s[nt][1]));
          s[nt][2] = fmaf(p1.x, d[2], fmaf(p1.y, qs[nt][j][0], s[nt][2]));
          s[nt][3] = fmaf(p1.x, d[3], fmaf(p1.y, qs[nt][j][1], s[nt][3]));
        }
      }
    }
    uint32_t vp[2][NG];
    float step_max = 0.f;
#pragma unroll
    for (int r = 0; r < 2; r++) {
      lds_words<NG>(blk + v_pairs(HD) + (g + 8 * r) * NG * 4, vp[r]);
      const bool seen = !EDGE || (key0 + g + 8 * r >= first && key0 + g + 8 * r <= pos_hi);   // by any row: the others' steps say nothing
#pragma unroll
      for (int j = 0; j < NG; j++) vp[r][j] = seen ? vp[r][j] : 0u;
#pragma unroll
      for (int j = 0; j < NG; j++) step_max = fmaxf(step_max, open_pair<T>(vp[r][j]).x);
    }
    bool over = step_max > step_lim;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[nt][i] *= sc;
        if (EDGE) {
          const int key = key0 + g + 8 * (i >> 1);
          if (key < first || key > cpos[nt][i & 1]) s[nt][i] = -INFINITY;
        }
        over = over || s[nt][i] > m[nt][i & 1] + TAU;
      }
    if (__any_sync(0xffffffffu, over)) {
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(step_max)));   // (no step is negative; fmaxf drops NaN)
      float up = 0.f;   // change of ce
      if (top > step_lim && top <= 3.402823466e38f) {
        const float e = fminf(fmaxf(130.f - (float)(__float_as_uint(top) >> 23), -100.f), 100.f);   // 8 <= top 2^e < 16
        up = e - ce;
        ce = e;
        step_lim = ex2(9.f - e);
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float mn = fmaxf(m[nt][e], mx), f = ex2(m[nt][e] - mn + up);
          m[nt][e] = mn;
          l[nt][e] *= f;
#pragma unroll
          for (int j = 0; j < NG; j++) mid[nt][j][e] *= f;
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
        s[nt][i] = ex2(s[nt][i] - (m[nt][i & 1] - ce));
        l[nt][i & 1] += s[nt][i];
      }
    auto times = [](float w, float x) { return EDGE && w == 0.f ? 0.f : w * x; };   // a key that a row does not see may be anything
#pragma unroll
    for (int w = 0; w < NG / 2; w++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int j = 2 * w + h;
        uint32_t x[4], y[4];
        pairs_f16(__byte_perm(vw[w], vw[NG / 2 + w], h ? 0x7632 : 0x5410), -8.f, x);
        pairs_f16(__byte_perm(vw[NG + w], vw[3 * NG / 2 + w], h ? 0x7632 : 0x5410), -8.f, y);
        const float2 p0 = open_pair<T>(vp[0][j]), p1 = open_pair<T>(vp[1][j]);
        const float m0 = fmaf(8.f, p0.x, p0.y), m1 = fmaf(8.f, p1.x, p1.y);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint32_t b0 = turn8x8(pack2x<__half>(times(s[nt][0], p0.x), times(s[nt][1], p0.x)));
          const uint32_t b1 = turn8x8(pack2x<__half>(times(s[nt][2], p1.x), times(s[nt][3], p1.x)));
          float(&u)[4] = o[nt][2 * j], (&v)[4] = o[nt][2 * j + 1];
          mma16<__half>(u, x[0], x[1], y[0], y[1], b0, b1, u[0], u[1], u[2], u[3]);
          mma16<__half>(v, x[2], x[3], y[2], y[3], b0, b1, v[0], v[1], v[2], v[3]);
          mid[nt][j][0] += times(s[nt][0], m0) + times(s[nt][2], m1);
          mid[nt][j][1] += times(s[nt][1], m0) + times(s[nt][3], m1);
        }
      }
  };
  for (int i = 0; i < n_mine; i++) {
    const int st = i % SP_STAGES;
    mbar_wait_lim(&bar[st], (uint32_t)(i / SP_STAGES) & 1u, p.err, left);
    const unsigned char *blk = ring + st * block_bytes(HD);
    const int key0 = (mine0 + warp + i * SP_WARPS) * 16;
    if (key0 < first || key0 + 15 > pos_lo) body(std::true_type{}, blk, key0);
    else body(std::false_type{}, blk, key0);
    __syncwarp();   // every lane has read the stage
    if (lane == 0 && i + SP_STAGES < n_mine) {
      mbar_arrive_expect_tx_if(left, &bar[st], block_bytes(HD));
      bulk_in(ring + st * block_bytes(HD), src + (size_t)(i + SP_STAGES) * SP_WARPS * block_bytes(HD), block_bytes(HD), &bar[st], left);
    }
  }
  // a warp that gave up lets its copies end before its ring is anything else
  if (!__all_sync(0xffffffffu, left != 0) && lane == 0)
    for (int i = max(0, n_mine - SP_STAGES); i < n_mine; i++) mbar_drain(&bar[i % SP_STAGES], (uint32_t)(i / SP_STAGES) & 1u);

  // ---- the warp's sums, then the CTA's -------------------------------------------------------------------------------
#pragma unroll
  for (int x = 4; x < 32; x <<= 1)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
#pragma unroll
        for (int j = 0; j < NG; j++) mid[nt][j][e] += __shfl_xor_sync(0xffffffffu, mid[nt][j][e], x);
      }
  __syncthreads();   // every ring is free
  float *so = reinterpret_cast<float *>(sp_raw);                       // [warp][col][OUT_LD]
  float *sm = so + SP_WARPS * COLS * OUT_LD, *sl = sm + SP_WARPS * COLS;   // [warp][col]
  float *sw = sl + SP_WARPS * COLS;                                      // [col]: what the merge multiplies by
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = nt * 8 + 2 * t + e;
      if (g == 0) {
        sm[warp * COLS + col] = l[nt][e] == 0.f ? -INFINITY : m[nt][e] - ce;
        sl[warp * COLS + col] = l[nt][e];
      }
#pragma unroll
      for (int j = 0; j < NG; j++)
        *reinterpret_cast<float4 *>(&so[(warp * COLS + col) * OUT_LD + 32 * j + 4 * g]) =
            make_float4(o[nt][2 * j][e] + mid[nt][j][e], o[nt][2 * j][2 + e] + mid[nt][j][e], o[nt][2 * j + 1][e] + mid[nt][j][e],
                        o[nt][2 * j + 1][2 + e] + mid[nt][j][e]);
    }
  __syncthreads();
  constexpr size_t PART = (size_t)COLS * (HD + 2);
  float *part = p.ws + ((size_t)unit * p.splits + split) * PART;
  if (threadIdx.x < COLS) {
    const int col = threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < SP_WARPS; w++) M = fmaxf(M, sm[w * COLS + col]);
    for (int w = 0; w < SP_WARPS; w++) {
      const float f = sm[w * COLS + col] == -INFINITY ? 0.f : ex2(sm[w * COLS + col] - M);
      L += f * sl[w * COLS + col];
      sm[w * COLS + col] = f;
    }
    sw[col] = p.splits > 1 ? 1.f : L == 0.f ? 0.f : 1.f / L;
    if (p.splits > 1) {
      part[COLS * HD + col] = M;
      part[COLS * HD + COLS + col] = L;
    }
  }
  __syncthreads();
  auto put = [&](int col, int d, const float (&v)[4]) {
    const int c = c0 + col, tok = c / G;
    T *y = reinterpret_cast<T *>(a.out) + ((size_t)(b * (long long)a.S + tok) * a.n_heads + kvh * G + c - tok * G) * HD + d;
    *reinterpret_cast<uint2 *>(y) = make_uint2(pack2x<T>(v[0], v[1]), pack2x<T>(v[2], v[3]));
  };
  for (int i = threadIdx.x; i < n_cols * (HD / 4); i += SP_WARPS * 32) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float v[4] = {};
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) {
      const float f = sm[w * COLS + col];
      const float4 x = *reinterpret_cast<const float4 *>(&so[(w * COLS + col) * OUT_LD + d]);
      if (f != 0.f) {
        v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= sw[col];
    if (p.splits > 1) *reinterpret_cast<float4 *>(&part[col * HD + d]) = make_float4(v[0], v[1], v[2], v[3]);
    else put(col, d, v);
  }
  if (p.splits == 1) return;
  // ---- the last CTA of a unit joins its parts, in the order of the splits ----------------------------------------------
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *last = atomicAdd(&p.tickets[unit], 1u) == (unsigned)p.splits - 1;
  __syncthreads();
  if (!*last) return;
  __threadfence();
  const float *all = p.ws + (size_t)unit * p.splits * PART;
  for (int i = threadIdx.x; i < n_cols * (HD / 4); i += SP_WARPS * 32) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float M = -INFINITY, L = 0.f, v[4] = {};
    for (int s = 0; s < p.splits; s++) M = fmaxf(M, __ldcg(all + s * PART + COLS * HD + col));
    for (int s = 0; s < p.splits; s++) {
      const float mm = __ldcg(all + s * PART + COLS * HD + col);
      if (mm == -INFINITY) continue;
      const float f = ex2(mm - M);
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(all + s * PART + col * HD + d));
      L = fmaf(f, __ldcg(all + s * PART + COLS * HD + COLS + col), L);
      v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= inv;
    put(col, d, v);
  }
  if (threadIdx.x == 0) p.tickets[unit] = 0;   // for the next launch
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
    return launch(s, launches, write_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, a);
  });
}
int read(cudaStream_t s, int dtype, const Read &a, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    const long long warps = ((long long)a.B * a.n_kv * a.n * (a.hd / 8) + 31) / 32;
    return launch(s, launches, read_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, a);
  });
}
// The form of a call: 16 rows a CTA where there are more than 8 (heads of 256 entries: always 8, whose sums fill the registers), and as many CTAs per
// (batch row, key head, rows) as are resident together, with a block for every warp.
template <typename T, int HD, int NT> static int attend_split(cudaStream_t s, const Attend &a, const Scratch &x, uint64_t *launches) {
  Split p{a};
  p.cols = a.S * (a.n_heads / a.n_kv);
  p.ws = x.ws; p.tickets = x.tickets; p.err = x.err;
  const long long units = (long long)a.B * a.n_kv * ((p.cols + 8 * NT - 1) / (8 * NT)), slots = (long long)x.sms * (HD * NT <= 128 ? 2 : 1);
  const int n_blk = a.d_pos ? a.blocks : (a.pos0 + a.S - 1) / BLOCK - a.first / BLOCK + 1;
  p.splits = (int)std::max(1ll, std::min<long long>(slots / units, (n_blk + SP_WARPS - 1) / SP_WARPS));
  return launch(s, launches, attend_split_kernel<T, HD, NT>, dim3((unsigned)(units * p.splits)), dim3(SP_WARPS * 32), (size_t)sp_smem<HD, NT>(), p);
}
int attend(cudaStream_t s, int dtype, const Attend &a, const Scratch &x, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    constexpr int HD = hd.value;
    if constexpr (HD == 256) return attend_split<T, HD, 1>(s, a, x, launches);
    else if (a.S * (a.n_heads / a.n_kv) <= 8) return attend_split<T, HD, 1>(s, a, x, launches);
    else return attend_split<T, HD, 2>(s, a, x, launches);
  });
}
size_t scratch_floats(int sms) { return (size_t)sms * 2 * 16 * (256 + 2); }
size_t scratch_tickets(int sms) { return (size_t)sms * 2; }
template <typename T, int HD, int NT> static int big_smem() {
  cudaError_t e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, sp_smem<HD, NT>());
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  return (int)e;
}
int prepare(int dtype, int hd) {
  return by_type(dtype, hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    constexpr int HD = hd.value;
    const int e = big_smem<T, HD, 1>();
    if constexpr (HD == 256) return e;
    else return e ? e : big_smem<T, HD, 2>();
  });
}

}  // namespace pc
}  // namespace cake
