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
template <typename T> __device__ __forceinline__ uint32_t most2() { return std::is_same<T, __half>::value ? 0x7bff7bffu : 0x7f7f7f7fu; }   // D's largest number, twice
template <typename T> __device__ __forceinline__ uint32_t bits(T v) { return *reinterpret_cast<const uint16_t *>(&v); }
template <typename T> __device__ __forceinline__ float2 open_pair(uint32_t p) { return DT<T>::unpack2(p); }   // (step, lo)

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


// pairs of D in a word
template <typename T> struct Two;
template <> struct Two<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct Two<__half> { typedef __half2 type; };
template <typename T> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {   // NaN where either is
  typedef typename Two<T>::type U;
  const U r = __hmin2_nan(*reinterpret_cast<const U *>(&a), *reinterpret_cast<const U *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  typedef typename Two<T>::type U;
  const U r = __hmax2_nan(*reinterpret_cast<const U *>(&a), *reinterpret_cast<const U *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <typename T> __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {   // one rounding
  typedef typename Two<T>::type U;
  const U r = __hfma2(*reinterpret_cast<const U *>(&a), *reinterpret_cast<const U *>(&b), *reinterpret_cast<const U *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t m, uint32_t c) {   // (as two constants the compiler takes two operations)
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(m), "r"(c));
  return r;
}

// ------------------------------------------------------------------------------------------ rows into the cache
// Bound by memory: 16 bits read and 5 written an entry.  A warp takes 8 positions of one head, a lane (r, t) of them entries 32 j + 8 t .. + 7 of
// position r for all groups j: that is K's words of the lane as the cache has them, so that codes leave as one piece of 16 bytes a lane (hd 128);
// V's words take a 16-bit half from the neighbouring position's lane.  Minimum and maximum of a group are taken in pairs (D's own comparisons, which
// keep a NaN), minimum and negated maximum together over its four lanes; each lane then has the division of one group in four.  A code is
// fma, add with rounding down (the integer in the lowest bits) and a multiply-add that moves it to its place: n = floor((x - lo) / step + 1/2).
// inv is 1 / step rounded up and the fma rounds down: a tie (common, with eight bits an entry) is never taken for less, and what is below one only where
// it lies closer than 2^-23 of the quotient, fp32's own step.  (Ties by a constant 2^-19 on top: an entry near zero, 2^-20 steps below a tie, went up.)
// 8 x 4096 rows of 8 heads of 128, written and read back: a row per 16 lanes, V in 16-bit stores 102 + 71 us on the device; so 39 + 30 (29 without the arithmetic).
template <typename T, bool ODDS_LAST> __device__ __forceinline__ uint32_t encode8(const uint32_t (&c)[4], float lo, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 x = DT<T>::unpack2(c[i]);
    const uint32_t a = __float_as_uint(__fadd_rd(__fmaf_rd(x.x - lo, inv, 0.5f), 8388608.f));
    const uint32_t b = __float_as_uint(__fadd_rd(__fmaf_rd(x.y - lo, inv, 0.5f), 8388608.f));
    w += a * (1u << (4 * (ODDS_LAST ? i : 2 * i)));
    w += b * (1u << (4 * (ODDS_LAST ? 4 + i : 2 * i + 1)));
  }
  return w - 0xfb000000u;   // the exponents: 0x4b000000 (1 + 16 + 16^2 ..) mod 2^32
}
// BARE: rows as they are, without norm and rotation (41.5 us with their code beside it, unused).
template <typename T, int HD, bool BARE>
__global__ void __launch_bounds__(128) write_kernel(const Write a) {
  pdl_launch_dependents();
  constexpr int NG = HD / 32;
  const int lane = threadIdx.x & 31, t = lane & 3;
  const int heads = a.n_q + 2 * a.n_kv;
  pdl_wait();
  const int pos0 = a.d_pos ? *a.d_pos : a.pos0, eights = ((pos0 & 7) + a.S + 7) >> 3;   // runs of 8 positions that the step touches
  const unsigned item = blockIdx.x * 4 + (threadIdx.x >> 5);   // (the rows that fit a GPU's memory are fewer)
  if (item >= (unsigned)a.B * eights * heads) return;
  const int head = (int)(item % heads), run = (int)(item / heads % eights), b = (int)(item / heads / eights);
  const int pos = (pos0 & ~7) + 8 * run + (lane >> 2), tok = pos - pos0;
  const bool in = tok >= 0 && tok < a.S;
  const bool is_q = head < a.n_q, is_v = head >= a.n_q + a.n_kv;
  const int h = is_q ? head : is_v ? head - a.n_q - a.n_kv : head - a.n_q;
  const T *src = is_q ? reinterpret_cast<const T *>(a.q) + b * a.k_batch + tok * a.k_tok
                 : is_v ? reinterpret_cast<const T *>(a.v) + b * a.v_batch + tok * a.v_tok : reinterpret_cast<const T *>(a.k) + b * a.k_batch + tok * a.k_tok;
  src += (size_t)h * HD + 8 * t;
  uint32_t c[NG][4];
#pragma unroll
  for (int j = 0; j < NG; j++) {
    const uint4 v = in ? *reinterpret_cast<const uint4 *>(src + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
    c[j][0] = v.x; c[j][1] = v.y; c[j][2] = v.z; c[j][3] = v.w;
  }
  if (!BARE && !is_v) {   // (a warp's head is one)
    const T *nw = reinterpret_cast<const T *>(is_q ? a.q_norm : a.k_norm);
    float inv = 0.f;
    if (nw) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NG; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 x = DT<T>::unpack2(c[j][e]);
          ss += x.x * x.x + x.y * x.y;
        }
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
    }
    auto normed = [&](uint32_t (&x)[4], int at) {   // entries at .. at + 7 of the head
      if (!nw) return;
      const uint4 w = *reinterpret_cast<const uint4 *>(nw + at);
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 y = DT<T>::unpack2(x[e]), g = DT<T>::unpack2(ww[e]);
        x[e] = pack2x<T>(y.x * inv * g.x, y.y * inv * g.y);
      }
    };
    const int half = a.rot / 2;   // pairs (i, i + half), a multiple of 8: a lane's 8 entries are all of one half
    // the other ones of the pairs: this lane's, or, where half is no whole number of groups, read again
    const bool same = half == HD / 2;
    uint32_t far[NG][4];
    if (a.cos_t && !same)
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const int at = 32 * j + 8 * t, other = at < half ? at + half : at - half;
        const uint4 v = in && at < a.rot ? *reinterpret_cast<const uint4 *>(src - 8 * t + other) : make_uint4(0u, 0u, 0u, 0u);
        far[j][0] = v.x; far[j][1] = v.y; far[j][2] = v.z; far[j][3] = v.w;
        if (at < a.rot) normed(far[j], other);
      }
#pragma unroll
    for (int j = 0; j < NG; j++) normed(c[j], 32 * j + 8 * t);
    if (a.cos_t) {
      auto turn = [&](uint32_t x, uint32_t y, uint32_t cw, uint32_t sw, bool low) {
        const float2 xf = DT<T>::unpack2(x), yf = DT<T>::unpack2(y), cf = DT<T>::unpack2(cw), sf = DT<T>::unpack2(sw);
        return low ? pack2x<T>(rnd<T>(xf.x * cf.x) - rnd<T>(yf.x * sf.x), rnd<T>(xf.y * cf.y) - rnd<T>(yf.y * sf.y))
                   : pack2x<T>(rnd<T>(xf.x * cf.x) + rnd<T>(yf.x * sf.x), rnd<T>(xf.y * cf.y) + rnd<T>(yf.y * sf.y));
      };
      const T *cr = reinterpret_cast<const T *>(a.cos_t) + (size_t)(in ? pos : pos0) * half, *sr = reinterpret_cast<const T *>(a.sin_t) + (size_t)(in ? pos : pos0) * half;
      if (same) {
#pragma unroll
        for (int j = 0; j < NG / 2; j++) {
          const uint4 cv = *reinterpret_cast<const uint4 *>(cr + 32 * j + 8 * t), sv = *reinterpret_cast<const uint4 *>(sr + 32 * j + 8 * t);
          const uint32_t cw[4] = {cv.x, cv.y, cv.z, cv.w}, sw[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t x = c[j][e], y = c[j + NG / 2][e];
            c[j][e] = turn(x, y, cw[e], sw[e], true);
            c[j + NG / 2][e] = turn(y, x, cw[e], sw[e], false);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < NG; j++) {
          const int at = 32 * j + 8 * t;
          if (at < a.rot) {
            const int o = at < half ? at : at - half;
            const uint4 cv = *reinterpret_cast<const uint4 *>(cr + o), sv = *reinterpret_cast<const uint4 *>(sr + o);
            const uint32_t cw[4] = {cv.x, cv.y, cv.z, cv.w}, sw[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
            for (int e = 0; e < 4; e++) c[j][e] = turn(c[j][e], far[j][e], cw[e], sw[e], at < half);
          }
        }
      }
    }
    if (is_q) {
      __syncwarp();   // (every lane has read what it needs of the row)
      if (in)
#pragma unroll
        for (int j = 0; j < NG; j++) *reinterpret_cast<uint4 *>(const_cast<T *>(src) + 32 * j) = make_uint4(c[j][0], c[j][1], c[j][2], c[j][3]);
    }
  }
  if (is_q) return;
  uint32_t ends[NG];   // a group's minimum and negated maximum
#pragma unroll
  for (int j = 0; j < NG; j++) {
    uint32_t lo = min2<T>(min2<T>(c[j][0], c[j][1]), min2<T>(c[j][2], c[j][3])), hi = max2<T>(max2<T>(c[j][0], c[j][1]), max2<T>(c[j][2], c[j][3]));
    lo = min2<T>(lo, __byte_perm(lo, lo, 0x1032));
    hi = max2<T>(hi, __byte_perm(hi, hi, 0x1032));
    uint32_t e = __byte_perm(lo, hi ^ 0x80008000u, 0x5410);
    e = min2<T>(e, __shfl_xor_sync(0xffffffffu, e, 1));
    ends[j] = min2<T>(e, __shfl_xor_sync(0xffffffffu, e, 2));
  }
  char *blk = reinterpret_cast<char *>(a.cache) + ((size_t)(b * a.n_kv + h) * a.blocks + (pos >> 4)) * block_bytes(HD);
  const int r = pos & 15;
  float invs[(NG + 3) / 4];   // of groups t, t + 4
#pragma unroll
  for (int i = 0; i < (NG + 3) / 4; i++) {
    uint32_t e = ends[4 * i];
#pragma unroll
    for (int j = 1; j < 4 && j < NG; j++) e = t == j ? ends[4 * i + j] : e;
    const float2 x = DT<T>::unpack2(e);
    const float span = -x.y - x.x;   // NaN or infinite: the group has no code
    const bool fine = span <= 3.402823466e38f;
    T st = round_up<T>(fine ? span / 15.f : 0.f);
    if (DT<T>::to_f(st) < 1.17549435e-38f && span > 0.f) st = DT<T>::from_f(1.17549435e-38f);
    const float step = DT<T>::to_f(st);
    invs[i] = fine && step > 0.f ? __frcp_ru(step) : 0.f;
    if (in && 4 * i + t < NG)
      reinterpret_cast<uint32_t *>(blk + (is_v ? v_pairs(HD) : k_pairs(HD)))[pair_word(HD, r, 4 * i + t)] = fine ? bits(st) | e << 16 : 0x7fff7fffu;
  }
  uint32_t w[NG];
#pragma unroll
  for (int j = 0; j < NG; j++) {
    const float inv = __shfl_sync(0xffffffffu, invs[j / 4], (lane & ~3) | (j & 3)), lo = DT<T>::unpack2(ends[j]).x;
    w[j] = is_v ? encode8<T, false>(c[j], lo, inv) : encode8<T, true>(c[j], lo, inv);
  }
  auto store = [](char *p, const uint32_t *x) {
    if (NG == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(x[0], x[1]);
    else *reinterpret_cast<uint4 *>(p) = make_uint4(x[0], x[1], x[2 % NG], x[3 % NG]);
  };
  if (!is_v) {
    if (in)
#pragma unroll
      for (int j = 0; j < NG; j += 4) store(blk + k_word(HD, r, t) * 4 + j * 4, w + j);
    return;
  }
  // V: an even position's lane has word g = 2 t, an odd one's g = 2 t + 1, of both positions
  const bool odd = r & 1, pair_in = __shfl_xor_sync(0xffffffffu, (int)in, 4) && in;
  const int g = 2 * t + (odd ? 1 : 0);
#pragma unroll
  for (int j = 0; j < NG; j++) {
    const uint32_t theirs = __shfl_xor_sync(0xffffffffu, w[j], 4);
    if (!pair_in) {   // the neighbour stays as it is
      if (in) {
        uint16_t *v = reinterpret_cast<uint16_t *>(blk + v_codes(HD));
        v[v_half(HD, r, 2 * t, j)] = (uint16_t)w[j];
        v[v_half(HD, r, 2 * t + 1, j)] = (uint16_t)(w[j] >> 16);
      }
    }
    w[j] = odd ? __byte_perm(theirs, w[j], 0x7632) : __byte_perm(w[j], theirs, 0x5410);
  }
  if (pair_in)
#pragma unroll
    for (int j = 0; j < NG; j += 4) store(blk + v_codes(HD) + v_half(HD, r & ~1, g, j) * 2, w + j);
}

// ------------------------------------------------------------------------------------------ rows out of the cache
// Bound by memory too: 5 bits read and 16 written an entry.  A warp takes a block: K's words as they lie (a row's four lanes write 64 bytes of it
// together), V's likewise (8 lanes write 64 bytes of a row).  A value is one fma in pairs of D on exact codes: one rounding; as step is rounded up, the
// highest codes of a group that reaches D's end may lie beyond it: they become D's largest number (an infinity would be one that nobody wrote, and NaN for
// every row whose weight for it is zero).
// 32768 positions of 8 heads of 128, K and V: 71 us with 2-byte reads of V and 64-bit divisions a lane; so 30 (5.8 TB/s).
// As operands of matrix products (a.nan): a group that reads as NaN becomes zero, so that it counts for no row that does not see it, and the
// block's word says where: byte 0 the first position (in the block) whose K has such a group, byte 1 + j that of V's group j, 255 none.
template <typename T> struct Codes;   // n as pairs of D, nibbles i and 4 + i of w
template <> struct Codes<__half> {
  static __device__ __forceinline__ void open(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t v = w >> 8;
    r[0] = fma2<__half>(and_or(w, 0x000f000fu, 0x64006400u), 0x3c003c00u, 0xe400e400u);   // (1024 + n) - 1024
    r[1] = fma2<__half>(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd400d400u);   // (1024 + 16 n) / 16 - 64
    r[2] = fma2<__half>(and_or(v, 0x000f000fu, 0x64006400u), 0x3c003c00u, 0xe400e400u);
    r[3] = fma2<__half>(and_or(v, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd400d400u);
  }
};
template <> struct Codes<__nv_bfloat16> {
  static __device__ __forceinline__ void open(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = fma2<__nv_bfloat16>(and_or(w >> (4 * i), 0x000f000fu, 0x43004300u), 0x3f803f80u, 0xc300c300u);   // (128 + n) - 128
  }
};
template <typename T, int HD>
__global__ void __launch_bounds__(128) read_kernel(const Read a) {
  pdl_launch_dependents();
  constexpr int NG = HD / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int blk0 = a.first >> 4, n_blk = ((a.first + a.n - 1) >> 4) - blk0 + 1;
  const unsigned item = blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  if (item >= (unsigned)a.B * a.n_kv * n_blk) return;
  const int i = (int)(item % n_blk), slab = (int)(item / n_blk);
  const char *blk = reinterpret_cast<const char *>(a.cache) + ((size_t)slab * a.blocks + blk0 + i) * block_bytes(HD);
  const int row0 = 16 * (blk0 + i) - a.first;   // the output row of the block's first position
  bool any_nan = false;
  auto value = [](uint32_t n, const uint32_t (&q)[2]) { return min2<T>(fma2<T>(n, q[0], q[1]), most2<T>()); };   // (keeps a NaN)
  auto pair_of = [&](uint32_t p, uint32_t (&q)[2]) {   // step and lo, twice each
    if (a.nan && (p & 0x7fffu) > (sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u)) {
      any_nan = true;
      p = 0;
    }
    q[0] = __byte_perm(p, p, 0x1010);
    q[1] = __byte_perm(p, p, 0x3232);
  };
  if (a.k) {
    T *out = reinterpret_cast<T *>(a.k) + ((size_t)slab * a.out_rows + row0) * HD;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int r = g + 8 * half, row = row0 + r;
      uint32_t w[NG], p[NG];
      lds_words<NG>(blk + (half * 32 + lane) * NG * 4, w);
      lds_words<NG>(blk + k_pairs(HD) + r * NG * 4, p);
      const bool in = row >= 0 && row < a.n;
#pragma unroll
      for (int j = 0; j < NG; j++) {
        uint32_t c[4], q[2];
        Codes<T>::open(w[j], c);
        if (in) pair_of(p[(j & 1) * (NG / 2) + j / 2], q);
        else q[0] = q[1] = 0u;
        if (in)
          *reinterpret_cast<uint4 *>(out + (size_t)r * HD + 32 * j + 8 * t) =
              make_uint4(value(c[0], q), value(c[1], q), value(c[2], q), value(c[3], q));
      }
    }
  }
  if (a.v) {
    T *out = reinterpret_cast<T *>(a.v) + ((size_t)slab * a.out_rows + row0) * HD;
#pragma unroll
    for (int half = 0; half < 2; half++) {   // positions 8 half + 2 t and its neighbour
      const int r = 8 * half + 2 * t;
      uint32_t p0[NG], p1[NG];
      lds_words<NG>(blk + v_pairs(HD) + r * NG * 4, p0);
      lds_words<NG>(blk + v_pairs(HD) + (r + 1) * NG * 4, p1);
      const bool in0 = row0 + r >= 0 && row0 + r < a.n, in1 = row0 + r + 1 >= 0 && row0 + r + 1 < a.n;
#pragma unroll
      for (int j = 0; j < NG; j++) {
        // entries 4 g .. + 3 of the group: nibbles 0 .. 3 of either half; as pairs of neighbouring entries
        const uint32_t w = *reinterpret_cast<const uint32_t *>(blk + v_codes(HD) + v_half(HD, r, g, j) * 2);
        uint32_t c[4], q[2];
        Codes<T>::open(w, c);   // c[e]: entry e of both positions
        const uint32_t a0 = __byte_perm(c[0], c[1], 0x5410), a1 = __byte_perm(c[2], c[3], 0x5410), b0 = __byte_perm(c[0], c[1], 0x7632),
                       b1 = __byte_perm(c[2], c[3], 0x7632);
        if (in0) {
          pair_of(p0[(j & 1) * (NG / 2) + j / 2], q);
          *reinterpret_cast<uint2 *>(out + (size_t)r * HD + 32 * j + 4 * g) = make_uint2(value(a0, q), value(a1, q));
        }
        if (in1) {
          pair_of(p1[(j & 1) * (NG / 2) + j / 2], q);
          *reinterpret_cast<uint2 *>(out + (size_t)(r + 1) * HD + 32 * j + 4 * g) = make_uint2(value(b0, q), value(b1, q));
        }
      }
    }
  }
  if (HD <= 128 && a.nan) {   // (heads of 256 entries have more groups than a word has bytes, and no such products)
    unsigned long long word = ~0ull;
    if (__any_sync(0xffffffffu, any_nan)) {
      const int r = lane & 15;   // lanes 0 .. 15: positions
      const bool in = lane < 16 && row0 + r >= 0 && row0 + r < a.n;
      for (int j = -1; j < NG; j++) {
        bool bad = false;
        for (int k = max(j, 0); k <= (j < 0 ? NG - 1 : j); k++) {
          const float step = open_pair<T>(reinterpret_cast<const uint32_t *>(blk + (j < 0 ? k_pairs(HD) : v_pairs(HD)))[pair_word(HD, r, k)]).x;
          bad = bad || step != step;
        }
        const unsigned who = __ballot_sync(0xffffffffu, in && bad);
        if (who) word = (word & ~(0xffull << (8 * (j + 1)))) | (unsigned long long)(__ffs(who) - 1) << (8 * (j + 1));
      }
    }
    if (lane == 0) a.nan[(size_t)slab * n_blk + i] = word;
  }
}

// ------------------------------------------------------------------------------------------ attention of a few rows, keys split
// A CTA serves up to 8 NT / PK query rows (row = token G + head of one key head) and a range of blocks; its warps take the blocks in turn, each through
// a ring of its own (cp.async, 16 bytes a lane; a bulk copy and an mbarrier a block took a fifth of the loop), so that no warp waits for another
// until the end.  Per block, with m16n8k16 products in fp16:
//   S^T = K Q^T   A: 16 keys' codes less 8, B: the rows' queries, kept in registers.  A group's sum is taken apart from the others', then
//                 s += step sum + (lo + 8 step) (sum of the group's q): the codes go in exactly, and no entry is formed.  Queries are scaled by a power of
//                 two that puts a row's largest below 2^15: an entry down to 2^-29 of it keeps its bits, or 2^-25 where it meets an odd nibble.
//   O^T += V^T P  A: 16 entries' codes less 8, B: weights times steps in fp16, an operand per group; what is left of the value, lo + 8 step, is a number
//                 per key and group and is summed in fp32.  P^T turns into an operand by movmatrix.  One operand has 11 bits, three more than a result in
//                 bf16; in f16 a second one takes what rounding the first one left (with one, 31 positions: 0.000223 of the norm from 64 bits, rounding
//                 the result alone is 0.000200; 32 sequences at 4000 positions 39.7 -> 44.4 us).
// Four bits become fp16 by one logic operation a pair (Kim, Henry, Fahim and Hassan 2022): n under the exponent of 1024 is 1024 + n in the lowest four bits, 1024 + 16 n
// in the next.  The 16 stays in: K's queries are divided by it, V's sums at the end.  1024 + 8 (1024 + 128) is subtracted, exactly: left in K's sums,
// which then start from -1024 sum of q, it took their last ten bits; V's weights would count for all of 1024 + n, and so for 8 steps at most.  (K's
// codes cost 32 of 376 instructions a block and warp: one token at 131072 39.8 -> 40.7 us; the registers of the sums that they started from are
// free again, 32 sequences of 2 rows at 4000 51.0 -> 47.4.)
// PK = 2, up to 4 rows: columns 0 .. 3 of an operand belong to a group and columns 4 .. 7 to its neighbour (the queries of the other are zero there),
// so that no lane works for columns without a row; a row's two halves join by a shuffle.
// A row's reference m moves when a score exceeds it by 2^6 (TAU).  Every group has a power of two `up` that keeps its steps at 512 at most, the first ones at
// 8 to 16: weights times steps then use fp16's range whatever the size of V's entries and of other groups' (one power for all groups took a
// group 2^24 times smaller than its neighbour for one value).  It is the same for all rows; a block with positions that only later rows of the call see, and
// much larger steps there, is taken in the order of those positions, so that a row's own weights meet the power of what it sees.  (A power per row
// and group: 32 sequences of 2 rows at 4000 positions 62.6 us, 46.7 with one power in all.)
//
// Who takes which blocks: a unit is 8 NT / PK rows of a (batch row, key head).  Short caches: the CTAs of a cluster cut a unit's blocks between them and
// join over the cluster's shared memory.  Else all units' blocks lie in one line that the grid, two CTAs per SM, cuts into equal parts; a CTA's part of
// a unit that others have parts of goes to ws, and the last one to come joins them, in the order of the line.  (A cluster's CTAs send their sums to
// the one that joins them: one barrier behind, where reading them there takes a second one before anybody leaves.)
constexpr int SP_STAGES = 4, SP_WARPS = 8, SP_CLUSTER_LOG2 = 3;
constexpr int sp_per_sm(int hd, int nt) { return hd * nt <= 128 ? 2 : 1; }   // CTAs that 128 or 255 registers a thread leave room for
struct Split {
  Attend a;
  int cols, col_blocks, units;   // rows of a (batch row, key head), pieces that they are cut into; units in all
  int cluster_log2;              // CTAs of a cluster, a unit for each of the grid's (y, z); -1: the line
  float *ws;                     // [2 CTA + (part that begins behind the CTA's first block)] of {O [col][hd], m [col], l [col]}
  unsigned *tickets;             // [first CTA of a cut unit], zero between launches
};
// what a CTA of a cluster is sent: for its share of the results, from every CTA, four sums and their m and l
template <int HD, int NT> __host__ __device__ constexpr int sp_recv() { return 8 * NT * (HD / 4) * 32; }
template <int HD, int NT> __host__ __device__ constexpr int sp_smem() {
  const int w = SP_WARPS, ring = w * SP_STAGES * block_bytes(HD), out = w * 8 * NT * (HD * 4 + 16) + w * 8 * NT * 8;
  return (ring > out ? ring : out) + sp_recv<HD, NT>() + 16;
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
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t c) {   // pairs of fp16; exact here
  const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
// nibbles i and 4 + i of w as a pair of fp16: n - 8 for even i, 16 (n - 8) for odd i
__device__ __forceinline__ void open_centred(uint32_t w, uint32_t (&r)[4]) {
  const uint32_t v = w >> 8;
  r[0] = add2(and_or(w, 0x000f000fu, 0x64006400u), 0xe408e408u);   // 1024 + n less 1024 + 8
  r[1] = add2(and_or(w, 0x00f000f0u, 0x64006400u), 0xe480e480u);   // 1024 + 16 n less 1024 + 16 * 8
  r[2] = add2(and_or(v, 0x000f000fu, 0x64006400u), 0xe408e408u);
  r[3] = add2(and_or(v, 0x00f000f0u, 0x64006400u), 0xe480e480u);
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

template <typename T, int HD, int NT, int PK>
__global__ void __launch_bounds__(SP_WARPS * 32, sp_per_sm(HD, NT)) attend_split_kernel(const Split p) {
  // a lane's groups: all (PK 1), or those of its half of the columns (PK 2); its heads: columns 2 t and 2 t + 1, of the half
  constexpr int WARPS = SP_WARPS, NG = HD / 32, MG = NG / PK, COLS = 8 * NT / PK, OUT_LD = HD + 4;
  constexpr bool TWO = std::is_same<T, __half>::value;   // operands of a weight times a step
  const Attend &a = p.a;
  extern __shared__ __align__(128) unsigned char sp_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int half = PK == 2 ? t >> 1 : 0, tc = PK == 2 ? t & 1 : t;
  unsigned char *ring = sp_raw + warp * SP_STAGES * block_bytes(HD);
  int *last = reinterpret_cast<int *>(sp_raw + sp_smem<HD, NT>() - 16);
  float *recv = reinterpret_cast<float *>(last) - sp_recv<HD, NT>() / 4;   // [item of mine][CTA of the cluster][8]
  const bool in_line = p.cluster_log2 < 0;
  if (p.cluster_log2 > 0) cluster_arrive_relaxed();   // (waited for where the first sums go to another CTA: it has begun by then)
  pdl_launch_dependents();
  pdl_wait();
  const int G = a.n_heads / a.n_kv;
  const int pos0 = a.d_pos ? *a.d_pos : a.pos0;
  const int first = a.d_pos ? (a.window > 0 ? max(0, pos0 + 1 - a.window) : 0) : a.first;
  const int blk0 = first >> 4, n_blk = max(0, ((pos0 + a.S - 1) >> 4) - blk0 + 1);   // of a unit (its own rows may see fewer)
  const long long line = in_line ? (long long)p.units * n_blk : 0;
  const long long ctas = min((long long)gridDim.x, (line + WARPS - 1) / WARPS);   // that the line is cut between: none of them without a block
  if (in_line && blockIdx.x >= ctas) return;
  // first block of a CTA, CTA of a block (whole CTAs for a unit where their number divides: a part of its own costs a CTA some 3 us)
  auto start_of = [&](int cta) {
    return line * ctas >> 32 ? line * cta / ctas : (long long)((unsigned)line * (unsigned)cta / (unsigned)ctas);
  };
  auto cta_of = [&](long long x) {
    return line * ctas >> 32 ? (int)(((x + 1) * ctas - 1) / line) : (int)(((unsigned)(x + 1) * (unsigned)ctas - 1u) / (unsigned)line);
  };
  const int rank = in_line ? 0 : (int)blockIdx.x, lg = max(0, p.cluster_log2);
  // this CTA's blocks of the line, or of its unit
  long long at = in_line ? start_of(blockIdx.x) : n_blk * rank >> lg;
  const long long end = in_line ? start_of(blockIdx.x + 1) : n_blk * (rank + 1) >> lg;
  // ---- one unit's blocks
#pragma unroll 1
  for (bool again = true; again;) {
  const int unit = in_line ? (int)(at / n_blk) : 0;
  const int heads_at = in_line ? unit : (int)blockIdx.y, piece = p.col_blocks == 1 ? 0 : heads_at % p.col_blocks;
  const int kvh_b = p.col_blocks == 1 ? heads_at : heads_at / p.col_blocks;
  const int c0 = piece * COLS, kvh = in_line ? kvh_b % a.n_kv : kvh_b, b = in_line ? kvh_b / a.n_kv : (int)blockIdx.z;
  const long long unit0 = (long long)unit * n_blk, stop = min(end, unit0 + n_blk);
  auto tok_of = [&](int c) { return a.S == 1 ? 0 : c / G; };
  const int n_cols = min(COLS, p.cols - c0), pos_lo = pos0 + tok_of(c0), pos_hi = pos0 + tok_of(c0 + n_cols - 1);   // the rows' first and last position
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
  float qs[NT][MG][2], sc[NT][2];   // a group's sums of q; scale log2(e) and the power of two back
  int cpos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int c = c0 + (PK == 2 ? g & 3 : nt * 8 + g), tok = tok_of(c);
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
    const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - e) << 23);
    sc[nt][0] = __shfl_sync(0xffffffffu, down, 8 * tc);
    sc[nt][1] = __shfl_sync(0xffffffffu, down, 8 * tc + 4);
#pragma unroll
    for (int j = 0; j < NG; j++) {
      float f[8], sum = 0.f;
      unpack8<T>(raw[j], f);
#pragma unroll
      for (int i = 0; i < 8; i++) sum += f[i] *= up;
      const bool here = PK == 1 || (j & 1) == g >> 2;
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const uint32_t x = pack2x<__half>(f[2 * h] * (h & 1 ? 0.0625f : 1.f), f[2 * h + 1] * (h & 1 ? 0.0625f : 1.f));
        qf[nt][j][h] = here ? x : 0u;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int e2 = 0; e2 < 2; e2++) {
        const float s2 = __shfl_sync(0xffffffffu, sum, 8 * tc + 4 * e2);
        if (PK == 1 || (j & 1) == half) qs[nt][j / PK][e2] = s2;
      }
    }
#pragma unroll
    for (int e2 = 0; e2 < 2; e2++) cpos[nt][e2] = pos0 + tok_of(min(c0 + nt * 8 + 2 * tc + e2, p.cols - 1));
  }
  float o[NT][2 * NG][4] = {}, mid[NT][MG][2] = {}, m[NT][2], l[NT][2] = {};
  float up[MG];   // of the group of the lane's i-th word of pairs
  constexpr float TAU = 6.f;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -3.402823466e38f;
#pragma unroll
  for (int i = 0; i < MG; i++) up[i] = 8.50705917e37f;   // 2^126
  auto group_of = [](int i) { return PK == 1 ? 2 * (i % (NG / 2)) + i / (NG / 2) : i; };   // the lane's group that its i-th word of pairs belongs to

  // the finite one of a pair's step, as the 16 bits of D that it is (no step is negative: as integers they have their order)
  auto step_bits = [](uint32_t pair) { return (pair & 0xffffu) < bits(DT<T>::from_f(INFINITY)) ? pair & 0xffffu : 0u; };
  // EDGE: of the block's positions from .. to, those that a row sees
  auto body = [&](auto edge_, const unsigned char *blk, int key0, int from, int to) {
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
          open_centred(kw[0][2 * w + h], x[h]);
          open_centred(kw[1][2 * w + h], y[h]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint32_t(&q0)[4] = qf[nt][2 * w], (&q1)[4] = qf[nt][2 * w + 1];
          auto join = [&](int i, float(&d)[4]) {   // d: sums of the group that is the lane's i-th word of pairs
            const float2 p0 = open_pair<T>(kp[0][i]), p1 = open_pair<T>(kp[1][i]);
            const int jj = group_of(i);
            const float m0 = fmaf(8.f, p0.x, p0.y), m1 = fmaf(8.f, p1.x, p1.y);
            s[nt][0] = fmaf(p0.x, d[0], fmaf(m0, qs[nt][jj][0], s[nt][0]));
            s[nt][1] = fmaf(p0.x, d[1], fmaf(m0, qs[nt][jj][1], s[nt][1]));
            s[nt][2] = fmaf(p1.x, d[2], fmaf(m1, qs[nt][jj][0], s[nt][2]));
            s[nt][3] = fmaf(p1.x, d[3], fmaf(m1, qs[nt][jj][1], s[nt][3]));
          };
          if constexpr (PK == 2) {   // 8 entries of either group a product
            float d[4] = {};
#pragma unroll
            for (int h = 0; h < 4; h++) mma16(d, x[0][h], y[0][h], x[1][h], y[1][h], q0[h], q1[h]);
            join(w, d);
          } else {
            float d[4] = {};
            mma16(d, x[0][0], y[0][0], x[0][1], y[0][1], q0[0], q0[1]);
            mma16(d, x[0][2], y[0][2], x[0][3], y[0][3], q0[2], q0[3]);
            join(w, d);
            float f[4] = {};
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
#pragma unroll
    for (int r = 0; r < 2; r++) {
      lds_words<MG>(blk + v_pairs(HD) + ((g + 8 * r) * NG + half * MG) * 4, vp[r]);
      const bool seen = !EDGE || (key0 + g + 8 * r >= from && key0 + g + 8 * r <= to);   // by any row: the others' steps say nothing
#pragma unroll
      for (int i = 0; i < MG; i++) vp[r][i] = seen ? vp[r][i] : 0u;
    }
    bool more = false;   // steps beyond what `up` is for
#pragma unroll
    for (int i = 0; i < MG; i++) more = more || fmaxf(open_pair<T>(vp[0][i]).x, open_pair<T>(vp[1][i]).x) * up[i] > 512.f;
    // scores less their reference, in powers of two
    float far = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (EDGE) {
          const int key = key0 + g + 8 * (i >> 1);
          if (key < from || key > to || key > cpos[nt][i & 1]) s[nt][i] = -INFINITY;
        }
        far = fmaxf(far, fmaf(s[nt][i], sc[nt][i & 1], -m[nt][i & 1]));
      }
    if (__any_sync(0xffffffffu, far > TAU || more)) {
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = fmaxf(s[nt][e], s[nt][2 + e]) * sc[nt][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float mn = fmaxf(m[nt][e], mx);
          f[nt][e] = ex2(m[nt][e] - mn);
          m[nt][e] = mn;
          l[nt][e] *= f[nt][e];
        }
#pragma unroll
      for (int i = 0; i < MG; i++) {
        const int j = group_of(i);
        uint32_t top = max(step_bits(vp[0][i]), step_bits(vp[1][i]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float most = open_pair<T>(top).x;
        const uint32_t was = __float_as_uint(up[i]), now = most * up[i] > 512.f ? (257u - (__float_as_uint(most) >> 23)) << 23 : was;   // 8 <= most up < 16
        const float change = now + 0x3f800000u > was ? __uint_as_float(now + 0x3f800000u - was) : 0.f;   // now / was, a power of two
        up[i] = __uint_as_float(now);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            mid[nt][j][e] *= f[nt][e];
            const float fc = f[nt][e] * change;
#pragma unroll
            for (int k = 2 * PK * j; k < 2 * PK * (j + 1); k++) {   // the group's sums (PK 2: and the neighbour's, which the lane's columns don't have)
              o[nt][k][e] *= fc;
              o[nt][k][2 + e] *= fc;
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
        s[nt][i] = EDGE && s[nt][i] == -INFINITY ? 0.f : ex2(fmaf(s[nt][i], sc[nt][i & 1], -m[nt][i & 1]));   // (sc may have become 0)
        l[nt][i & 1] += s[nt][i];
      }
    // weight i of a row times a number of its key: a key that the row does not see may be anything (one that it does may be NaN, whatever the weight)
    auto times = [&](int nt, int i, float x) { return EDGE && key0 + g + 8 * (i >> 1) > min(cpos[nt][i & 1], to) ? 0.f : s[nt][i] * x; };
#pragma unroll
    for (int w = 0; w < NG / 2; w++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        uint32_t b0[2], b1[2], r0[2], r1[2];   // weights times steps, and what rounding them left
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (PK == 2 && h) {
            b0[1] = b0[0];
            b1[1] = b1[0];
            r0[1] = r0[0];
            r1[1] = r1[0];
            continue;
          }
          const int i = PK == 2 ? w : h * (NG / 2) + w, jj = group_of(i);   // the pair's word; its sums' place
          const float2 p0 = open_pair<T>(vp[0][i]), p1 = open_pair<T>(vp[1][i]);
          const float m0 = fmaf(8.f, p0.x, p0.y), m1 = fmaf(8.f, p1.x, p1.y), x0 = p0.x * up[i], x1 = p1.x * up[i];
          auto operand = [&](float v0, float v1, uint32_t &b, uint32_t &r) {
            b = pack2x<__half>(v0, v1);
            if (TWO) {
              const float2 y = DT<__half>::unpack2(b);
              r = turn8x8(pack2x<__half>(v0 - y.x, v1 - y.y));
            }
            b = turn8x8(b);
          };
          operand(times(nt, 0, x0), times(nt, 1, x0), b0[h], r0[h]);
          operand(times(nt, 2, x1), times(nt, 3, x1), b1[h], r1[h]);
          mid[nt][jj][0] += times(nt, 0, m0);
          mid[nt][jj][0] += times(nt, 2, m1);
          mid[nt][jj][1] += times(nt, 1, m0);
          mid[nt][jj][1] += times(nt, 3, m1);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t x[4], y[4];
          open_centred(vw[2 * w + h], x);
          open_centred(vw[NG + 2 * w + h], y);
          float(&u)[4] = o[nt][2 * (2 * w + h)], (&v)[4] = o[nt][2 * (2 * w + h) + 1];
          mma16(u, x[0], x[1], y[0], y[1], b0[h], b1[h]);
          mma16(v, x[2], x[3], y[2], y[3], b0[h], b1[h]);
          if (TWO) {
            mma16(u, x[0], x[1], y[0], y[1], r0[h], r1[h]);
            mma16(v, x[2], x[3], y[2], y[3], r0[h], r1[h]);
          }
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
    else if (key0 < first || key0 + 15 > pos_lo) {
      // positions that not all rows see and whose steps are far beyond what `up` is for and the others have: one after the other
      const int all = max(pos_lo, max(key0, first));   // those up to here come first
      bool far = false;
      if (all < pos_hi) {
#pragma unroll
        for (int i = 0; i < MG; i++) {
          uint32_t top = 0;   // the largest step of the first ones in the low half, of the others in the high one
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const uint32_t st = step_bits(reinterpret_cast<const uint32_t *>(blk + v_pairs(HD) + ((g + 8 * r) * NG + half * MG) * 4)[i]);
            const int key = key0 + g + 8 * r;
            top = __vmaxu2(top, key < first || key > pos_hi ? 0u : key <= all ? st : st << 16);
          }
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float2 most = open_pair<T>(top);
          far = far || (most.y > 64.f * most.x && most.y * up[i] > 512.f);
        }
        far = __any_sync(0xffffffffu, far);
      }
      const int end = min(pos_hi, key0 + 15);
      for (int from = first, to = far ? min(all, end) : end;; from = ++to) {
        body(std::true_type{}, blk, key0, from, to);
        if (to == end) break;
      }
    }
    else body(std::false_type{}, blk, key0, 0, 0);
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
        sm[warp * COLS + col] = l[nt][e] == 0.f ? -INFINITY : m[nt][e];
        sl[warp * COLS + col] = l[nt][e];
      }
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const float z = mid[nt][j / PK][e], down = __uint_as_float((254u << 23) - __float_as_uint(up[PK == 2 ? j / 2 : (j & 1) * (NG / 2) + j / 2]));   // 1 / up
        if (PK == 1 || (j & 1) == half)
          *reinterpret_cast<float4 *>(&so[(warp * COLS + col) * OUT_LD + 32 * j + 4 * g]) =
              make_float4(fmaf(down, o[nt][2 * j][e], z), fmaf(0.0625f * down, o[nt][2 * j][2 + e], z), fmaf(down, o[nt][2 * j + 1][e], z),
                          fmaf(0.0625f * down, o[nt][2 * j + 1][2 + e], z));
      }
    }
  __syncthreads();
  const bool whole = in_line ? n_here == n_blk : lg == 0;   // nobody else has a part
  auto put = [&](int col, int d, const float (&v)[4], float L) {
    const int c = c0 + col, tok = tok_of(c);
    const float f = L == 0.f ? 0.f : 1.f / L;   // 0: the row sees nothing
    auto held = [](float x) {   // the highest codes' values may lie beyond D's end, see read_kernel
      const float most = DT<T>::unpack2(most2<T>()).x;
      return x > most ? most : x < -most ? -most : x;
    };
    T *y = reinterpret_cast<T *>(a.out) + ((size_t)(b * (long long)a.S + tok) * a.n_heads + kvh * G + c - tok * G) * HD + d;
    *reinterpret_cast<uint2 *>(y) = make_uint2(pack2x<T>(held(v[0] * f), held(v[1] * f)), pack2x<T>(held(v[2] * f), held(v[3] * f)));
  };
  // parts of this unit, where there are several: CTAs first_cta .., in the line
  const bool parted = in_line && !whole;
  const int first_cta = parted ? cta_of(unit0) : 0, parts = parted ? cta_of(unit0 + n_blk - 1) - first_cta + 1 : 1;
  const bool behind = parted && start_of(first_cta) < unit0;   // the first CTA has blocks of another unit in front
  auto slot_of = [&](int cta) { return p.ws + (size_t)(2 * cta + (cta == first_cta && behind ? 1 : 0)) * PART; };
  const int items = n_cols * (HD / 4);
  if (lg) cluster_wait();   // every CTA of the cluster has begun
  for (int i = threadIdx.x; i < items; i += WARPS * 32) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float mw[WARPS], M = -INFINITY, L = 0.f, v[4] = {};
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      mw[w] = sm[w * COLS + col];
      M = fmaxf(M, mw[w]);
    }
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = mw[w] == -INFINITY ? 0.f : ex2(mw[w] - M);
      const float4 x = *reinterpret_cast<const float4 *>(&so[(w * COLS + col) * OUT_LD + d]);
      L = fmaf(f, sl[w * COLS + col], L);
      v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);   // (NaN also where f is too small for a number)
    }
    if (whole) put(col, d, v, L);
    else if (parted) {
      float *part = slot_of(blockIdx.x);
      *reinterpret_cast<float4 *>(&part[col * HD + d]) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) {
        part[COLS * HD + col] = M;
        part[COLS * HD + COLS + col] = L;
      }
    } else {   // result i is CTA i mod 2^lg's
      const uint32_t to = cluster_map(smem_u32(recv + ((size_t)(i >> lg << lg) + rank) * 8), (uint32_t)(i & ((1 << lg) - 1)));
      st_cluster4(to, v[0], v[1], v[2], v[3]);
      st_cluster4(to + 16, M, L, 0.f, 0.f);
    }
  }
  if (lg) {
    // ---- the cluster's CTAs join an equal share of the results each, from what they were sent: nobody reads another's memory ----
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    for (int i = ((int)threadIdx.x << lg) + rank; i < items; i += WARPS * 32 << lg) {
      const float *x = recv + (size_t)(i - rank) * 8;
      float M = -INFINITY, L = 0.f, v[4] = {};
      for (int s = 0; s < 1 << lg; s++) M = fmaxf(M, x[8 * s + 4]);
      for (int s = 0; s < 1 << lg; s++) {
        const float f = x[8 * s + 4] == -INFINITY ? 0.f : ex2(x[8 * s + 4] - M);
        L = fmaf(f, x[8 * s + 5], L);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = fmaf(f, x[8 * s + e], v[e]);
      }
      put(i / (HD / 4), i % (HD / 4) * 4, v, L);
    }
  } else if (parted) {
    // ---- the last CTA of a unit joins its parts, in their order -----------------------------------------------------------
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *last = atomicAdd(&p.tickets[first_cta], 1u) == (unsigned)parts - 1;
    __syncthreads();
    if (*last) {
      __threadfence();
      // Into shared memory, as many as it holds at a time, then weights by a warp a column and sums by a thread a result: short code, as it comes from memory
      // once per launch (131072 positions: straight from memory, unrolled, 42.6 us of which it is 5.3; so 40.7).
      constexpr int ROOM = (sp_smem<HD, NT>() - 16 - COLS * 8) / (PART * 4);
      static_assert(ROOM >= 2, "");
      float *held = reinterpret_cast<float *>(sp_raw), *ml = reinterpret_cast<float *>(last) - 2 * COLS;   // [part][results, m, l]
      for (int s0 = 0; s0 < parts;) {   // after the first time, held[0] is what came before
        const int from = s0 > 0, n = min(ROOM, from + parts - s0);
#pragma unroll 1
        for (int x = threadIdx.x; x < (n - from) * (PART / 4); x += WARPS * 32) {
          const int e = x / (PART / 4), r = x - e * (PART / 4);
          const float *src = slot_of(first_cta + s0 + e) + r * 4;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + (from + e) * PART + r * 4)), "l"(src) : "memory");
        }
        copies_commit();
        copies_wait<0>();
        if (from && (int)threadIdx.x < 2 * COLS) held[COLS * HD + threadIdx.x] = ml[threadIdx.x];
        __syncthreads();
#pragma unroll 1
        for (int col = warp; col < n_cols; col += WARPS) {
          float *x = held + COLS * HD + col, M = -INFINITY, L = 0.f;
#pragma unroll 1
          for (int e = lane; e < n; e += 32) M = fmaxf(M, x[e * PART]);
#pragma unroll
          for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll 1
          for (int e = lane; e < n; e += 32) {
            const float f = x[e * PART] == -INFINITY ? 0.f : ex2(x[e * PART] - M);
            L = fmaf(f, x[e * PART + COLS], L);
            x[e * PART] = f;
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
          if (lane == 0) {
            ml[col] = M;
            ml[COLS + col] = L;
          }
        }
        __syncthreads();
        s0 += n - from;
#pragma unroll 1
        for (int i = threadIdx.x; i < n_cols * (HD / 4); i += WARPS * 32) {
          const int col = i / (HD / 4), d = i % (HD / 4) * 4;
          float *x = held + col * HD + d, v[4] = {};
          const float *f = held + COLS * HD + col;
#pragma unroll 4
          for (int e = 0; e < n; e++) {
            const float w = f[e * PART];
            const float4 y = *reinterpret_cast<const float4 *>(x + e * PART);
            v[0] = fmaf(w, y.x, v[0]); v[1] = fmaf(w, y.y, v[1]); v[2] = fmaf(w, y.z, v[2]); v[3] = fmaf(w, y.w, v[3]);
          }
          if (s0 == parts) put(col, d, v, ml[COLS + col]);
          else *reinterpret_cast<float4 *>(x) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (s0 < parts) __syncthreads();
      }
      if (threadIdx.x == 0) p.tickets[first_cta] = 0;   // for the next launch
    }
  }
  at = stop;
  again = in_line && at < end;
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
    const int eights = a.d_pos ? (a.S + 14) / 8 : ((a.pos0 & 7) + a.S + 7) / 8;   // (at any position on the device)
    const long long warps = (long long)a.B * eights * (a.n_q + 2 * a.n_kv);
    const dim3 grid((unsigned)((warps + 3) / 4)), block(128);
    if (!a.n_q && !a.cos_t && !a.k_norm) return launch(s, launches, write_kernel<T, hd.value, true>, grid, block, 0, 1, a);
    return launch(s, launches, write_kernel<T, hd.value, false>, grid, block, 0, 1, a);
  });
}
int read(cudaStream_t s, int dtype, const Read &a, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    const long long warps = (long long)a.B * a.n_kv * read_blocks(a.first, a.n);
    return launch(s, launches, read_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, 1, a);
  });
}
// The form of a call: 4, 8 or 16 rows a CTA (heads of 256 entries: 4 or 8, whose sums fill the registers), and as many CTAs per (batch row, key head,
// rows) as are resident together, with a block for every warp.
template <typename T, int HD, int NT, int PK> static int attend_split(cudaStream_t s, const Attend &a, const Scratch &x, uint64_t *launches) {
  constexpr int COLS = 8 * NT / PK;
  Split p{a};
  p.cols = a.S * (a.n_heads / a.n_kv);
  p.col_blocks = (p.cols + COLS - 1) / COLS;
  p.ws = x.ws; p.tickets = x.tickets;
  const long long units = (long long)a.B * a.n_kv * p.col_blocks, slots = (long long)x.sms * sp_per_sm(HD, NT);
  const int n_blk = a.d_pos ? a.blocks : std::max(1, (a.pos0 + a.S - 1) / BLOCK - a.first / BLOCK + 1);
  p.units = (int)units;
  int lg = 0;
  while (lg < SP_CLUSTER_LOG2 && SP_WARPS << lg < n_blk && units << (lg + 1) <= slots) lg++;
  const int cluster = 1 << lg;
  // few clusters: so much shared memory that their CTAs come to lie on an SM each (16384 positions 20.2 -> 16.8 us); of more, two come to lie on one
  const bool apart = 2 * units * cluster <= x.sms;
  // Microseconds of either way behind what both cost: a block takes a quarter of an SM 0.3 (hd 128, 8 columns), a CTA alone twice as long a warp; parts
  // in the line cost 6, or 5 where no CTA has parts of two units (one token, 32 / 8 heads, 128 entries, cluster and line: batch 1 at 4096 positions 7.2,
  // 9.4 us, at 12000 12.6, 11.8, at 32768 26.0, 16.6; batch 2 at 8192 14.2, 15.2, at 12000 18.3, 17.0, at 16384 22.7, 19.0; batch 4 at 16384 25.0, 26.6;
  // batch 16 at 8192 40.9, 43.4)
  const double each = 0.3 * std::max(1.0, HD * NT / 128.0);
  const double ctas = apart ? 1. : std::max((double)sp_per_sm(HD, NT), (double)((units * cluster + x.sms - 1) / x.sms));
  const bool line = (long long)a.n_kv * p.col_blocks > 65535 || a.B > 65535 ||
                    each * units * n_blk / (4.0 * x.sms) + (slots % units ? 6 : 5) < 2 * each * ctas * n_blk / (SP_WARPS * cluster);
  p.cluster_log2 = line ? -1 : lg;
  const dim3 grid = line ? dim3((unsigned)std::min<long long>(slots, (units * n_blk + SP_WARPS - 1) / SP_WARPS))
                         : dim3((unsigned)cluster, (unsigned)(a.n_kv * p.col_blocks), (unsigned)a.B);
  const int smem = !line && apart ? std::max(sp_smem<HD, NT>(), 120 * 1024) : sp_smem<HD, NT>();
  return launch(s, launches, attend_split_kernel<T, HD, NT, PK>, grid, dim3(SP_WARPS * 32), (size_t)smem, line ? 1 : cluster, p);
}
int attend(cudaStream_t s, int dtype, const Attend &a, const Scratch &x, uint64_t *launches) {
  if (!a.d_pos && a.first >= (long long)a.pos0 + a.S)   // no row sees anything (and a line of no blocks would have no CTA to say so)
    return (int)cudaMemsetAsync(a.out, 0, (size_t)a.B * a.S * a.n_heads * a.hd * 2, s);
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    constexpr int HD = hd.value;
    const long long cols = (long long)a.S * (a.n_heads / a.n_kv), heads = (long long)a.B * a.n_kv;
    // more rows are cut into smaller pieces while their clusters leave a third of the SMs without work and a warp has few blocks (4 rows of 8 / 2
    // heads of 64 at 1000 positions 7.3 -> 5.2 us, 4 of 32 / 8 of 128 at 500 8.7 -> 6.7; on all SMs it costs more than it saves: 3 at 2000 9.6 -> 10.3)
    const int n_blk = a.d_pos ? a.blocks : (a.pos0 + a.S - 1) / BLOCK - a.first / BLOCK + 1;
    int lg = 0;
    while (lg < SP_CLUSTER_LOG2 && SP_WARPS << lg < n_blk) lg++;
    auto room = [&](int rows) { return n_blk <= 8 * SP_WARPS << lg && 3 * (heads * ((cols + rows - 1) / rows) << lg) <= 2 * x.sms; };
    if (cols <= 4 || room(4)) return attend_split<T, HD, 1, 2>(s, a, x, launches);
    if (HD == 256 || cols <= 8 || room(8)) return attend_split<T, HD, 1, 1>(s, a, x, launches);
    return attend_split<T, HD, HD == 256 ? 1 : 2, 1>(s, a, x, launches);
  });
}
// two parts a CTA, two CTAs per SM
size_t scratch_floats(int sms) { return (size_t)sms * 4 * 16 * (256 + 2); }
size_t scratch_tickets(int sms) { return (size_t)sms * 2; }
template <typename T, int HD, int NT, int PK> static int big_smem() {
  cudaError_t e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT, PK>, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(sp_smem<HD, NT>(), 120 * 1024));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_split_kernel<T, HD, NT, PK>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
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
