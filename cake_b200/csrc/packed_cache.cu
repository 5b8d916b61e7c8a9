// packed_cache.cu — kernels of the cache in four bits (format and interface: packed_cache.cuh)
#include "packed_cache.cuh"
#include "common.cuh"

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

// a warp takes one query row of one head and walks its keys, 256 / HD at a time
template <typename T, int HD>
__global__ void __launch_bounds__(128) attend_rows_kernel(const Attend a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LPR = HD / 8, RW = 32 / LPR, NG = HD / 32;
  const int lane = threadIdx.x & 31, u = lane % LPR, sub = lane / LPR;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (long long)a.B * a.S * a.n_heads) return;
  const int h = (int)(item % a.n_heads), t = (int)(item / a.n_heads % a.S), b = (int)(item / a.n_heads / a.S);
  const int pos = (a.d_pos ? *a.d_pos : a.pos0) + t;
  const int first = a.d_pos ? (a.window > 0 ? max(0, pos + 1 - a.window) : 0) : a.first;
  const char *slab = reinterpret_cast<const char *>(a.cache) + (size_t)(b * a.n_kv + h / (a.n_heads / a.n_kv)) * a.blocks * block_bytes(HD);
  float q[8], acc[8] = {};
  unpack8<T>(*reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.q) + b * a.q_batch + t * a.q_tok + (size_t)h * HD + 8 * u), q);
  float qs = 0.f, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) qs += q[i];
  for (int j0 = first; j0 <= pos; j0 += RW) {
    const int j = j0 + sub, r = j & 15;
    const bool seen = j <= pos;
    float s = 0.f;
    uint32_t vw = 0;
    float2 vp = {0.f, 0.f};
    if (seen) {
      const char *blk = slab + (size_t)(j >> 4) * block_bytes(HD);
      const uint32_t kw = codes8<HD>(blk, 0, r, u);
      const float2 kp = open_pair<T>(reinterpret_cast<const uint32_t *>(blk + k_pairs(HD))[r * NG + (u >> 2)]);
#pragma unroll
      for (int i = 0; i < 8; i++) s = fmaf(q[i], (float)(kw >> (4 * i) & 15u), s);
      s = fmaf(s, kp.x, qs * kp.y);
      vw = codes8<HD>(blk, 1, r, u);
      vp = open_pair<T>(reinterpret_cast<const uint32_t *>(blk + v_pairs(HD))[r * NG + (u >> 2)]);
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (!seen) continue;   // (the lanes of a row agree)
    s *= a.scale;
    const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), e = expf(s - mn);
    m = mn;
    l = fmaf(l, f, e);
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = fmaf(acc[i], f, e * fmaf(vp.x, (float)(vw >> (4 * i) & 15u), vp.y));
  }
  // the warp's rows of keys join
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o), mn = fmaxf(m, m2);
    const float f = m == -INFINITY ? 0.f : expf(m - mn), f2 = m2 == -INFINITY ? 0.f : expf(m2 - mn);
    m = mn;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = acc[i] * f + __shfl_xor_sync(0xffffffffu, acc[i], o) * f2;
  }
  if (sub) return;
  const float inv = first > pos ? 0.f : 1.f / l;
  *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + ((size_t)(b * (long long)a.S + t) * a.n_heads + h) * HD + 8 * u) =
      make_uint4(pack2x<T>(acc[0] * inv, acc[1] * inv), pack2x<T>(acc[2] * inv, acc[3] * inv), pack2x<T>(acc[4] * inv, acc[5] * inv),
                 pack2x<T>(acc[6] * inv, acc[7] * inv));
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
int attend(cudaStream_t s, int dtype, const Attend &a, uint64_t *launches) {
  return by_type(dtype, a.hd, [&](auto t, auto hd) {
    typedef decltype(t) T;
    const long long warps = (long long)a.B * a.S * a.n_heads;
    return launch(s, launches, attend_rows_kernel<T, hd.value>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, a);
  });
}

}  // namespace pc
}  // namespace cake
