// packed_cache.cuh — a session's K and V rows in four bits (cake_b200_cache_create_packed): the format, and the launch interface of the
// kernels in packed_cache.cu that write rows, read them back and attend over them.
//
// Format.  A row of hd entries (K: after norm and rotation) is cut into hd / 32 groups of neighbours.  With lo = min x (a D number) and step the
// smallest D number that is not below (max x - lo) / 15 (D = bf16: and not below 2^-126 where the span is not 0), entry x is held as
// n = floor((x - lo) / step + 1/2), 0 <= n <= 15, and stands for lo + step n.  A pair (step, lo) in D and 32 codes are 20 bytes for 32 entries.
// step is rounded up so that 15 steps reach the maximum; lo and step are D numbers, so that n step is exact in fp32.  Span and distances are formed in
// fp32 and exact there unless the exponents lie so far apart that 24 bits do not hold a difference of two D numbers: step can then be its neighbour (f16,
// lo = -2^-24, max = 15360: 1024 for 1025).  A group whose span is not finite (an infinity, a NaN) has the pair (NaN, NaN): all of it reads as NaN.  What lies beyond D's
// largest number, as 15 steps may, is rounded to it.
//
// Place.  16 positions of one (batch row, key head) are one block of 20 hd bytes: K's codes, K's pairs, V's codes, V's pairs; the blocks of a
// (batch row, key head) follow one another, so that keys and values of a range of positions are one piece of memory.  Inside a block the
// codes lie as the m16n8k16 products of the attention take them, a lane's codes side by side (lane = 4 g + t holds rows g and g + 8 and
// columns 2t, 2t + 1, 2t + 8, 2t + 9 of an operand); 8 codes are a 32-bit word:
//   K, position r:  word t hd/32 + j of the row holds entries 32 j + 8 t .. + 7; nibble i entry 2 i, nibble 4 + i entry 2 i + 1
//   V, positions r and r + 1 (r even): lane 4 g + (r & 7) / 2 has a word for every group j, r >> 3 and r's neighbour: entries 32 j + 4 g .. + 3 of r in
//                   nibbles 0 .. 3 and of r + 1 in nibbles 4 .. 7; a lane's words lie in pieces of 16 bytes, the pieces of all lanes side by side
//   pairs:          a row's even groups, then its odd ones: word r hd/32 + (j & 1) hd/64 + j / 2, step in the low half, lo in the high half
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace cake {
namespace pc {

constexpr int GROUP = 32, BLOCK = 16;   // entries of a pair; positions of a block
__host__ __device__ constexpr int block_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int k_pairs(int hd) { return 8 * hd; }        // byte offsets inside a block
__host__ __device__ constexpr int v_codes(int hd) { return 10 * hd; }
__host__ __device__ constexpr int v_pairs(int hd) { return 18 * hd; }
// word (of the block's K or V codes) that holds entries 8u .. 8u + 7 of K's position r
__host__ __device__ constexpr int k_word(int hd, int r, int u) { return r * (hd / 8) + (u & 3) * (hd / 32) + (u >> 2); }
// 16-bit half of V's codes that holds entries 32 j + 4 g .. + 3 of position r
__host__ __device__ constexpr int v_half(int hd, int r, int g, int j) {
  const int lane = 4 * g + ((r & 7) >> 1), idx = (r >> 3) * (hd / 32) + j;
  return (((idx >> 2) * 32 + lane) * 4 + (idx & 3)) * 2 + (r & 1);
}
__host__ __device__ constexpr int pair_word(int hd, int r, int j) { return r * (hd / 32) + (j & 1) * (hd / 64) + (j >> 1); }   // group j of position r
inline int cap_blocks(int cap) { return (cap + 63) / 64 * 4; }   // whole tiles of 64 positions
inline bool head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }

// dtype codes are those of include/cake_b200.h (0 bf16, 1 f16).  Every function returns a cudaError_t cast to int and adds its launches to *launches.

// Rows of a step join the cache.  In a block: of a fused projection [tokens, n_q + 2 n_kv heads, hd], q and k heads are normed (q_norm, k_norm)
// and rotated (cos_t), q in place; by itself (n_q == 0): k and v as they are.
struct Write {
  void *cache;
  const void *k, *v;             // rows of head 0, 16-byte aligned
  long long k_tok, k_batch, v_tok, v_batch;   // strides in elements, multiples of 8; heads lie side by side
  void *q = nullptr;             // [n_q heads] of a token, strides as k's
  const void *cos_t = nullptr, *sin_t = nullptr, *q_norm = nullptr, *k_norm = nullptr;
  int B, S, n_q = 0, n_kv, hd, rot = 0, blocks, pos0;   // blocks: of a (batch row, head)
  const int *d_pos = nullptr;    // the position on the device instead of pos0
  float eps = 0.f;
};
int write(cudaStream_t, int dtype, const Write &, uint64_t *launches);

// positions [first, first + n) of K and V (either may be nullptr) -> [B, n_kv, n, hd] in D, a (batch row, head) every out_rows rows
struct Read {
  const void *cache;
  void *k, *v;
  int B, n_kv, hd, blocks, first, n;
  long long out_rows;
  unsigned long long *nan = nullptr;   // as operands of products: [B n_kv][read_blocks], see nan_groups
};
inline int read_blocks(int first, int n) { return ((first + n - 1) >> 4) - (first >> 4) + 1; }
int read(cudaStream_t, int dtype, const Read &, uint64_t *launches);

// Row t of S (position pos0 + t) of q attends to the positions first <= j <= pos0 + t; a row without any is zero.
struct Attend {
  const void *cache, *q;         // q: heads side by side, 16-byte aligned
  long long q_tok, q_batch;      // strides in elements, multiples of 8
  void *out;                     // [B, S, n_heads, hd] D
  int B, S, n_heads, n_kv, hd, blocks, pos0, first;
  const int *d_pos = nullptr;    // S == 1: the position on the device instead of pos0; first = max(0, position + 1 - window) with window > 0
  int window = 0;
  float scale;
};
// what the calls of one stream share: sums of keys cut over several CTAs, and how many of them have come (all zero between calls)
struct Scratch {
  float *ws;          // scratch_floats
  unsigned *tickets;  // scratch_tickets
  int sms;
};
size_t scratch_floats(int sms);
size_t scratch_tickets(int sms);
int prepare(int dtype, int hd);   // once per device and kind of cache, in front of the first call
int attend(cudaStream_t, int dtype, const Attend &, const Scratch &, uint64_t *launches);
// Whether keys and values expanded once, for the kernel of prompts, are the faster way for heads of 128.  Microseconds of either:
//   on codes   a wave of pieces of 16 rows over the SMs 7, and 0.15 for each of their blocks
//   expanded   12, 2 per 1000 positions (a tile's steps) and 0.21 per 1000 positions and (batch row, key head): five bits read, 16 written and 16 read
//              again an entry
// Codes / expanded, by (batch row, key head)s in all, rows of each, and positions: 8, 64 rows: at 0 5.2 / 7.7, at 1000 10 / 16, at 16000 40 / 65;
// 8, 256: 7.6 / 8.7, 15 / 21, 122 / 75; 64, 32: 7.1 / 8.0, 15 / 24, 123 / 230; 64, 128: 26 / 10, 54 / 31, 460 / 236; 256, 20: 23 / 9, 51 / 61, 456 / 849;
// 256, 64: 45 / 11, 94 / 63, 901 / 861; 1024, 32: 94 / 26, 201 / 229, 1790 / 3600.  Of 810 such pairs (1 to 1024 of them, 17 to 256 rows, 0 to 16000
// positions, 1 to 8 query heads a key head) 19 go a way that takes over a tenth longer, 25 % at most: those of 16 clusters, which the SMs have no room for at once.
inline bool many_rows(const Attend &a, int sms) {
  const long long cols = (long long)a.S * (a.n_heads / a.n_kv), heads = (long long)a.B * a.n_kv, pieces = heads * ((cols + 15) / 16);
  const double keys = a.pos0 + 0.5 * a.S - a.first;
  const double codes = 7 * (double)((pieces + sms - 1) / sms) + 0.15 * (double)pieces / sms * keys / BLOCK;
  return a.hd == 128 && cols > 16 && codes > 12 + (2 + 0.21 * (double)heads) * keys / 1000;
}

}  // namespace pc
}  // namespace cake
