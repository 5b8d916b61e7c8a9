// paged_cache.cuh — K and V rows of many sequences in pages of one pool (cake_b200_pages_create): the format, and the launch interface of the kernels in
// paged_cache.cu that append a step's rows, attend over them and read them back.  Which page belongs to whom: paged_plan.hpp.
//
// Place.  A page of a block is, for every key head, `page` rows of K and behind them `page` rows of V, in D.  Rows lie in groups of eight; a group is hd / 64
// pieces of 1024 bytes, the eight rows' 64 entries of that range, and in a piece the 16-byte chunk c of row r (r = 0 .. 7) lies at place c ^ r.  That
// is how an operand of a matrix product lies in shared memory under the 128-byte swizzle, rows side by side as well as entries side by side, so that plain bulk
// copies of whole groups, of any page size, are what ldmatrix reads without bank conflicts and what tcgen05 takes by a descriptor (groups hd / 64 KB apart,
// the 64-entry ranges 1 KB).
//
// Marks.  A word for each page and key head of a block says whether a V row with an infinity or a NaN has ever been written there; the pool begins as zeros.  So
// where there is no mark, a weight of zero makes zero of whatever the page holds (rows behind a sequence's last, a former owner's), and nothing of it has to
// be looked at; where there is one, the kernels sum only what a row sees.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "paged_plan.hpp"

namespace cake {
namespace pg {

// byte offset of chunk c (8 entries) of row r in the K or V rows of a page and key head
__host__ __device__ constexpr size_t chunk_at(int hd, int r, int c) {
  return (size_t)((r >> 3) * (hd >> 6) + (c >> 3)) * 1024 + (size_t)((r & 7) * 128 + (((c & 7) ^ (r & 7)) * 16));
}
__host__ __device__ constexpr size_t rows_bytes(int hd, int rows) { return (size_t)rows * hd * 2; }
inline bool head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }
inline bool page_ok(int page) { return page >= 16 && page <= 1024 && (page & (page - 1)) == 0; }

// dtype codes are those of include/cake_b200.h (0 bf16, 1 f16).  Every function returns a cudaError_t cast to int and adds its launches to *launches.

struct StepHead { uint64_t shape; int n_seqs, n_rows, n_updates, pad[3]; };   // then SeqRow[n_seqs], then the updates of the table
// A step's sequences and rows for the kernels: the table's new entries and, for every row, its sequence's row of the table and its position
int spread(cudaStream_t, const StepHead *step, int n_seqs, int n_updates, int most_rows, int *table, int2 *rows, uint64_t *launches);

// what all calls on one block of a cache have in common
struct Pool {
  char *pages;                   // this block's
  uint32_t *marks;               // [page][key head]
  const int *table;              // [sequence][per_seq]
  const StepHead *step;          // on the device: the shape it has now
  uint64_t shape;                // the shape that the call was made for; another one now (a replayed graph): *bad is set, nothing is done
  int *bad;
  int n_kv, hd, page_log2, per_seq;
};
struct Append {
  const int2 *rows;              // [n_rows] (sequence, position)
  const void *q, *k, *v;         // rows of head 0, 16-byte aligned; q may be nullptr (then n_q is 0)
  void *q_out;                   // may be q
  long long q_tok, k_tok, v_tok, out_tok;   // strides of rows in entries, multiples of 8; heads lie side by side
  const float *cos_t, *sin_t;    // [positions][rot / 2], or nullptr: no rotation
  const void *q_norm, *k_norm;   // RMS norms over hd in front of the rotation, or nullptr
  int n_rows, n_q, rot;
  float eps;
  bool as_blocks;                // rounded to D behind the norm and behind each product of the rotation
};
int append(cudaStream_t, int dtype, const Pool &, const Append &, int sms, uint64_t *launches);

// rows of the present step (rows), or positions first .. of sequence slot (rows == nullptr) -> k, v [n][n_kv][hd]; either may be nullptr
struct Read { const int2 *rows; int slot, first, n; void *k, *v; };
int read(cudaStream_t, const Pool &, const Read &, int sms, uint64_t *launches);

// A step's attention as it is cut for one window (paged_plan.hpp), on the device: this head, few_ctas workers and as many cuts of the few-row kernel, the items of
// the many-row kernel.  What the calls on a cache share: sums of runs and tiles that are cut
struct PlanHead { int W, n_cuts, n_items, parts, n_cut_tiles, pad[3]; };   // workers, cut runs; items, parts of tiles that are cut, such tiles (their first items behind the items)
struct Scratch {
  float *few_ws, *tiles_ws;      // few_floats; tiles_floats (nullptr: the step has no sequence of many rows)
  int sms;
  const struct Clusters *clusters;
};
// clusters of 1, 2, 4 and 8 CTAs of the few-row kernel (up to 8 query rows, up to 16) that are on the chip at once
struct Clusters { int most[2][4]; };
int few_ctas(int hd, int sms);             // CTAs of the few-row kernel: no more workers than that
int room(int hd, int sms, int n_kv);       // items of the many-row kernel that fill the chip (parts of cut ones: twice as many at most)
size_t few_floats(int hd, int sms);
size_t tiles_floats(int hd, int sms, int n_kv);
int prepare(int dtype, int hd, Clusters *);   // once per device and kind of cache, in front of the first call
struct Attend {
  const void *q;
  long long q_tok;               // multiple of 8
  void *out;                     // [rows, n_heads, hd]
  const SeqRow *seqs;
  int n_heads;
  float scale;
  Window win;
  const PlanHead *plan;
  int n_few, few_cols;           // sequences of few rows, query rows of a key head that they have at most
  int longest, tiles;            // tiles of their longest run, of all; of a captured call, whose lengths may become any: the most that a run can have, and 0
  int n_cuts, n_items;           // runs that are cut, items of the many-row kernel; of a captured call: as many as any plan of the step's shape can have
  int most_items;                // that many items: the list of cut tiles is behind them
  int n_cut_tiles;               // tiles that are cut (of a captured call: as many as may be)
  int *err;
};
int attend(cudaStream_t, int dtype, const Pool &, const Attend &, const Scratch &, uint64_t *launches);

}  // namespace pg
}  // namespace cake
