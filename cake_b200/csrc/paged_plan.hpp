// paged_plan.hpp — the host's side of a cache in pages (cake_b200_pages_create): which page belongs to which sequence, what a step brings, and how
// attention over it is cut.  No CUDA in here.
//
// A page holds `page` consecutive positions of one sequence, for every block under the same number.  A sequence takes pages as it grows and gives them back
// when it is dropped or cut; which ones it has stands in its row of the page table.
#pragma once
#include <algorithm>
#include <cstdint>
#include <vector>

namespace cake {
namespace pg {

constexpr int TILE = 64;          // positions of a tile of keys
constexpr int TOKEN_COLS = 16;    // query rows (tokens x query heads of a key head) that the kernel of few rows takes at once
constexpr int TILE_ROWS = 128;    // query rows of a tile of the kernel of many rows

struct SeqRow { int slot, pos0, count, row0; };   // a sequence of a step: its row of the page table, held positions, new rows, the first of them in the step

// One CTA's share of the few-row kernel's work: `left` tiles from tile `tile` of (sequence i, key head kvh) on, in the order of sequences, key heads, tiles
struct Worker { int i, kvh, tile, left; SeqRow s; };
// A run (sequence, key head) that is cut: in `parts` neighbouring shares from `first` on
struct Cut { SeqRow s; int kvh, first, parts, pad; };
// One CTA row of the many-row kernel (for every key head): tokens tok0 .. of sequence i against key tiles [t0, t1); part of parts, whose sums are in the
// places part0 .. of the workspace (for key head 0; the parts of all tiles follow one another)
struct Item { int i, tok0, t0, t1, part, parts, part0, tile; SeqRow s; };

struct Window { int w = 0; bool by_call = false; };   // by_call: all rows of a call see the same first position, the one of its last row (0 for a first call)
inline int first_seen(const SeqRow &s, const Window &w) {   // by the row that sees the earliest
  if (w.w <= 0) return 0;
  if (w.by_call) return s.pos0 > 0 ? std::max(0, s.pos0 + s.count - w.w) : 0;
  return std::max(0, s.pos0 + 1 - w.w);
}
inline int tile_first(const SeqRow &s, const Window &w) { return first_seen(s, w) / TILE; }
inline int tiles_of(const SeqRow &s, const Window &w) { return (s.pos0 + s.count - 1) / TILE - tile_first(s, w) + 1; }

struct Book {
  int n_pages = 0, page = 0, max_seqs = 0, max_seq = 0, per_seq = 0;   // per_seq: entries of a row of the page table
  struct Seq { bool live = false; int len = 0; std::vector<int> pages; };
  std::vector<Seq> seqs;
  std::vector<int> free_pages;
  // the present step: sequences of few rows first
  std::vector<SeqRow> step;
  std::vector<int> ids;          // the sequences as the step was given
  int n_few = 0, n_rows = 0;
  uint64_t shape = 0;            // of the counts in their order: what a captured call depends on
  std::vector<int> updates;      // (place in the table, page) of pages taken for it

  void init(int pages, int page_, int max_seqs_, int max_seq_) {
    n_pages = pages; page = page_; max_seqs = max_seqs_; max_seq = max_seq_;
    per_seq = (max_seq + page - 1) / page;
    seqs.assign((size_t)max_seqs, Seq());
    free_pages.resize((size_t)n_pages);
    for (int i = 0; i < n_pages; i++) free_pages[(size_t)i] = n_pages - 1 - i;   // taken from the end: page 0 first
  }
  bool has(int s) const { return s >= 0 && s < max_seqs && seqs[(size_t)s].live; }
  int add() {
    for (int s = 0; s < max_seqs; s++)
      if (!seqs[(size_t)s].live) {
        seqs[(size_t)s].live = true;
        seqs[(size_t)s].len = 0;
        return s;
      }
    return -1;
  }
  bool any() const { return std::any_of(seqs.begin(), seqs.end(), [](const Seq &q) { return q.live; }); }
  bool in_step(int s) const { return std::find(ids.begin(), ids.end(), s) != ids.end(); }
  void end_step() { step.clear(); ids.clear(); updates.clear(); n_few = n_rows = 0; shape = 0; }
  void cut(int s, int len) {   // what is behind len is given back
    Seq &q = seqs[(size_t)s];
    if (in_step(s)) end_step();   // (its rows have no place any more)
    const size_t keep = (size_t)((len + page - 1) / page);
    while (q.pages.size() > keep) {
      free_pages.push_back(q.pages.back());
      q.pages.pop_back();
    }
    q.len = len;
  }
  void drop(int s) {
    cut(s, 0);
    seqs[(size_t)s].live = false;
  }

  // nullptr: the step stands; else what is wrong (*which: with which entry), and nothing has changed
  enum Bad { OK, NOT_LIVE, TWICE, COUNT, TOO_LONG, NO_PAGES };
  Bad plan(const int *which, const int *counts, int n, int G, int *bad) {
    *bad = 0;
    std::vector<char> seen((size_t)max_seqs, 0);
    long long need = 0, rows = 0;
    for (int i = 0; i < n; i++) {
      *bad = i;
      if (!has(which[i])) return NOT_LIVE;
      if (seen[(size_t)which[i]]++) return TWICE;
      if (counts[i] < 1) return COUNT;
      const Seq &q = seqs[(size_t)which[i]];
      if ((long long)q.len + counts[i] > max_seq) return TOO_LONG;
      need += (long long)(q.len + counts[i] + page - 1) / page - (long long)q.pages.size();
      rows += counts[i];
    }
    if (need > (long long)free_pages.size()) return NO_PAGES;
    std::vector<SeqRow> many;   // (all memory first: what can throw does so in front of any change)
    std::vector<int> who(which, which + n);
    many.reserve((size_t)n);
    step.reserve((size_t)n);
    updates.reserve(2 * (size_t)need);
    for (int i = 0; i < n; i++) seqs[(size_t)which[i]].pages.reserve((size_t)((seqs[(size_t)which[i]].len + counts[i] + page - 1) / page));
    end_step();
    ids.swap(who);
    n_rows = (int)rows;
    shape = 1469598103934665603ull;
    for (int i = 0; i < n; i++) shape = (shape ^ (uint64_t)(uint32_t)counts[i]) * 1099511628211ull;
    shape = (shape ^ (uint64_t)n) * 1099511628211ull;
    int row0 = 0;
    for (int i = 0; i < n; i++) {
      Seq &q = seqs[(size_t)which[i]];
      const SeqRow r{which[i], q.len, counts[i], row0};
      if ((long long)counts[i] * G <= TOKEN_COLS) step.push_back(r);
      else many.push_back(r);
      row0 += counts[i];
      q.len += counts[i];
      while ((long long)q.pages.size() * page < q.len) {
        updates.push_back(which[i] * per_seq + (int)q.pages.size());
        updates.push_back(free_pages.back());
        q.pages.push_back(free_pages.back());
        free_pages.pop_back();
      }
    }
    n_few = (int)step.size();
    step.insert(step.end(), many.begin(), many.end());
    return OK;
  }

  // Few rows: all (sequence, key head)s' tiles in one line, cut into shares of the same cost: a tile 1, a piece of a run RUN_COST more (its sums have to be
  // brought together).  A piece that would leave a single tile to the next share takes it.  RUN_COST 0.5, 1, 2, 4:  32 sequences to 8191 positions (8 key heads of 128)
  // 60.6, 59.0, 60.1, 62.5 us, 9 of 3 to 5 rows to 5000 17.1, 18.3, 22.5, 26.4, 100 in a window of 1024 (2 of 64) 10.7, 11.3, 12.7, 16.3.
  void cut_few(const Window &win, int n_kv, int most, std::vector<Worker> *out, std::vector<Cut> *cuts) const {
    constexpr double RUN_COST = 0.5;
    out->clear();
    cuts->clear();
    long long total = 0;
    for (int i = 0; i < n_few; i++) total += (long long)tiles_of(step[(size_t)i], win) * n_kv;
    const int W = (int)std::min<long long>(most, total);
    double rest = (double)total + RUN_COST * n_few * n_kv;
    int i = 0, h = 0, k = 0, t = W ? tiles_of(step[0], win) : 0, first = 0;   // the next tile; the share where its run began
    for (int w = 0; w < W && i < n_few; w++) {
      const double goal = rest / (W - w);
      Worker x{i, h, k, 0, step[(size_t)i]};
      double load = 0;
      while (i < n_few) {
        const double room = goal - load - RUN_COST;
        if (x.left && room < 0.5) break;
        int n = std::max(1, std::min(t - k, (int)(room + 0.5)));
        if (t - k - n <= 1 || w == W - 1) n = t - k;
        if (!k) first = w;
        x.left += n;
        k += n;
        load += RUN_COST + n;
        rest -= n;
        if (k < t) break;
        if (first < w) cuts->push_back(Cut{step[(size_t)i], h, first, w - first + 1, 0});
        rest -= RUN_COST;
        k = 0;
        if (++h == n_kv) {
          h = 0;
          if (++i < n_few) t = tiles_of(step[(size_t)i], win);
        }
      }
      out->push_back(x);
    }
  }
  // Many rows: a CTA row per tile of 128 query rows, the one with the most keys first.  `room` CTA rows run at once; a tile with more keys than an equal share
  // of them is cut into parts of a like size, of LEAST key tiles or more.  Returns the parts of all tiles that are cut, at most 2 room
  int cut_many(const Window &win, int G, int room, std::vector<Item> *out) const {
    constexpr int LEAST = 4;
    out->clear();
    const int tpt = TILE_ROWS / G;
    std::vector<Item> whole;
    long long total = 0;
    for (int i = n_few; i < (int)step.size(); i++) {
      const SeqRow &s = step[(size_t)i];
      for (int tok = 0; tok < s.count; tok += tpt) {
        const int last = s.pos0 + std::min(tok + tpt, s.count) - 1;
        SeqRow head = s;   // the tile's first token sees the earliest position
        if (!win.by_call) head.pos0 += tok;
        const int t0 = tile_first(head, win), t1 = last / TILE + 1;
        whole.push_back(Item{i, tok, t0, t1, 0, 1, 0, 0, s});
        total += t1 - t0;
      }
    }
    std::stable_sort(whole.begin(), whole.end(), [](const Item &a, const Item &b) { return a.t1 - a.t0 > b.t1 - b.t0; });
    // key tiles of a part: an equal share of the chip, and more where the parts would not fit it side by side
    long long share = std::max<long long>(LEAST, (total + room - 1) / room);
    auto cut = [&](int n) { return n > share ? (int)((n + share - 1) / share) : 1; };
    auto all = [&]() {
      long long p = 0;
      for (const Item &x : whole) p += cut(x.t1 - x.t0);
      return p;
    };
    if ((int)whole.size() <= room)
      while (all() > room) share++;
    int parts = 0;
    for (size_t k = 0; k < whole.size(); k++) {
      Item it = whole[k];
      const int n = it.t1 - it.t0, p = cut(n);
      it.tile = (int)k;
      it.parts = p;
      it.part0 = p > 1 ? parts : 0;
      if (p > 1) parts += p;
      for (int j = 0; j < p; j++) {
        Item x = it;
        x.part = j;
        x.t0 = it.t0 + (int)((long long)n * j / p);
        x.t1 = it.t0 + (int)((long long)n * (j + 1) / p);
        out->push_back(x);
      }
    }
    return parts;
  }
  // what a step of at most `rows` rows can need at most
  static size_t most_items(long long rows, int max_seqs, int G, int room) {
    const int tpt = TILE_ROWS / G;
    return (size_t)(rows / tpt + max_seqs + 2 * room);
  }
};

}  // namespace pg
}  // namespace cake
