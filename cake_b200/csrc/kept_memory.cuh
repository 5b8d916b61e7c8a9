// kept_memory.cuh — scratch memory of a ctx that grows with the calls that use it, where captured calls may use it too.
//
// A captured call leaves the memory's address in its graph (kernel arguments, tensor maps), and the graph may be replayed whenever nothing else of
// the ctx runs: after later calls too, which may have needed more.  So memory that a capture has used is never given back before the ctx goes: it is kept
// beside the larger one.  Memory that no capture has used is given back before the larger one is asked for.
#pragma once
#include <algorithm>
#include <cstddef>
#include <vector>

namespace cake {

struct KeptMemory {
  void *now = nullptr;        // what the next call takes
  size_t cap = 0;
  bool recorded = false;      // a capture has used it
  std::vector<void *> kept;   // replaced ones that captures have used

  // Whether a call has to make memory first (a call inside a capture cannot); where it has not, the call's use is noted.
  bool short_of(size_t need, bool capturing) {
    if (need > cap) return true;
    recorded = recorded || capturing;
    return false;
  }
  // `need` bytes for a call outside a capture, at least twice what there was where that is no more than `most`, so that growing calls seldom grow it.
  // make(bytes): the memory or nullptr; release(p).  Without memory for it: nullptr, and what captures have used is still there.
  template <typename Make, typename Release> void *grow(size_t need, size_t most, Make &&make, Release &&release) {
    const size_t more = std::max(need, std::min(2 * cap, most));
    kept.reserve(kept.size() + 1);
    if (now) {
      if (recorded) kept.push_back(now);
      else release(now);
    }
    now = nullptr; cap = 0; recorded = false;
    for (size_t bytes : {more, need}) {
      now = make(bytes);
      if (now) { cap = bytes; break; }
      if (bytes == need) break;
    }
    return now;
  }
  template <typename Release> void release_all(Release &&release) {
    for (void *p : kept) release(p);
    if (now) release(now);
    kept.clear();
    now = nullptr; cap = 0; recorded = false;
  }
};

}  // namespace cake
