// Whether any memory that a call writes is also another tensor's that it writes or reads: plain C++.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>

namespace tms {

// The written ranges and the ones only read, each in order of their addresses (a model's mostly are
// already), are gone through together, each against the range that reaches furthest so far.
class RangeList {
  struct Range {
    uintptr_t begin, end;
    int64_t tensor;
    bool operator<(const Range& o) const { return begin < o.begin; }
  };
  Range few[512];
  std::unique_ptr<Range[]> many;
  Range *written = nullptr, *read = nullptr;  // one from the front, one from the back of the room
  int64_t nw = 0, nr = 0;

 public:
  bool room(int64_t ranges) {
    Range* at = few;
    if (ranges > 512) {
      many.reset(new (std::nothrow) Range[(size_t)ranges]);
      at = many.get();
      if (!at) return false;
    }
    written = at;
    read = at + ranges;
    return true;
  }
  void writes(const void* p, int64_t bytes, int64_t tensor) { written[nw++] = {(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, tensor}; }
  void reads(const void* p, int64_t bytes, int64_t tensor) {
    *--read = {(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, tensor};
    nr++;
  }
  // The tensors of two ranges that overlap, one of them written.
  bool overlap(int64_t& one, int64_t& two) {
    std::reverse(read, read + nr);
    if (!std::is_sorted(written, written + nw)) std::sort(written, written + nw);
    if (!std::is_sorted(read, read + nr)) std::sort(read, read + nr);
    Range far = {}, far_written = {};  // of all, and of those written
    for (int64_t w = 0, r = 0; w < nw || r < nr;) {
      const bool writes = r == nr || (w < nw && written[w].begin <= read[r].begin);
      const Range& x = writes ? written[w++] : read[r++];
      const Range& other = writes ? far : far_written;
      if (x.begin < other.end) {
        one = other.tensor;
        two = x.tensor;
        return true;
      }
      if (x.end > far.end) far = x;
      if (writes) far_written = x;  // written ranges that passed do not overlap: the last one reaches furthest
    }
    return false;
  }
};

}  // namespace tms
