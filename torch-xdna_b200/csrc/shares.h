// How paged_attention's work is shared out and which parts of an item are joined: arithmetic that the host can check too.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define XDNA_BOTH __host__ __device__ __forceinline__
#else
#define XDNA_BOTH inline
#endif

namespace xdna {

// All units (tiles, or steps of one tile for each of a CTA's warps) in order, shared out evenly: the first `more` shares
// have one more than the others.
struct Shares {
  int64_t work, each, more;
  XDNA_BOTH Shares(int64_t work, uint32_t shares) : work(work) {
    each = work >> 31 ? work / shares : static_cast<uint32_t>(work) / shares;
    more = work - each * shares;
  }
  XDNA_BOTH int64_t begin(int64_t i) const { return i * each + (i < more ? i : more); }
  XDNA_BOTH int owner(int64_t unit) const {  // the share that has it
    const int64_t cut = more * (each + 1), from = unit < cut ? unit : unit - cut, by = unit < cut ? each + 1 : each;
    const int64_t i = work >> 31 ? from / by : static_cast<uint32_t>(from) / static_cast<uint32_t>(by);
    return static_cast<int>(unit < cut ? i : more + i);
  }
};

// The parts of an item are those of shares first .. last, the first one's in `slot` (a share has the slots 2 i and 2 i + 1),
// the others' in slot 2 i. Whether an item's entry is such a one: where a share's wait ran out, the entries of the items
// that begin in what was left of it have not been written, and hold whatever was in the workspace.
XDNA_BOTH bool parts_exist(int first, int last, int slot, int shares) {
  return 0 <= first && first <= last && last < shares && (slot >> 1) == first;
}

}  // namespace xdna
