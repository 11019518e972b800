// The rotation of whole heads (layer.cu), as xdna_rotary and the append to a paged cache (paged.cu) launch it.
#pragma once

#include "host_util.h"

namespace xdna {

struct RotaryArgs {
  const void* x;        // [T, H, D]
  int64_t x_st, x_sh;   // strides of a token and of a head, in elements
  void* out;            // [T, H, D], contiguous
  const void* positions;  // [T], or NULL: the tokens of sequences that have starts[i] tokens before them
  int position_bytes;
  const int32_t *starts, *cu;  // cu NULL: token i is sequence i's next one
  int n_seqs;
  const float* inv_freq;
  int n_freq;
  float factor;
  const void* norm;
  int norm_dtype;
  int64_t norm_sh;  // 0: one norm for all heads
  float eps;
  int64_t T;
  int H, D, wpt;  // wpt: warps of a token
};

int launch_rotary(const RotaryArgs& a, int dtype, bool interleaved, int sms, cudaStream_t s);

#ifdef __CUDACC__
// A token's sequence and position; `there` is false for tokens of no sequence.
struct Place {
  int64_t position;
  int seq;
  bool there;
};

// Sequence i has the tokens cu[i] .. cu[i + 1] - 1, clamped to [0, T]; starts[i] < 0: nothing of it is taken.
__device__ __forceinline__ Place place_in(const int32_t* starts, const int32_t* cu, int n_seqs, int64_t token) {
  if (cu == nullptr) {
    const int start = starts[token];
    return {start, static_cast<int>(token), start >= 0};
  }
  int lo = 0, hi = n_seqs;  // the last word that is not past the token lies in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= token)
      lo = mid;
    else
      hi = mid;
  }
  if (n_seqs < 1) return {0, 0, false};
  const int first = max(cu[lo], 0), start = starts[lo];
  return {static_cast<int64_t>(start) + token - first, lo, start >= 0 && token >= first && token < cu[lo + 1]};
}

__device__ __forceinline__ Place place_of(const RotaryArgs& a, int64_t token) {
  if (a.positions == nullptr) return place_in(a.starts, a.cu, a.n_seqs, token);
  return {a.position_bytes == 8 ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int32_t*>(a.positions)[token], 0,
          true};
}
#endif

}  // namespace xdna
