// A cache of keys and values in pages and in 8 bits, and the two calls that a decode step makes of it: appending
// (xdna_cache_append), with the norm and the rotation of the keys on the way, and attention (xdna_paged_attention).
//
// Codes lie as [pages][Hkv][page][D] bytes, int8 or e4m3, a page being 16, 32, 64 or 128 tokens; a block is one head's
// part of a page, D * page contiguous bytes, and has one scale: x = code * scale. An append writes powers of two.
// table[b][i] is the page of sequence b's tokens i * page .. (i + 1) * page - 1.
#include <cuda_fp8.h>

#include <algorithm>

#include "host_util.h"
#include "rotary.cuh"
#include "rotary.h"
#include "shares.h"

namespace xdna {

// ---------------------------------------------------------------------------- codes
// A block's scale is the least 2^e, e >= -126, with max |x| <= top * 2^e (top 127 for int8, 448 for e4m3), so x / 2^e is
// exact, no code is out of range, and a code whose block's scale grows is only halved, which loses nothing in e4m3 but at
// its lowest values, and less than one step of the new scale in int8 however often it happens (1/2 + 1/4 + ...).
// An infinity or a NaN makes the block's scale NaN.
__device__ __forceinline__ int block_exponent(uint32_t top_bits, bool e4m3) {
  const int e = static_cast<int>(top_bits >> 23) - 127;
  const uint32_t mantissa = top_bits & 0x7fffffu;
  return max(e4m3 ? e - 8 + (mantissa > 0x600000u) : e - 6 + (mantissa > 0x7e0000u), -126);
}
constexpr uint32_t kNotFinite = 0x7f800000u;
constexpr uint32_t kMostScale = 0x7e800000u;  // 2^126; above it as bits: what is larger, not finite or below zero
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // -126 .. 127

// What an append makes of a block: the scale, 1 / scale for the new values, and the factor of the older codes.
struct BlockChange {
  float scale, inverse, older;  // inverse 0: not finite; older 1: they stay
};
__device__ __forceinline__ BlockChange change_block(uint32_t top_bits, bool has_older, uint32_t old_bits, bool e4m3) {
  if (top_bits >= kNotFinite || (has_older && old_bits > kMostScale)) return {__uint_as_float(0x7fc00000u), 0.f, 1.f};
  int e = block_exponent(top_bits, e4m3);
  float older = 1.f;
  if (has_older) {  // their scale is held by the least power of two from it on: itself, where an append wrote it
    e = max(e, static_cast<int>(old_bits >> 23) - 127 + ((old_bits & 0x7fffffu) != 0));
    older = __uint_as_float(old_bits) * power_of_two(-e);
  }
  return {power_of_two(e), power_of_two(-e), older};
}

// Four values to codes; they are within the codes' range.
template <bool E4M3>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    return lo | static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16;
  } else {
    // 1.5 * 2^23 + x is x's rounding to whole numbers, in the lowest bits
    auto whole = [](float x) { return __float_as_uint(x + 12582912.f); };
    return __byte_perm(__byte_perm(whole(a), whole(b), 0x0040), __byte_perm(whole(c), whole(d), 0x0040), 0x5410);
  }
}
// Two half pairs, exactly, of the four codes of a word, lowest first. int8: 1024 + (code + 128) is the half 0x6400 | byte.
template <bool E4M3>
__device__ __forceinline__ void to_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), off), q = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&q);
  }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t rescale_codes(uint32_t w, float by) {
  uint32_t lo, hi;
  to_halves<E4M3>(w, lo, hi);
  const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&lo)), q = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return to_codes<E4M3>(p.x * by, p.y * by, q.x * by, q.y * by);
}
// The first `bytes` (a multiple of 16) of a block, by `threads` threads of which this is number i.
template <bool E4M3>
__device__ __forceinline__ void rescale_block(uint8_t* block, int bytes, float by, int i, int threads) {
#pragma unroll 4
  for (int at = i * 16; at < bytes; at += threads * 16) {
    uint4 u = *reinterpret_cast<const uint4*>(block + at);
    u.x = rescale_codes<E4M3>(u.x, by), u.y = rescale_codes<E4M3>(u.y, by);
    u.z = rescale_codes<E4M3>(u.z, by), u.w = rescale_codes<E4M3>(u.w, by);
    *reinterpret_cast<uint4*>(block + at) = u;
  }
}
__device__ __forceinline__ void rescale_block(uint8_t* block, int bytes, float by, bool e4m3, int i, int threads) {
  e4m3 ? rescale_block<true>(block, bytes, by, i, threads) : rescale_block<false>(block, bytes, by, i, threads);
}

// ---------------------------------------------------------------------------- append
struct AppendArgs {
  const void *k, *v, *q;  // q NULL: no queries
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;
  uint8_t *kc, *vc;       // codes
  int64_t kc_sp, vc_sp;   // bytes from page to page
  float *ks, *vs;         // scales
  int64_t ks_sp, vs_sp;
  const int32_t* table;
  int64_t ld_table;
  const int32_t *starts, *cu;
  const float* inv_freq;
  const void *k_norm, *q_norm;
  int64_t k_norm_sh, q_norm_sh;
  void* q_out;
  int64_t tokens;
  float factor, eps;
  int k_norm_dtype, q_norm_dtype;
  int n_freq, n_seqs, hq, hkv, page, page_shift, pages, max_pages;
  bool e4m3;
  int heads;  // of a block of threads (packed)
};

template <int D, int V>
struct RowShape {
  static constexpr int kLanes = V == 8 ? D / 16 : 32, kUnits = V == 8 ? 1 : D / 64, kRows = 32 / kLanes;
  static constexpr int kPerLane = 2 * V * kUnits;
  static_assert(V == 8 || V == 1, "16-byte pieces, or single entries where pairs lie at odd distances");
};

template <typename T, int D, int V>
struct RawRow {
  Pack<T, V> p[RowShape<D, V>::kUnits][2];
};
template <typename T, int D, int V>
__device__ __forceinline__ RawRow<T, D, V> load_row(const T* x, const UnitAt* u) {
  RawRow<T, D, V> r;
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) r.p[k][0] = load_pack<T, V>(x + u[k].lo), r.p[k][1] = load_pack<T, V>(x + u[k].hi);
  return r;
}
template <typename T, int D, int V>
__device__ __forceinline__ void row_floats(const RawRow<T, D, V>& r, float (*f)[2 * V]) {
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) to_floats<T, V>(r.p[k][0], f[k]), to_floats<T, V>(r.p[k][1], f[k] + V);
}
// 1 / sqrt(mean of x^2 + eps) of a row, on all its lanes.
template <int D, int V>
__device__ __forceinline__ float row_inverse(const float (*f)[2 * V], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) {
    ss += squares<2 * V>(f[k]);
  }
  return inverse_root(fmaf(sum_of_lanes<RowShape<D, V>::kLanes>(ss), 1.f / D, eps));
}
template <int D, int V>
__device__ __forceinline__ void norm_row(float (*f)[2 * V], const UnitAt* u, const void* norm, int dtype, int64_t at, float inverse) {
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) {
    float g[2 * V];
    load_weights<V>(norm, dtype, at + u[k].lo, g);
    load_weights<V>(norm, dtype, at + u[k].hi, g + V);
    scale_by<2 * V>(f[k], inverse, g);
  }
}
// The largest |x| of a lane's share of a row, as bits, NaN where one is (above infinity, and that above all numbers); of
// the row.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int D, int V>
__device__ __forceinline__ uint32_t lane_top(const float (*f)[2 * V]) {
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) {
#pragma unroll
    for (int i = 0; i < 2 * V; i += 2) top = max_abs(top, f[k][i], f[k][i + 1]);
  }
  return __float_as_uint(top) & 0x7fffffffu;
}
template <int D, int V>
__device__ __forceinline__ uint32_t row_top(const float (*f)[2 * V]) {
  uint32_t top = lane_top<D, V>(f);
#pragma unroll
  for (int o = RowShape<D, V>::kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  return top;
}
template <int D, int V, bool E4M3>
__device__ __forceinline__ void store_codes(uint8_t* row, const float (*f)[2 * V], const UnitAt* u, float inverse) {
#pragma unroll
  for (int k = 0; k < RowShape<D, V>::kUnits; ++k) {
    float x[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; i += 2) {
      const float2 y = __fmul2_rn(make_float2(f[k][i], f[k][i + 1]), make_float2(inverse, inverse));
      x[i] = y.x, x[i + 1] = y.y;
    }
    if constexpr (V == 8) {
      *reinterpret_cast<uint2*>(row + u[k].lo) = make_uint2(to_codes<E4M3>(x[0], x[1], x[2], x[3]), to_codes<E4M3>(x[4], x[5], x[6], x[7]));
      *reinterpret_cast<uint2*>(row + u[k].hi) = make_uint2(to_codes<E4M3>(x[8], x[9], x[10], x[11]), to_codes<E4M3>(x[12], x[13], x[14], x[15]));
    } else {
      const uint32_t c = to_codes<E4M3>(x[0], x[1], 0.f, 0.f);
      row[u[k].lo] = static_cast<uint8_t>(c);
      row[u[k].hi] = static_cast<uint8_t>(c >> 8);
    }
  }
}
// inverse 0: a block that is not finite, whose codes are 0.
template <int D, int V>
__device__ __forceinline__ void store_codes(uint8_t* row, const float (*f)[2 * V], const UnitAt* u, float inverse, bool e4m3) {
  if (inverse == 0.f) {
    const float zeros[RowShape<D, V>::kUnits][2 * V] = {};
    store_codes<D, V, false>(row, zeros, u, 0.f);
    return;
  }
  e4m3 ? store_codes<D, V, true>(row, f, u, inverse) : store_codes<D, V, false>(row, f, u, inverse);
}

constexpr int kAppendThreads = 256;

// One token of each sequence: a block of threads per token, whose rows are its query heads, its keys and its values.
// Latency is what counts: everything of a row is asked for at once, and only a block whose scale grows (a few times in a
// page) is read and written again, by the whole warp. One token with 16 query heads over 8 of 128: 3.0 us in a graph; 128
// of them in pages of 16: 3.7.
template <typename T, int D, int V, bool INTER>
__global__ void __launch_bounds__(kAppendThreads) append_token_kernel(const AppendArgs a) {
  using S = RowShape<D, V>;
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = lane_id(), r = lane / S::kLanes, j0 = lane % S::kLanes;
  const int64_t token = blockIdx.x;
  const int position = a.starts[token];
  const bool there = position >= 0;
  const int number = position >> a.page_shift, slot = position & (a.page - 1);
  int page = -1;
  if (there && number < a.max_pages) page = a.table[token * a.ld_table + number];
  if (page >= a.pages) page = -1;
  UnitAt u[S::kUnits];
  float cos_[S::kUnits][V], sin_[S::kUnits][V];
#pragma unroll
  for (int k = 0; k < S::kUnits; ++k) {
    u[k] = unit_at<V, INTER>(j0 + k * S::kLanes, a.n_freq);
    constexpr int kPer = V / S::kRows;
    float2 mine[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = (j0 + k * S::kLanes) * V + r * kPer + i;
      mine[i] = p < a.n_freq ? turn_of(turns_of(a.inv_freq[p]) * static_cast<uint64_t>(static_cast<int64_t>(position)), a.factor) : make_float2(1.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int src = (i / kPer) * S::kLanes + j0;
      cos_[k][i] = __shfl_sync(kAll, mine[i % kPer].x, src);
      sin_[k][i] = __shfl_sync(kAll, mine[i % kPer].y, src);
    }
  }
  const int hq = a.q ? a.hq : 0, rows = hq + 2 * a.hkv;
  for (int r0 = warp_id() * S::kRows; r0 < rows; r0 += kAppendThreads / 32 * S::kRows) {
    const int row = r0 + r, kind = row < hq ? 0 : row < hq + a.hkv ? 1 : 2;  // query, key, value
    const int h = kind == 0 ? row : kind == 1 ? row - hq : row - hq - a.hkv;
    const bool mine = row < rows && there;
    const T* src = kind == 0   ? static_cast<const T*>(a.q) + token * a.q_st + h * a.q_sh
                   : kind == 1 ? static_cast<const T*>(a.k) + token * a.k_st + h * a.k_sh
                               : static_cast<const T*>(a.v) + token * a.v_st + h * a.v_sh;
    const bool cached = mine && kind > 0 && page >= 0;
    float* scale = nullptr;
    uint8_t* block = nullptr;
    uint32_t old_bits = 0;
    if (cached) {
      scale = (kind == 1 ? a.ks + page * a.ks_sp : a.vs + page * a.vs_sp) + h;
      block = (kind == 1 ? a.kc + page * a.kc_sp : a.vc + page * a.vc_sp) + static_cast<int64_t>(h) * a.page * D;
      old_bits = __float_as_uint(*scale);
    }
    float f[S::kUnits][2 * V];
    row_floats<T, D, V>(mine ? load_row<T, D, V>(src, u) : RawRow<T, D, V>{}, f);
    if (a.q_norm || a.k_norm) {  // every lane takes part in the sum
      const float inverse = row_inverse<D, V>(f, a.eps);
      const void* norm = kind == 0 ? a.q_norm : a.k_norm;
      if (mine && kind != 2 && norm)
        norm_row<D, V>(f, u, norm, kind == 0 ? a.q_norm_dtype : a.k_norm_dtype, kind == 0 ? h * a.q_norm_sh : h * a.k_norm_sh, inverse);
    }
    if (kind != 2) {
#pragma unroll
      for (int k = 0; k < S::kUnits; ++k) turn_unit<V, INTER>(f[k], cos_[k], sin_[k], u[k].turning);
    }
    if (kind == 0 && row < rows) {
      T* dst = static_cast<T*>(a.q_out) + (token * a.hq + h) * D;
#pragma unroll
      for (int k = 0; k < S::kUnits; ++k) {
        store_pack<T, V>(dst + u[k].lo, mine ? from_floats<T, V>(f[k]) : Pack<T, V>{});
        store_pack<T, V>(dst + u[k].hi, mine ? from_floats<T, V>(f[k] + V) : Pack<T, V>{});
      }
    }
    const uint32_t top = row_top<D, V>(f);
    BlockChange c{0.f, 0.f, 1.f};
    if (cached) {
      c = change_block(top, slot > 0, old_bits, a.e4m3);
      store_codes<D, V>(block + slot * D, f, u, c.inverse, a.e4m3);
      if (j0 == 0) *scale = c.scale;
    }
    unsigned grows = __ballot_sync(kAll, c.older != 1.f && j0 == 0);
    while (grows) {
      const int who = __ffs(grows) - 1;
      grows &= grows - 1;
      uint8_t* p = reinterpret_cast<uint8_t*>(__shfl_sync(kAll, reinterpret_cast<unsigned long long>(block), who));
      rescale_block(p, slot * D, __shfl_sync(kAll, c.older, who), a.e4m3, lane, 32);
    }
  }
}

// Page number `item` of those that the new tokens touch, sequence by sequence: found by every warp for itself, a sequence
// per lane.
struct PageItem {
  int seq, number;     // the sequence and its page's number
  int64_t first;       // the sequence's first new token
  int64_t start, end;  // its first and behind its last new position
};
__device__ __forceinline__ bool find_page(const AppendArgs& a, int64_t item, PageItem* found) {
  constexpr unsigned kAll = 0xffffffffu;
  for (int base = 0; base < a.n_seqs; base += 32) {
    const int seq = base + lane_id();
    int64_t first = 0, start = -1, end = -1;
    int count = 0;
    if (seq < a.n_seqs) {
      first = min(max(static_cast<int64_t>(a.cu[seq]), int64_t{0}), a.tokens);
      const int64_t last = min(max(static_cast<int64_t>(a.cu[seq + 1]), first), a.tokens);
      start = a.starts[seq];
      end = min(start + (last - first), static_cast<int64_t>(a.max_pages) << a.page_shift);
      if (start >= 0 && end > start) count = static_cast<int>(((end - 1) >> a.page_shift) - (start >> a.page_shift)) + 1;
    }
    int64_t upto = count;  // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(kAll, upto, o);
      if (lane_id() >= o) upto += y;
    }
    const unsigned here = __ballot_sync(kAll, item < upto);
    if (here) {
      const int who = __ffs(here) - 1;
      const int64_t mine = (start >> a.page_shift) + item - (upto - count);
      *found = {base + who, static_cast<int>(__shfl_sync(kAll, mine, who)), __shfl_sync(kAll, first, who), __shfl_sync(kAll, start, who),
                __shfl_sync(kAll, end, who)};
      return true;
    }
    item -= __shfl_sync(kAll, upto, 31);
  }
  return false;
}

// The new tokens of packed sequences: a block of threads per page that they touch, K or V (blockIdx.z), and a.heads heads
// (blockIdx.y). A head's part of the page, MOST tokens for each of a block's rows of lanes (pages of fewer tokens than rows:
// several heads at once), stays in registers between the search for its largest value and its codes, while the next heads'
// part is on its way. The angles' cosines and sines, which are those of all heads, are worked out once, in shared memory.
// 12968 tokens of 16 prompts, 8 heads of 128 in bf16, pages of 64, e4m3: 31.3 us, 3.0 TB/s (int8 31.8; pages of 16: 33.1,
// of 128: 31.3). Nothing is full: 60 % of the issue slots are busy, and without norm and rotation it is still 26.5 us.
// There is one wave of blocks, whose start and end overlap with nothing, a barrier for each head, and those of keys have
// more to do than those of values (an SM has 47300 cycles on average, 61129 at most). Many sequences cost the search for a
// block's page: 1000 tokens of as many sequences beside a prompt of 1900 take 158 us, 100 of them 21, the prompt alone 8.8.
// Norm and rotation done twice, so that what was read stays in 16 bits: 48 us; one kernel for all page sizes, with rounds
// for 128 tokens in each: 47 (pages of 16: 160).
template <typename T, int D, int V, bool INTER, int MOST>
__global__ void __launch_bounds__(kAppendThreads, V == 8 ? (MOST <= 2 ? 3 : 2) : 1) append_packed_kernel(const AppendArgs a) {
  using S = RowShape<D, V>;
  constexpr int kAtOnce = kAppendThreads / 32 * S::kRows;       // rows of lanes
  constexpr int kSplit = D / (2 * V), kPitch = D / 2 + D / 16;  // of a token's turns; a lane's are kSplit apart
  extern __shared__ __align__(16) float2 turns[];
  __shared__ uint32_t tops[32];
  PageItem it;
  if (!find_page(a, blockIdx.x, &it)) return;
  const int page = a.table[it.seq * a.ld_table + it.number];
  if (page < 0 || page >= a.pages) return;
  if (threadIdx.x < 32) tops[threadIdx.x] = 0;
  const bool value = blockIdx.z != 0;
  const int64_t page_first = static_cast<int64_t>(it.number) << a.page_shift;
  const int lo = static_cast<int>(max(it.start - page_first, int64_t{0}));
  const int n = static_cast<int>(min(it.end - page_first, static_cast<int64_t>(a.page))) - lo;  // new tokens, in slots lo ..
  const int64_t token = it.first + (page_first + lo - it.start);
  const int lane = lane_id(), row = warp_id() * S::kRows + lane / S::kLanes, j0 = lane % S::kLanes;
  // the row's token and which of the heads at once it has, the same for a warp
  const int t0 = MOST > 1 ? row : row & (a.page - 1), heads = MOST > 1 ? 1 : max(kAtOnce >> a.page_shift, 1);
  const int mine = MOST > 1 ? 0 : row >> a.page_shift;
  const int n_freq = value ? 0 : a.n_freq;
  UnitAt u[S::kUnits];
#pragma unroll
  for (int k = 0; k < S::kUnits; ++k) u[k] = unit_at<V, INTER>(j0 + k * S::kLanes, n_freq);
  const int h0 = static_cast<int>(blockIdx.y) * a.heads, h1 = min(h0 + a.heads, a.hkv);
  const int64_t st = value ? a.v_st : a.k_st, sh = value ? a.v_sh : a.k_sh;
  const T* src = static_cast<const T*>(value ? a.v : a.k) + (token + t0) * st;
  float* scale = value ? a.vs + page * a.vs_sp : a.ks + page * a.ks_sp;
  uint8_t* block = value ? a.vc + page * a.vc_sp : a.kc + page * a.kc_sp;
  RawRow<T, D, V> later[MOST];
  uint32_t later_bits = 0;
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < MOST; ++i) later[i] = t0 + i * kAtOnce < n && h < h1 ? load_row<T, D, V>(src + h * sh + i * kAtOnce * st, u) : RawRow<T, D, V>{};
    if (lo > 0 && h < h1) later_bits = __float_as_uint(scale[h]);
  };
  load(h0 + mine);
  if (n_freq > 0) {  // n_freq threads to a token
    const int tokens = kAppendThreads / n_freq, p = static_cast<int>(threadIdx.x) % n_freq;
    int t = static_cast<int>(threadIdx.x) / n_freq;
    if (t < tokens) {
      const uint64_t each = turns_of(a.inv_freq[p]);
      uint64_t at = each * static_cast<uint64_t>(page_first + lo + t);
      for (; t < n; t += tokens, at += each * tokens) turns[t * kPitch + (p % V) * kSplit + p / V] = turn_of(at, a.factor);
    }
  }
  __syncthreads();
  for (int first = h0; first < h1; first += heads) {
    const int h = first + mine;
    float f[MOST][S::kUnits][2 * V];
#pragma unroll
    for (int i = 0; i < MOST; ++i) row_floats<T, D, V>(later[i], f[i]);
    const uint32_t old_bits = later_bits;
    load(h + heads);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int t = t0 + i * kAtOnce;
      if (!value) {
        if (a.k_norm) {
          const float inverse = row_inverse<D, V>(f[i], a.eps);
          if (h < h1) norm_row<D, V>(f[i], u, a.k_norm, a.k_norm_dtype, h * a.k_norm_sh, inverse);
        }
#pragma unroll
        for (int k = 0; k < S::kUnits; ++k) {
          if (t < n && u[k].turning > 0) {
            float c[V], s[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float2 y = turns[t * kPitch + e * kSplit + j0 + k * S::kLanes];  // of no use from u.turning on
              c[e] = y.x, s[e] = y.y;
            }
            turn_unit<V, INTER>(f[i][k], c, s, u[k].turning);
          }
        }
      }
      top = max(top, lane_top<D, V>(f[i]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && h < h1) atomicMax(&tops[h - h0], top);
    __syncthreads();
    if (h >= h1) continue;
    const BlockChange c = change_block(tops[h - h0], lo > 0, old_bits, a.e4m3);
    uint8_t* to = block + static_cast<int64_t>(h) * a.page * D;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int t = t0 + i * kAtOnce;
      if (t < n) store_codes<D, V>(to + (lo + t) * D, f[i], u, c.inverse, a.e4m3);
    }
    if (j0 == 0 && t0 == 0) scale[h] = c.scale;
    const int threads = kAppendThreads / heads;
    if (c.older != 1.f) rescale_block(to, lo * D, c.older, a.e4m3, static_cast<int>(threadIdx.x) - mine * threads, threads);
  }
}

template <typename T, int D, int V, bool INTER, int MOST>
static int launch_packed(const AppendArgs& a, dim3 grid, cudaStream_t s) {
  auto kern = append_packed_kernel<T, D, V, INTER, MOST>;
  constexpr int kTurn = (D / 2 + D / 16) * static_cast<int>(sizeof(float2));  // bytes of a token's turns
  static std::atomic<bool> allowed[64];
  int rc = allow_shared(allowed, kern, 128 * kTurn);
  if (rc != XDNA_OK) return rc;
  kern<<<grid, kAppendThreads, a.n_freq > 0 ? a.page * kTurn : 0, s>>>(a);
  return check_launch("append_packed_kernel");
}

template <typename T, int D, int V, bool INTER>
static int launch_append_as(AppendArgs a, int sms, cudaStream_t s) {
  if (a.cu == nullptr) {
    append_token_kernel<T, D, V, INTER><<<static_cast<unsigned>(a.tokens), kAppendThreads, 0, s>>>(a);
    return check_launch("append_token_kernel");
  }
  // pages that n tokens of N sequences can touch
  const int64_t items = std::min(a.tokens, a.tokens / a.page + 2 * static_cast<int64_t>(a.n_seqs));
  // heads of a block: few enough that the SMs have blocks (pages of 128 as above: 31.7 us, all 8 heads in a block 40.8)
  a.heads = std::min(a.hkv, 32);
  while (a.heads > 1 && items * 2 * ((a.hkv + a.heads - 1) / a.heads) < 3 * sms) a.heads = (a.heads + 1) / 2;
  constexpr int kAtOnce = kAppendThreads / 32 * RowShape<D, V>::kRows;
  // tokens of a page for each row of lanes; registers for four at pages of 64, that need two: 42.8 us instead of 31.3, of 32:
  // 64.8 instead of 32.4
  const int rounds = a.page / kAtOnce;
  const dim3 grid(static_cast<unsigned>(items), static_cast<unsigned>((a.hkv + a.heads - 1) / a.heads), 2);
  if constexpr (V == 1)
    return launch_packed<T, D, V, INTER, 16>(a, grid, s);
  else if (rounds >= 4)
    return launch_packed<T, D, V, INTER, 4>(a, grid, s);
  else
    return rounds >= 2 ? launch_packed<T, D, V, INTER, 2>(a, grid, s) : launch_packed<T, D, V, INTER, 1>(a, grid, s);
}

template <typename T>
static int launch_append(const AppendArgs& a, int64_t d, bool interleaved, int sms, cudaStream_t s) {
  if (interleaved) return d == 64 ? launch_append_as<T, 64, 8, true>(a, sms, s) : launch_append_as<T, 128, 8, true>(a, sms, s);
  if (a.n_freq % 8 == 0) return d == 64 ? launch_append_as<T, 64, 8, false>(a, sms, s) : launch_append_as<T, 128, 8, false>(a, sms, s);
  return d == 64 ? launch_append_as<T, 64, 1, false>(a, sms, s) : launch_append_as<T, 128, 1, false>(a, sms, s);
}

// ---------------------------------------------------------------------------- attention
struct PagedArgs {
  const void* q;
  int64_t q_sb, q_st, q_sh;
  const float *ks, *vs;
  int64_t ks_sp, vs_sp;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  float scale_log2;
  int* err;
  int B, T, hkv, group, page_shift, pages, max_pages;
  int splits;            // CLUSTER: CTAs of an item
  int shares;            // else: shares of the work
  int col_groups, cols;  // columns: query heads of a key head times T; of an item 8 * NT of them
  void* out;             // [B, T, hq, D]
  int4* shared;          // per item: the first and the last share that has a part of it, the first one's slot
  float* part_o;         // [2 * shares][8 * NT][D]
  float4* part_ml;       // [2 * shares][8 * NT]: m, l, m'
};

constexpr int kPaWarps = 4;
constexpr int kPaTile = 32;      // keys of a warp's step
constexpr int kPaSite = 70;      // of its waits, in the device error word
constexpr int kMostSplits = 8;   // CTAs of a cluster
// Units of 128 keys of one CTA up to which items go to clusters. 16 heads over 8 of 128, with clusters and without: one
// sequence of 764 keys 6.4 and 7.9 us, of 2000 8.1 and 8.6; 16 of up to 300: 7.6 and 9.1; 50 of up to 900: 17.7 and 19.3; a
// share longer than the average, one of 4000: 10.5 and 9.3. Shares of twelve units, whatever the average: 24 sequences of
// up to 3001 with 28 columns 23.3 and 20.4.
constexpr int kClusterUnits = 8;
constexpr float kPaSlack = 8.f;  // how far (log2) a score may pass the running maximum before that is raised
// The weights that meet V, rounded to f16, are between 2^12 and 2^15 for the largest (65504 is the most), so that they have
// all of f16's bits down to 2^-26 of it and are lost from 2^-37 on: many small weights beside a large one count in full.
// (From 1 on, with a slack of eight, they had all bits down to 2^-14 and were lost from 2^-25 on: a thousand keys of e^-15
// beside a peak without a value were off by 2.6 %. From 2^14 on the slack is one, and the sums are rescaled more often: 24
// sequences of up to 3001 with 28 columns 20.8 us instead of 20.4.)
constexpr float kPaWeight = 12.f, kPaWeightSlack = 3.f;
constexpr float kPaUnit = 2.44140625e-04f;  // 2^-kPaWeight

template <int D, int NT>
struct PaShape {
  static constexpr int kC = D / 64;                       // 16-byte pieces of a lane's key row
  static constexpr int kVBytes = D / 8;                   // bytes of a lane's value row
  static constexpr int kHalf = kPaTile * D;               // a tile's keys, and as much of values
  static constexpr int kCtas = NT == 1 ? 3 : 2;
  static constexpr int kStages = (NT == 1 ? 16384 : 24576) / (2 * kHalf);
  static constexpr int kRing = kPaWarps * kStages * 2 * kHalf, kSmem = kRing + 1024;  // aligned to 1024
  static_assert(kRing >= (kPaWarps + 1) * 8 * NT * (D + 4) * 4, "the warps' sums, and a cluster's part, lie where the ring was");
  // Tiles lie in shared memory row by row, swizzled by TMA: 16-byte piece p of row r is at p ^ turn(r). So that no load of
  // a warp meets itself in a bank, row g of a fragment is key row(g) of its block, and lane group g takes part(g) of a
  // value row.
  static __device__ __forceinline__ constexpr int turn(int r) { return D == 128 ? r & 7 : (r >> 1) & 3; }
  static __device__ __forceinline__ constexpr int row(int g) { return D == 128 ? (g & 1) << 2 | g >> 1 : g ^ g >> 1; }
  static __device__ __forceinline__ constexpr int part(int g) { return D == 128 ? (g & 1) << 2 | g >> 1 : (g & 1) | (g & 2) << 1 | (g & 4) >> 1; }
};

__device__ __forceinline__ int paged_len(const PagedArgs& a, int b) {
  return static_cast<int>(min(static_cast<int64_t>(max(a.lens[b], 0)), static_cast<int64_t>(a.max_pages) << a.page_shift));
}

// Where a place in the order of all units is: the sequence, its length and units, the units before it (of one head), the
// (key head, column group), the unit in it, and the item's unit behind the last one of a share that ends at `end`.
struct ItemAt {
  int b, len, units, hc, unit, stop;
  int64_t base;
  __device__ __forceinline__ void load(const PagedArgs& a, int keys) {
    len = paged_len(a, b);
    units = (len + keys - 1) / keys;
  }
  __device__ __forceinline__ void go(const PagedArgs& a, int keys, int per_b, int64_t at, int64_t end) {
    while (at >= (base + units) * per_b) {
      base += units;
      ++b;
      load(a, keys);
    }
    const int64_t in_b = at - base * per_b;
    hc = static_cast<int>(in_b >> 31 ? in_b / units : static_cast<uint32_t>(in_b) / static_cast<uint32_t>(units));
    unit = static_cast<int>(in_b - static_cast<int64_t>(hc) * units);
    stop = static_cast<int>(min(static_cast<int64_t>(units), unit + (end - at)));
  }
};

__device__ __forceinline__ float sum_of_groups(float x) {  // over the lanes with the same lane & 3
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

// log2 of a value block's scale: NaN below zero, -inf of zero, else to 2^-22 of itself (of powers of two below one to 2^-23,
// above whole, as measured), so that weights are off by 2^-20 at a scale of 2^-6 and by 2^-16 at 2^-126.
__device__ __forceinline__ float log2_scale(float scale) {
  float e;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(scale));
  return e;
}

// What a row's sums with V are to be multiplied with, after kPaUnit: 1 / the softmax's sum, brought from the weights'
// reference to the scores'.
__device__ __forceinline__ float inverse_of(float m, float sum, float mv) {
  const float up = (mv == -INFINITY ? 0.f : mv + kPaWeight) - (m == -INFINITY ? 0.f : m);
  return sum > 0.f || __isnanf(sum) ? fast_exp2(up) / sum : 0.f;
}

enum { PAGED_WARPS, PAGED_TOGETHER, PAGED_CLUSTER };  // how paged_kernel shares out its work

__device__ __forceinline__ float4 load_remote(uint32_t cluster_address) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(cluster_address)
               : "memory");
  return x;
}

// Attention of B sequences with T query tokens each (the last T of the sequence) over the paged cache. Few rows, so its
// time is the reading of the codes. The work is all tiles of 32 keys of all (sequence, key head, 8 NT columns), in that
// order, shared out evenly, whatever the lengths are; they are read on the device. A share begins and ends inside an item
// as it comes; parts of items go to the workspace and are joined by paged_join_kernel (joined by the last one to write a
// part, 0.5 to 6 us slower: its loads wait for one another behind the whole item).
// PAGED_TOGETHER: a share is of a CTA, whose warps take the tiles of a unit of 128 keys and add up at an item's end, so there
// are few parts. PAGED_WARPS: a share is of a warp, whose copies run on across the borders of items, so that many short
// sequences keep the memory as busy as a long one. PAGED_CLUSTER: items of few keys that the SMs hold all at once, where a
// second launch costs more than an even share gains: a cluster of up to eight CTAs has one item, as together, and joins its
// parts in their shared memory. Which one goes by the longest sequence that the table can hold and by the number of items
// (plan, below).
// 200 sequences of up to 300 keys, 16 heads over 8 of 128, e4m3: 27.4 us with warps' shares, 35.1 with CTAs'; 32 of 1175 to
// 4700: 40.2 us (4.9 TB/s) with CTAs' shares. One of 131071: 52.5 us, 5.1 TB/s; more keys of it are read at 6.4 TB/s (262144:
// 95.7, 524288: 180.1), so that 10.5 us are the start (lengths, pages and tiles wait for one another), the ends of the SMs'
// shares and the join.
// A tile's codes come by TMA into the warp's own ring in shared memory, and the products are mma.sync 16 x 8 x 16 with keys,
// then dimensions, as rows and the query rows as columns: S^T = K Q^T, O^T = V^T P^T. Of K, lane (g, t) reads bytes
// 64 c + 16 t .. + 15 of two keys: each word of them is, as two half pairs, A fragments when the queries' B fragments are
// read in the same order. Of V, D / 8 bytes of four keys: bytes of two keys, paired by byte permutes, are A fragments of
// output rows in the order of dimensions 2 i (row g of product i) and 2 i + 1 (row g + 8) of these D / 8. P^T is S^T's
// fragment, transposed by movmatrix.
// Codes are exact in f16, and so are queries of either type after a power of two per row has brought them to about one
// (bits below 2^-24 of the row's largest apart). The key block's scale goes into the scores. The value block's scale 2^e
// goes into the exponent of the weights that meet V, 2^(s + e - m'), with a reference m' of its own, 12 below the largest
// s + e, so that weights of 16 bits are full where they count, whatever the blocks' scales; the softmax's sum has
// 2^(s - m). Both are raised, and the sums rescaled, only when a score passes m by more than 8 or the reference by more
// than 15.
template <typename T, int D, bool E4M3, int NT, int MODE>
__global__ void __launch_bounds__(kPaWarps * 32, PaShape<D, NT>::kCtas)
    paged_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using S = PaShape<D, NT>;
  constexpr unsigned kAll = 0xffffffffu;
  constexpr bool TOGETHER = MODE != PAGED_WARPS, CLUSTER = MODE == PAGED_CLUSTER;
  constexpr int kCols = 8 * NT, kSteps = D / 16, kKeys = TOGETHER ? kPaTile * kPaWarps : kPaTile;  // of a unit
  extern __shared__ __align__(16) uint8_t paged_smem[];
  __shared__ __align__(8) uint64_t bars[kPaWarps][S::kStages];
  __shared__ float scales[kPaWarps][S::kStages][4];  // key and value scales of a tile's two blocks; -inf: no page
  __shared__ float sml[kPaWarps][kCols][3];
  __shared__ int abort_flag;
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, t = lane & 3;
  uint8_t* ring_all = paged_smem + (1024 - (smem_u32(paged_smem) & 1023)) % 1024;
  uint8_t* ring = ring_all + warp * (S::kStages * 2 * S::kHalf);
  float(*so)[kCols][D + 4] = reinterpret_cast<float(*)[kCols][D + 4]>(ring_all);
  if (lane < S::kStages) mbar_init(&bars[warp][lane], 1);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  fence_mbar_init();
  __syncthreads();
  const int key_row = S::row(g);
  const int page_mask = (1 << a.page_shift) - 1;
  const bool two_pages = a.page_shift == 4;  // a tile's two blocks of 16 keys lie in two pages

  // ---- this warp's share, and the sequence that it begins in. Shares of warps: neighbouring ones go to neighbouring CTAs,
  // so that few of them are spread over the SMs.
  const int per_b = a.hkv * a.col_groups, grid = static_cast<int>(gridDim.x);
  auto units_of = [&](int b) { return b < a.B ? (paged_len(a, b) + kKeys - 1) / kKeys : 0; };
  int64_t units = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < a.B && !CLUSTER; b0 += 32) units += __reduce_add_sync(kAll, units_of(b0 + lane));
  const Shares all(units * per_b, TOGETHER ? grid : grid * kPaWarps);
  const int share = TOGETHER ? static_cast<int>(blockIdx.x) : warp * grid + static_cast<int>(blockIdx.x);
  int64_t end = all.begin(share + 1);
  const int64_t start = CLUSTER ? 0 : all.begin(share);
  ItemAt it;  // what is worked on
  it.b = 0, it.base = 0;
  for (int64_t base = 0; !CLUSTER && start < end; it.b += 32) {
    const int mine = units_of(it.b + lane);
    int upto = mine;  // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(kAll, upto, o);
      if (lane >= o) upto += y;
    }
    const unsigned here = __ballot_sync(kAll, start < (base + upto) * per_b);
    if (here) {
      const int who = __ffs(here) - 1;
      it.b += who;
      it.base = base + __shfl_sync(kAll, upto - mine, who);
      break;
    }
    base += __shfl_sync(kAll, upto, 31);
  }
  // sequences without keys
  for (int b = warp * grid + static_cast<int>(blockIdx.x); b < a.B && !CLUSTER; b += grid * kPaWarps) {
    if (units_of(b) > 0) continue;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.T * a.hkv * a.group * D);
    for (int64_t i = lane; i < static_cast<int64_t>(a.T) * a.hkv * a.group * (D / 8); i += 32) dst[i] = make_uint4(0, 0, 0, 0);
    for (int i = lane; i < per_b; i += 32) a.shared[static_cast<int64_t>(b) * per_b + i] = make_int4(0, 0, 0, 0);
  }
  if constexpr (CLUSTER) {  // this CTA's part of its cluster's item
    const int item = static_cast<int>(blockIdx.x) / a.splits, rank = static_cast<int>(blockIdx.x) % a.splits;
    it.b = item / per_b, it.hc = item % per_b;
    it.load(a, kKeys);
    it.unit = static_cast<int>(static_cast<int64_t>(rank) * it.units / a.splits);
    it.stop = static_cast<int>(static_cast<int64_t>(rank + 1) * it.units / a.splits);
    end = it.stop - it.unit;
  } else if (start >= end) {
    return;
  }

  // ---- the copies
  const int first_key = TOGETHER ? warp * kPaTile : 0;  // of this warp's tile of a unit
  if constexpr (!CLUSTER) it.load(a, kKeys);
  ItemAt next = it;                              // next.unit is to be copied next
  next.unit = next.stop = 0;
  int left = static_cast<int>(end - start), more = left;  // units to be worked on, and to be copied (not TOGETHER)
  int looked = 0;                                // the number of next.unit among those whose pages the lanes have
  int pages[2] = {-1, -1};                       // of a tile's two blocks
  auto look = [&] {
    looked = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int unit = next.unit + lane, key = unit * kKeys + first_key + 16 * i;
      int p = -1;
      if ((i == 0 || two_pages) && unit < next.stop && key < next.len) p = a.table[next.b * a.ld_table + (key >> a.page_shift)];
      pages[i] = p < a.pages ? p : -1;
    }
  };
  auto fetch = [&](int st) {
    if (TOGETHER ? next.unit < next.stop : more > 0) {
      if (!TOGETHER && next.unit == next.stop) {
        next.go(a, kKeys, per_b, end - more, end);
        look();
      } else if (looked == 32) {
        look();
      }
      --more;
      const int key0 = next.unit * kKeys + first_key, h = next.hc / a.col_groups;
      const int p0 = __shfl_sync(kAll, pages[0], looked), p1 = two_pages ? __shfl_sync(kAll, pages[1], looked) : -1;
      if (lane == 0) {
        uint8_t* dst = ring + st * 2 * S::kHalf;
        uint64_t* bar = &bars[warp][st];
        const int block = two_pages ? S::kHalf / 2 : S::kHalf;
        const int row = (h << a.page_shift) + (key0 & page_mask);
        mbar_arrive_expect_tx(bar, ((p0 >= 0) + (p1 >= 0)) * 2 * block);
        if (p0 >= 0) {
          tma_load_3d(dst, &k_map, bar, 0, row, p0);
          tma_load_3d(dst + S::kHalf, &v_map, bar, 0, row, p0);
        }
        if (p1 >= 0) {
          tma_load_3d(dst + block, &k_map, bar, 0, row, p1);
          tma_load_3d(dst + S::kHalf + block, &v_map, bar, 0, row, p1);
        }
      }
      if (lane < (two_pages ? 4 : 2)) {
        const int page = lane < 2 ? p0 : p1;
        float* to = &scales[warp][st][lane];
        if (page >= 0)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)),
                       "l"(lane & 1 ? a.vs + page * a.vs_sp + h : a.ks + page * a.ks_sp + h)
                       : "memory");
        else
          *to = -INFINITY;
      }
      ++looked;
      ++next.unit;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  bool first = true;
  int st = 0;  // the stage of the next tile, and the parity of its barrier
  uint32_t parity = 0;
  for (bool once = true; CLUSTER ? once : left > 0; once = false) {
    if constexpr (!CLUSTER) it.go(a, kKeys, per_b, end - left, end);
    const int len = it.len, begin = it.unit;
    const int h = it.hc / a.col_groups, c0 = (it.hc % a.col_groups) * kCols;
    Pack<T, 4> raw[NT][kSteps];  // the queries, on their way while the pages are looked up
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int col = c0 + 8 * n + g, q_t = col / a.group;
      const T* qp = static_cast<const T*>(a.q) + it.b * a.q_sb + q_t * a.q_st + (h * a.group + col - q_t * a.group) * a.q_sh + 16 * t;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) raw[n][s] = col < a.cols ? load_pack<T, 4>(qp + 64 * (s / 4) + 4 * (s % 4)) : Pack<T, 4>{};
    }
    if constexpr (TOGETHER) {
      next = it;
      look();
    }
    if (TOGETHER || first) {
#pragma unroll
      for (int i = 0; i < S::kStages; ++i) fetch(st + i >= S::kStages ? st + i - S::kStages : st + i);
    }
    // the queries, brought to about one by a power of two per column, and what the products are to be multiplied with
    uint32_t qf[NT][kSteps][2];
    float by[NT][2];
    int limit[NT][2];  // keys that columns 2 t, 2 t + 1 see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t top = 0;
      float f[4];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        to_floats<T, 4>(raw[n][s], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(kAll, top, 1));
      top = max(top, __shfl_xor_sync(kAll, top, 2));
      const int e = top == 0 || top >= kNotFinite ? 0 : max(static_cast<int>(top >> 23) - 127, -126);
      const float inverse = e == 127 ? 5.877471754e-39f : power_of_two(-e);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        to_floats<T, 4>(raw[n][s], f);
        qf[n][s][0] = pack2<__half>(f[0] * inverse, f[1] * inverse);
        qf[n][s][1] = pack2<__half>(f[2] * inverse, f[3] * inverse);
      }
      const float back = fminf(power_of_two(e) * a.scale_log2, 3.4e38f);
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        by[n][e2] = __shfl_sync(kAll, back, (2 * t + e2) * 4);
        const int c = c0 + 8 * n + 2 * t + e2;
        limit[n][e2] = c < a.cols ? len - a.T + c / a.group + 1 : 0;
      }
    }
    const int seen_by_all = len - a.T + 1;

    float o[NT][kSteps][4], m[NT][2], mv[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      m[n][0] = m[n][1] = mv[n][0] = mv[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    for (; it.unit < it.stop; ++it.unit) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();  // the scales
      if (!mbar_wait_warp(&bars[warp][st], parity, &abort_flag, a.err, kPaSite)) break;
      const uint8_t* mine = ring + st * 2 * S::kHalf;
      const int key0 = it.unit * kKeys + first_key;
      const float4 sc = *reinterpret_cast<const float4*>(scales[warp][st]);  // K, V of block 0, K, V of block 1
      const float ks[2] = {sc.x, two_pages ? sc.z : sc.x};
      const float ev[2] = {log2_scale(sc.y), log2_scale(two_pages ? sc.w : sc.y)};
      // scores: s[n][x][e] is key 16 x + key_row (+ 8 for e >= 2) of the tile, column 2 t + (e & 1)
      float s[NT][2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float odd[NT][4];  // two sums, so that the products are two chains
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][x][e] = odd[n][e] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < S::kC; ++c) {
          const uint8_t* src = mine + (16 * x + key_row) * D + ((4 * c + t) ^ S::turn(key_row)) * 16;
          const uint4 k0 = *reinterpret_cast<const uint4*>(src), k1 = *reinterpret_cast<const uint4*>(src + 8 * D);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t f[4];
            to_halves<E4M3>(w0[w], f[0], f[2]);
            to_halves<E4M3>(w1[w], f[1], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<false>(w & 1 ? odd[n] : s[n][x], f, qf[n][4 * c + w][0], qf[n][4 * c + w][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // s = (sum * the block's scale) * what the column is to be multiplied with, two columns at a time
          const float2 both = make_float2(ks[x], ks[x]), col = make_float2(by[n][0], by[n][1]);
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            float2 y = __fadd2_rn(make_float2(s[n][x][e], s[n][x][e + 1]), make_float2(odd[n][e], odd[n][e + 1]));
            y = __fmul2_rn(__fmul2_rn(y, both), col);
            s[n][x][e] = y.x, s[n][x][e + 1] = y.y;
          }
        }
      }
      const bool whole = key0 + kPaTile <= seen_by_all && ks[0] != -INFINITY && ks[1] != -INFINITY;
      if (!whole) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (ks[x] == -INFINITY || key0 + 16 * x + key_row + 8 * (e >> 1) >= limit[n][e & 1]) s[n][x][e] = -INFINITY;
          }
        }
      }
      bool raise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a0 = fmaxf(s[n][0][e], s[n][0][2 + e]), a1 = fmaxf(s[n][1][e], s[n][1][2 + e]);
          raise |= fmaxf(a0, a1) > m[n][e] + kPaSlack || fmaxf(a0 + ev[0], a1 + ev[1]) > mv[n][e] + (kPaWeight + kPaWeightSlack);
        }
      }
      if (__any_sync(kAll, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float a0 = fmaxf(s[n][0][e], s[n][0][2 + e]), a1 = fmaxf(s[n][1][e], s[n][1][2 + e]);
            float top = fmaxf(a0, a1), tv = fmaxf(a0 + ev[0], a1 + ev[1]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(kAll, top, x));
              tv = fmaxf(tv, __shfl_xor_sync(kAll, tv, x));
            }
            const float mn = fmaxf(m[n][e], top), vn = fmaxf(mv[n][e], tv - kPaWeight);
            l[n][e] *= mn == -INFINITY ? 1.f : fast_exp2(m[n][e] - mn);
            f[e] = vn == -INFINITY ? 1.f : fast_exp2(mv[n][e] - vn);
            m[n][e] = mn;
            mv[n][e] = vn;
          }
#pragma unroll
          for (int j = 0; j < kSteps; ++j) o[n][j][0] *= f[0], o[n][j][1] *= f[1], o[n][j][2] *= f[0], o[n][j][3] *= f[1];
        }
      }
      uint32_t p[NT][2][2];  // B fragments of the weights
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 less = make_float2(m[n][0] == -INFINITY ? 0.f : -m[n][0], m[n][1] == -INFINITY ? 0.f : -m[n][1]);
        const float2 less_v = make_float2(mv[n][0] == -INFINITY ? 0.f : -mv[n][0], mv[n][1] == -INFINITY ? 0.f : -mv[n][1]);
        float2 sum = make_float2(l[n][0], l[n][1]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 less_x = __fadd2_rn(less_v, make_float2(ev[x], ev[x]));
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 y = make_float2(s[n][x][2 * r], s[n][x][2 * r + 1]);
            const float2 z = __fadd2_rn(y, less);
            sum = __fadd2_rn(sum, make_float2(fast_exp2(z.x), fast_exp2(z.y)));
            float2 w = __fadd2_rn(y, less_x);
            w = make_float2(fast_exp2(w.x), fast_exp2(w.y));
            if (!whole) {  // masked weights are zero whatever the block's scale
              if (y.x == -INFINITY) w.x = 0.f;
              if (y.y == -INFINITY) w.y = 0.f;
            }
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[n][x][r]) : "r"(pack2<__half>(w.x, w.y)));
          }
        }
        l[n][0] = sum.x, l[n][1] = sum.y;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t v[4][S::kVBytes / 4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // key of fragment place 2 t (+ 1), (+ 8)
          const int row = S::row(2 * t + (r & 1)), at = S::part(g) * S::kVBytes;
          const uint8_t* src = mine + S::kHalf + (16 * x + row + 8 * (r >> 1)) * D + ((at / 16) ^ S::turn(row)) * 16 + at % 16;
          if constexpr (S::kVBytes == 16) {
            const uint4 u = *reinterpret_cast<const uint4*>(src);
            v[r][0] = u.x, v[r][1] = u.y, v[r][2] = u.z, v[r][3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            v[r][0] = u.x, v[r][1] = u.y;
          }
          if (!whole) {  // what lies behind the last key and in the place of a page that is none: any byte, also a NaN
            if (ks[x] == -INFINITY || key0 + 16 * x + row + 8 * (r >> 1) >= len) {
#pragma unroll
              for (int w = 0; w < S::kVBytes / 4; ++w) v[r][w] = 0;
            }
          }
        }
#pragma unroll
        for (int w = 0; w < S::kVBytes / 4; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int sel = half ? 0x7362 : 0x5140;
            uint32_t f[4];
            to_halves<E4M3>(__byte_perm(v[0][w], v[1][w], sel), f[0], f[1]);
            to_halves<E4M3>(__byte_perm(v[2][w], v[3][w], sel), f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<false>(o[n][2 * w + half], f, p[n][x][0], p[n][x][1]);
          }
        }
      }
      __syncwarp();
      fetch(st);  // into the stage just read
      if (++st == S::kStages) st = 0, parity ^= 1;
    }
    if (TOGETHER ? __syncthreads_or(it.unit < it.stop) : it.unit < it.stop) {  // a wait ran out: the copies still under way, and out
      volatile int never = 0;
      for (int n = TOGETHER ? next.unit - it.unit : left - (it.unit - begin) - more; n > 0; --n) {
        mbar_wait(&bars[warp][st], parity, &never, a.err, kPaSite);
        if (++st == S::kStages) st = 0, parity ^= 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if constexpr (!CLUSTER) return;  // a cluster's CTAs still meet; what they write then is of no use
    }
    // ---- the item's sums, or a part of them; a share has at most two parts of items
    const int64_t slot = 2 * static_cast<int64_t>(share) + (first ? 0 : 1), item = static_cast<int64_t>(it.b) * per_b + it.hc;
    const bool whole_item = !CLUSTER && begin == 0 && it.stop == it.units;
    if (!CLUSTER && begin == 0 && lane == 0 && (warp == 0 || !TOGETHER))
      a.shared[item] = make_int4(share, whole_item ? share : all.owner(end - left + it.units - 1), static_cast<int>(slot), 0);
    auto row_of = [&](int col) {
      return static_cast<T*>(a.out) + ((static_cast<int64_t>(it.b) * a.T + col / a.group) * (a.hkv * a.group) + h * a.group + col % a.group) * D;
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float sum = sum_of_groups(l[n][e]);
        const int c = 8 * n + 2 * t + e, col = c0 + c, d = S::kVBytes * S::part(g);
        if (col >= a.cols) continue;
        float x[2 * kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) x[2 * j] = o[n][j][e], x[2 * j + 1] = o[n][j][2 + e];
        if constexpr (TOGETHER) {
          if (g == 0) sml[warp][c][0] = m[n][e], sml[warp][c][1] = sum, sml[warp][c][2] = mv[n][e];
          store_pack<float, 2 * kSteps>(&so[warp][c][d], from_floats<float, 2 * kSteps>(x));
        } else if (whole_item) {
          const float inv = inverse_of(m[n][e], sum, mv[n][e]);
#pragma unroll
          for (int j = 0; j < 2 * kSteps; ++j) x[j] = fit<T>(x[j] * kPaUnit * inv);
          store_pack<T, 2 * kSteps>(row_of(col) + d, from_floats<T, 2 * kSteps>(x));
        } else {
          store_pack<float, 2 * kSteps>(a.part_o + (slot * kCols + c) * D + d, from_floats<float, 2 * kSteps>(x));
          if (g == 0) a.part_ml[slot * kCols + c] = make_float4(m[n][e], sum, mv[n][e], 0.f);
        }
      }
    }
    if constexpr (TOGETHER) {
      float* mine_o = &so[kPaWarps][0][0];  // CLUSTER: this CTA's part
      float4* mine_ml = reinterpret_cast<float4*>(mine_o + kCols * D);
      __syncthreads();
      for (int i = threadIdx.x; i < min(kCols, a.cols - c0) * (D / 4); i += kPaWarps * 32) {
        const int c = i / (D / 4), d = (i % (D / 4)) * 4;
        float mm = -INFINITY, mmv = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < kPaWarps; ++w) mm = fmaxf(mm, sml[w][c][0]), mmv = fmaxf(mmv, sml[w][c][2]);
        const float m0 = mm == -INFINITY ? 0.f : mm, v0 = mmv == -INFINITY ? 0.f : mmv;
        float acc[4] = {};
#pragma unroll
        for (int w = 0; w < kPaWarps; ++w) {
          ll = fmaf(fast_exp2(sml[w][c][0] - m0), sml[w][c][1], ll);
          const float f = fast_exp2(sml[w][c][2] - v0);
          const float4 x = *reinterpret_cast<const float4*>(&so[w][c][d]);
          acc[0] = fmaf(f, x.x, acc[0]), acc[1] = fmaf(f, x.y, acc[1]), acc[2] = fmaf(f, x.z, acc[2]), acc[3] = fmaf(f, x.w, acc[3]);
        }
        if constexpr (CLUSTER) {
          store_pack<float, 4>(&mine_o[c * D + d], from_floats<float, 4>(acc));
          if (d == 0) mine_ml[c] = make_float4(mm, ll, mmv, 0.f);
        } else if (whole_item) {
          const float inv = inverse_of(mm, ll, mmv);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = fit<T>(acc[j] * kPaUnit * inv);
          store_pack<T, 4>(row_of(c0 + c) + d, from_floats<T, 4>(acc));
        } else {
          store_pack<float, 4>(a.part_o + (slot * kCols + c) * D + d, from_floats<float, 4>(acc));
          if (d == 0) a.part_ml[slot * kCols + c] = make_float4(mm, ll, mmv, 0.f);
        }
      }
      if constexpr (CLUSTER) {
        __syncwarp();
        cluster_sync();
        const int rank = static_cast<int>(blockIdx.x) % a.splits;
        for (int i = rank * kPaWarps * 32 + static_cast<int>(threadIdx.x); i < min(kCols, a.cols - c0) * (D / 4); i += a.splits * kPaWarps * 32) {
          const int c = i / (D / 4), d = (i % (D / 4)) * 4;
          float4 ml[kMostSplits], x[kMostSplits];
          float mm = -INFINITY, mmv = -INFINITY, ll = 0.f;
#pragma unroll
          for (int r = 0; r < kMostSplits; ++r) {
            const int from = min(r, a.splits - 1);
            ml[r] = load_remote(cluster_addr(mine_ml + c, from));
            x[r] = load_remote(cluster_addr(mine_o + c * D + d, from));
            mm = fmaxf(mm, ml[r].x), mmv = fmaxf(mmv, ml[r].z);
          }
          const float m0 = mm == -INFINITY ? 0.f : mm, v0 = mmv == -INFINITY ? 0.f : mmv;
          float acc[4] = {};
#pragma unroll
          for (int r = 0; r < kMostSplits; ++r) {
            if (r >= a.splits) break;
            ll = fmaf(fast_exp2(ml[r].x - m0), ml[r].y, ll);
            const float f = fast_exp2(ml[r].z - v0);
            acc[0] = fmaf(f, x[r].x, acc[0]), acc[1] = fmaf(f, x[r].y, acc[1]), acc[2] = fmaf(f, x[r].z, acc[2]), acc[3] = fmaf(f, x[r].w, acc[3]);
          }
          const float inv = inverse_of(mm, ll, mmv);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = fit<T>(acc[j] * kPaUnit * inv);
          store_pack<T, 4>(row_of(c0 + c) + d, from_floats<T, 4>(acc));
        }
        __syncwarp();
        cluster_sync();  // the others have read this CTA's part
      } else {
        fence_async_smem();  // the sums, before TMA writes there again
        __syncthreads();
      }
    }
    first = false;
    left -= it.stop - begin;
  }
}

// A row of an item (sequence, key head, column group): nothing where one share had all of it, else the parts of the shares,
// joined in a fixed order. W = 1: a warp per row, for many rows; W = 4: a block per row, each warp with every fourth part. A
// warp asks for 4 or 8 parts at once.
template <typename T, int D, int NT, int W>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a, int64_t items) {
  constexpr int kCols = 8 * NT, kV = D / 32, kAhead = W == 1 ? 4 : 8;
  __shared__ float sums[W][D];
  __shared__ float sml[W][3];
  const int rows = min(kCols, a.cols), warp = W == 1 ? 0 : warp_id(), lane = lane_id();
  const int64_t number = W == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + warp_id() : blockIdx.x;
  const int64_t item = number / rows;
  const int per_b = a.hkv * a.col_groups, hc = static_cast<int>(item % per_b), c = static_cast<int>(number - item * rows);
  const int64_t b = item / per_b;
  const int h = hc / a.col_groups, col = (hc % a.col_groups) * kCols + c;
  if (item >= items || col >= a.cols) return;
  T* dst = static_cast<T*>(a.out) + ((b * a.T + col / a.group) * (a.hkv * a.group) + h * a.group + col % a.group) * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 it = a.shared[item];
  if (it.x == it.y) return;
  if (!parts_exist(it.x, it.y, it.z, a.shares)) {  // a wait ran out, which the device error word says
    float none[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) none[i] = NAN;
    if (warp == 0) store_pack<T, kV>(dst + lane * kV, from_floats<T, kV>(none));
    return;
  }
  float mm = -INFINITY, mmv = -INFINITY, ll = 0.f, acc[kV] = {};
  for (int x0 = it.x + warp; x0 <= it.y; x0 += W * kAhead) {
    float4 ml[kAhead];
    Pack<float, kV> y[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int x = x0 + W * n;
      ml[n] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);  // none
      y[n] = Pack<float, kV>{};
      if (x <= it.y) {
        const int64_t from = (x == it.x ? it.z : 2 * static_cast<int64_t>(x)) * kCols + c;  // all but the first begin with it
        ml[n] = a.part_ml[from];
        y[n] = load_pack<float, kV>(a.part_o + from * D + lane * kV);
      }
    }
    float m1 = mm, v1 = mmv;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) m1 = fmaxf(m1, ml[n].x), v1 = fmaxf(v1, ml[n].z);
    const float m0 = m1 == -INFINITY ? 0.f : m1, v0 = v1 == -INFINITY ? 0.f : v1, f0 = fast_exp2(mmv - v0);
    ll *= fast_exp2(mm - m0);
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] *= f0;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      ll = fmaf(fast_exp2(ml[n].x - m0), ml[n].y, ll);
      const float f = fast_exp2(ml[n].z - v0);
#pragma unroll
      for (int i = 0; i < kV; ++i) acc[i] = fmaf(f, __uint_as_float(y[n].w[i]), acc[i]);
    }
    mm = m1, mmv = v1;
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < kV; ++i) sums[warp][lane * kV + i] = acc[i];
    if (lane == 0) sml[warp][0] = mm, sml[warp][1] = ll, sml[warp][2] = mmv;
    __syncthreads();
    if (warp > 0) return;
    const float wm = lane < W ? sml[lane % W][0] : -INFINITY, wl = lane < W ? sml[lane % W][1] : 0.f, wv = lane < W ? sml[lane % W][2] : -INFINITY;
    mm = wm, mmv = wv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o)), mmv = fmaxf(mmv, __shfl_xor_sync(0xffffffffu, mmv, o));
    ll = sum_of_lanes<32>(wl * fast_exp2(wm - (mm == -INFINITY ? 0.f : mm)));
    const float f = fast_exp2(wv - (mmv == -INFINITY ? 0.f : mmv));
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int i = 0; i < kV; ++i) acc[i] = fmaf(fw, sums[w][lane * kV + i], acc[i]);
    }
  }
  const float inv = inverse_of(mm, ll, mmv);
#pragma unroll
  for (int i = 0; i < kV; ++i) acc[i] = fit<T>(acc[i] * kPaUnit * inv);
  store_pack<T, kV>(dst + lane * kV, from_floats<T, kV>(acc));
}

// How a call's work is shared out, its CTAs, and where its workspace's parts lie.
struct PagedPlan {
  int nt, col_groups, mode, splits;
  int64_t resident, items, ctas, ml_at, o_at, bytes;
  void shape(int tiles, int64_t B, int64_t hkv, int64_t cols, int sms) {
    nt = tiles;  // of eight columns that a warp takes at once
    col_groups = static_cast<int>((cols + 8 * nt - 1) / (8 * nt));
    items = B * hkv * col_groups;
    resident = static_cast<int64_t>(sms) * (nt == 1 ? 3 : 2);
  }
  PagedPlan(int64_t B, int64_t T, int64_t hq, int64_t hkv, int64_t d, int64_t most_keys, int sms) {
    const int64_t cols = hq / hkv * T, units = (most_keys + kPaTile * kPaWarps - 1) / (kPaTile * kPaWarps);
    ml_at = o_at = bytes = 0;
    mode = PAGED_CLUSTER;
    // as many CTAs per item as the SMs hold, where a share of the longest item is about one of all work. Clusters leave some
    // of the places empty, so only seven eighths of them count: 72 items of up to 900 keys in clusters of five 8.9 us, in ones
    // of six (432 of 444 places) 11.7; 144 of up to 500, twos and threes, 7.6 and 11.0; 96 in 296 places, twos and threes,
    // 12.7 and 15.6. Clusters of two would always fit: 200 of up to 500 have one CTA each, 12.0 us, 8.6 with two.
    auto clusters = [&](int tiles) {
      shape(tiles, B, hkv, cols, sms);
      splits = static_cast<int>(std::max<int64_t>(1, std::min({static_cast<int64_t>(kMostSplits), units, resident * 7 / 8 / items})));
      ctas = items * splits;
      const int64_t longest = (units + splits - 1) / splits;
      return items <= resident && longest <= kClusterUnits && longest <= (items * units + resident - 1) / resident + 1;
    };
    if (clusters(1)) return;
    // two tiles of columns from nine columns on, which read the cache half as often (24 sequences of up to 12000 keys with 28
    // columns: 44.3 us, with one tile 51.6; in a cluster, of up to 1000, 12.7 and 11.5). Heads of 64 have registers for
    // four, but up to 3001 keys took 21.2 us with four and 20.3 with two (of up to 12000: 38.5 and 43.7)
    if (cols > 8 && clusters(2)) return;
    // 200 sequences (the shorter ones from a quarter of the longest on) of up to 500, 1024 and 1600 keys, 8 key heads of 128:
    // warps' shares 35.5, 56.1 and 77.3 us, CTAs' 42.5, 56.7 and 76.3; 100 of up to 4700: 110.2 and 105.6
    mode = most_keys > 1024 || items < resident ? PAGED_TOGETHER : PAGED_WARPS;
    splits = 0;
    ctas = std::max<int64_t>(1, std::min(resident, items * ((most_keys + kPaTile - 1) / kPaTile)));
    ml_at = (items * 16 + 255) / 256 * 256;
    o_at = ml_at + 2 * ctas * kPaWarps * 8 * nt * 16;
    bytes = o_at + 2 * ctas * kPaWarps * 8 * nt * d * 4;
  }
};

struct PagedMaps {
  CUtensorMap k, v;
};
// Codes [pages][Hkv * page][d] as TMA reads them, 32 keys or a page at a time.
static int codes_map(CUtensorMap* m, const void* codes, int64_t sp, int64_t pages, int64_t hkv, int64_t page, int64_t d) {
  const uint64_t dims[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(hkv * page), static_cast<uint64_t>(pages)};
  const uint64_t strides[2] = {static_cast<uint64_t>(d), static_cast<uint64_t>(pages > 1 ? sp : hkv * page * d)};
  const uint32_t box[3] = {static_cast<uint32_t>(d), static_cast<uint32_t>(std::min<int64_t>(page, kPaTile)), 1};
  return encode_tma(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, codes, dims, strides, box, "paged_attention codes",
                    d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <typename T, int D, bool E4M3, int NT, int MODE>
static int launch_paged_as(const PagedArgs& a, const PagedMaps& maps, int ctas, cudaStream_t s) {
  using S = PaShape<D, NT>;
  auto kern = paged_kernel<T, D, E4M3, NT, MODE>;
  static std::atomic<bool> allowed[64];
  int rc = allow_shared(allowed, kern, S::kSmem);
  if (rc != XDNA_OK) return rc;
  if constexpr (MODE == PAGED_CLUSTER) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kPaWarps * 32);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    XDNA_CUDA(cudaLaunchKernelEx(&cfg, kern, a, maps.k, maps.v));
    return check_launch("paged_kernel");
  } else {
    kern<<<static_cast<unsigned>(ctas), kPaWarps * 32, S::kSmem, s>>>(a, maps.k, maps.v);
    if ((rc = check_launch("paged_kernel")) != XDNA_OK) return rc;
    const int64_t items = static_cast<int64_t>(a.B) * a.hkv * a.col_groups;
    const int64_t rows = items * std::min(8 * NT, a.cols);
    // 16 rows of many parts (one sequence of 131071): 52.7 us with a block per row, 62.7 with a warp; 2048 rows of two or three
    // (16 sequences of 680 to 2700 with 4 tokens): 22.0 and 20.3
    return rows < 4 * 148
               ? launch_early("paged_join_kernel", paged_join_kernel<T, D, NT, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, s, a, items)
               : launch_early("paged_join_kernel", paged_join_kernel<T, D, NT, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, s, a, items);
  }
}

template <typename T, int D, bool E4M3, int NT>
static int launch_paged_as(const PagedArgs& a, const PagedMaps& m, const PagedPlan& plan, cudaStream_t s) {
  const int ctas = static_cast<int>(plan.ctas);
  if (plan.mode == PAGED_CLUSTER) return launch_paged_as<T, D, E4M3, NT, PAGED_CLUSTER>(a, m, ctas, s);
  return plan.mode == PAGED_TOGETHER ? launch_paged_as<T, D, E4M3, NT, PAGED_TOGETHER>(a, m, ctas, s)
                                     : launch_paged_as<T, D, E4M3, NT, PAGED_WARPS>(a, m, ctas, s);
}

template <typename T, int D>
static int launch_paged(const PagedArgs& a, const PagedMaps& m, bool e4m3, const PagedPlan& plan, cudaStream_t s) {
  if (plan.nt == 1) return e4m3 ? launch_paged_as<T, D, true, 1>(a, m, plan, s) : launch_paged_as<T, D, false, 1>(a, m, plan, s);
  return e4m3 ? launch_paged_as<T, D, true, 2>(a, m, plan, s) : launch_paged_as<T, D, false, 2>(a, m, plan, s);
}

// ---------------------------------------------------------------------------- host
static int check_cache(const char* what, int64_t pages, int64_t hkv, int64_t page, int64_t d, int format, int64_t max_pages) {
  if (d != 64 && d != 128) return fail(XDNA_ERR_UNSUPPORTED, "%s: head dimension %lld (64 or 128)", what, (long long)d);
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(XDNA_ERR_UNSUPPORTED, "%s: pages of %lld tokens (16, 32, 64 or 128)", what, (long long)page);
  XDNA_CHECK_ARG(format == XDNA_I8 || format == XDNA_E4M3, "%s: int8 or e4m3 codes", what);
  XDNA_CHECK_ARG(pages >= 0 && pages < (1ll << 31) && hkv >= 1 && hkv < (1 << 16) && max_pages >= 0 && max_pages < (1ll << 30) / page,
                 "%s: bad sizes", what);
  return XDNA_OK;
}
static bool cache_ok(const void* codes, int64_t sp, const void* scales, int64_t ssp, int64_t pages) {
  return ((codes && scales) || pages == 0) && aligned16(codes) && sp >= 0 && sp % 16 == 0 && ssp >= 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0;
}
static bool rows_ok(const void* p, int64_t st, int64_t sh) { return p && aligned16(p) && st > 0 && sh > 0 && st % 8 == 0 && sh % 8 == 0; }
static int shift_of(int64_t page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_cache_append(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, int dtype,
                      int64_t tokens, int64_t hkv, int64_t d, void* k_codes, int64_t kc_sp, void* v_codes, int64_t vc_sp,
                      int format, float* k_scales, int64_t ks_sp, float* v_scales, int64_t vs_sp, int64_t pages, int64_t page,
                      const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* starts,
                      const int32_t* cu_seqlens, int64_t n_seqs, const float* inv_freq, int64_t n_freq, float factor,
                      int interleaved, const void* k_norm, int k_norm_dtype, int64_t k_norm_sh, float eps, const void* q,
                      int64_t q_st, int64_t q_sh, int64_t hq, const void* q_norm, int q_norm_dtype, int64_t q_norm_sh,
                      void* q_out, void* stream) {
  int rc = check_cache("cache_append", pages, hkv, page, d, format, max_pages);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(dtype == XDNA_BF16 || dtype == XDNA_F16, "cache_append: bf16 or f16");
  XDNA_CHECK_ARG(tokens >= 0 && tokens < (1ll << 31) && n_seqs >= 0 && n_seqs < (1 << 24) && hq >= 0 && hq < (1 << 16) &&
                     (cu_seqlens || n_seqs == tokens),
                 "cache_append: bad sizes");
  XDNA_CHECK_ARG(n_freq >= 0 && 2 * n_freq <= d, "cache_append: %lld frequencies for heads of %lld", (long long)n_freq, (long long)d);
  XDNA_CHECK_ARG((!k_norm || (is_float_dtype(k_norm_dtype) && aligned16(k_norm) && k_norm_sh >= 0 && k_norm_sh % 8 == 0)) &&
                     (!q_norm || (is_float_dtype(q_norm_dtype) && aligned16(q_norm) && q_norm_sh >= 0 && q_norm_sh % 8 == 0)),
                 "cache_append: the norms' weights are f32, bf16 or f16, aligned");
  int sms = 0;
  if ((rc = check_device(&sms)) != XDNA_OK) return rc;
  if (tokens == 0) return XDNA_OK;
  XDNA_CHECK_ARG(rows_ok(k, k_st, k_sh) && rows_ok(v, v_st, v_sh) && (!q || (rows_ok(q, q_st, q_sh) && q_out && aligned16(q_out) && hq >= 1)) &&
                     cache_ok(k_codes, kc_sp, k_scales, ks_sp, pages) && cache_ok(v_codes, vc_sp, v_scales, vs_sp, pages) &&
                     (table || max_pages == 0) && (starts || n_seqs == 0) && (n_freq == 0 || inv_freq),
                 "cache_append: null pointer, unaligned rows or bad strides");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (q && cu_seqlens) {  // the queries of packed sequences
    RotaryArgs r{};
    r.x = q, r.x_st = q_st, r.x_sh = q_sh, r.out = q_out;
    r.starts = starts, r.cu = cu_seqlens, r.n_seqs = static_cast<int>(n_seqs);
    r.inv_freq = inv_freq, r.n_freq = static_cast<int>(n_freq), r.factor = factor;
    r.norm = q_norm, r.norm_dtype = q_norm_dtype, r.norm_sh = q_norm_sh, r.eps = eps;
    r.T = tokens, r.H = static_cast<int>(hq), r.D = static_cast<int>(d);
    if ((rc = launch_rotary(r, dtype, interleaved != 0, sms, s)) != XDNA_OK) return rc;
    q = nullptr;
  }
  if (n_seqs == 0) return XDNA_OK;
  AppendArgs a{};
  a.k = k, a.v = v, a.q = q;
  a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh, a.q_st = q_st, a.q_sh = q_sh;
  a.kc = static_cast<uint8_t*>(k_codes), a.vc = static_cast<uint8_t*>(v_codes), a.kc_sp = kc_sp, a.vc_sp = vc_sp;
  a.ks = k_scales, a.vs = v_scales, a.ks_sp = ks_sp, a.vs_sp = vs_sp;
  a.table = table, a.ld_table = ld_table, a.starts = starts, a.cu = cu_seqlens;
  a.inv_freq = inv_freq, a.n_freq = static_cast<int>(n_freq), a.factor = factor, a.eps = eps;
  a.k_norm = k_norm, a.k_norm_dtype = k_norm_dtype, a.k_norm_sh = k_norm_sh;
  a.q_norm = q_norm, a.q_norm_dtype = q_norm_dtype, a.q_norm_sh = q_norm_sh;
  a.q_out = q_out, a.tokens = tokens, a.n_seqs = static_cast<int>(n_seqs);
  a.hq = static_cast<int>(hq), a.hkv = static_cast<int>(hkv), a.page = static_cast<int>(page), a.page_shift = shift_of(page);
  a.pages = static_cast<int>(pages), a.max_pages = static_cast<int>(max_pages), a.e4m3 = format == XDNA_E4M3;
  return dtype == XDNA_BF16 ? launch_append<__nv_bfloat16>(a, d, interleaved != 0, sms, s)
                            : launch_append<__half>(a, d, interleaved != 0, sms, s);
}

size_t xdna_paged_attention_workspace(int64_t B, int64_t T, int64_t hq, int64_t hkv, int64_t d, int64_t most_keys) {
  int sms = 0;
  if (B < 1 || T < 1 || hkv < 1 || hq < hkv || d < 1 || most_keys < 0 || check_device(&sms) != XDNA_OK) return 0;
  return static_cast<size_t>(PagedPlan(B, T, hq, hkv, d, most_keys, sms).bytes);
}

int xdna_paged_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, int64_t B, int64_t T, int64_t hq,
                         int64_t hkv, int64_t d, const void* k_codes, int64_t kc_sp, const void* v_codes, int64_t vc_sp,
                         int format, const float* k_scales, int64_t ks_sp, const float* v_scales, int64_t vs_sp,
                         int64_t pages, int64_t page, const int32_t* table, int64_t ld_table, int64_t max_pages,
                         const int32_t* lens, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_cache("paged_attention", pages, hkv, page, d, format, max_pages);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(hq >= 1 && hq % hkv == 0 && hq / hkv <= 128, "paged_attention: %lld query heads over %lld key heads", (long long)hq, (long long)hkv);
  XDNA_CHECK_ARG(dtype == XDNA_BF16 || dtype == XDNA_F16, "paged_attention: bf16 or f16");
  XDNA_CHECK_ARG(scale > 0.f && scale * kLog2E < INFINITY, "paged_attention: the scale must be positive and at most 2.3e38");
  XDNA_CHECK_ARG(B >= 0 && T >= 0 && B < (1ll << 24) && T < (1 << 24) && B * T < (1ll << 31) / hq, "paged_attention: bad sizes");
  int sms = 0;
  if ((rc = check_device(&sms)) != XDNA_OK) return rc;
  if (B == 0 || T == 0) return XDNA_OK;
  XDNA_CHECK_ARG(q && aligned16(q) && q_sb > 0 && q_st > 0 && q_sh > 0 && q_sb % 8 == 0 && q_st % 8 == 0 && q_sh % 8 == 0 && out && aligned16(out) && lens &&
                     (table || max_pages == 0) && cache_ok(k_codes, kc_sp, k_scales, ks_sp, pages) && cache_ok(v_codes, vc_sp, v_scales, vs_sp, pages),
                 "paged_attention: null pointer, unaligned rows or bad strides");
  const PagedPlan plan(B, T, hq, hkv, d, max_pages * page, sms);
  XDNA_CHECK_ARG(plan.items < (1ll << 31) && plan.items * (max_pages * page / kPaTile + 1) / plan.ctas < (1ll << 31), "paged_attention: bad sizes");
  XDNA_CHECK_ARG(plan.bytes == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && workspace_bytes >= static_cast<size_t>(plan.bytes)),
                 "paged_attention: workspace too small or unaligned");
  PagedArgs a{};
  a.q = q, a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
  a.ks = k_scales, a.vs = v_scales, a.ks_sp = ks_sp, a.vs_sp = vs_sp, a.err = device_error_word();
  a.table = table, a.ld_table = ld_table, a.lens = lens, a.scale_log2 = scale * kLog2E;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.hkv = static_cast<int>(hkv), a.group = static_cast<int>(hq / hkv);
  a.page_shift = shift_of(page), a.pages = static_cast<int>(pages), a.max_pages = static_cast<int>(max_pages);
  a.splits = plan.splits, a.shares = static_cast<int>(plan.ctas) * (plan.mode == PAGED_WARPS ? kPaWarps : 1);
  a.col_groups = plan.col_groups, a.cols = static_cast<int>(a.group * T);
  a.out = out;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.shared = reinterpret_cast<int4*>(ws);
  a.part_ml = reinterpret_cast<float4*>(ws + plan.ml_at);
  a.part_o = reinterpret_cast<float*>(ws + plan.o_at);
  PagedMaps maps{};
  if (pages > 0) {  // without any, nothing is copied
    if ((rc = codes_map(&maps.k, k_codes, kc_sp, pages, hkv, page, d)) != XDNA_OK) return rc;
    if ((rc = codes_map(&maps.v, v_codes, vc_sp, pages, hkv, page, d)) != XDNA_OK) return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool e4m3 = format == XDNA_E4M3;
  if (dtype == XDNA_BF16)
    return d == 64 ? launch_paged<__nv_bfloat16, 64>(a, maps, e4m3, plan, s) : launch_paged<__nv_bfloat16, 128>(a, maps, e4m3, plan, s);
  return d == 64 ? launch_paged<__half, 64>(a, maps, e4m3, plan, s) : launch_paged<__half, 128>(a, maps, e4m3, plan, s);
}

}  // extern "C"
