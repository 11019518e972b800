// Attention of the generation path: causal attention over packed prompts of different lengths
// (xdna_packed_attention) and the decode attention of a batch that shares a prefix (xdna_prefix_attention).
//
//   packed   o[t, h] = sum_s p_s v[s, h / G],  p = softmax over the keys s <= t of t's own sequence of
//            scale * q[t, h] . k[s, h / G]                                  (G = Hq / Hkv query heads per key head)
//   prefix   o[b, h]: the same softmax over all P prefix keys and the first lens[b] keys of b's own cache
//
// A row with no keys at all, or with scores of -inf alone, is zero.
//
// Both read their long axis through one tcgen05 kernel (tile_attention_kernel). The G query heads that share a key
// head are packed into the rows of a tile: row r is token r / G, head r % G, so a tile of 128 rows holds 128 / G
// tokens (rounded down) and K and V are read once for all of them. An item is two such tiles (A and B) against a
// run of key blocks of 128; the kernel is persistent, one CTA per SM, and its roles run across item boundaries:
//   warp 0      TMA: both Q tiles per item, then K and V blocks in turn into one ring (K_j, V_j, K_j+1, ...). V is
//               taken as it lies in memory, keys by dimensions: the MN-major B operand of the second product.
//   warp 1      the MMAs, one thread:  S_A(0) S_B(0) | O_A += P_A(j) V(j), S_A(j+1) | O_B += P_B(j) V(j), S_B(j+1) | ...
//               While one tile's softmax works, the tensor core does the other's two products.
//   warps 4..7  softmax of tile A, warps 8..11 of tile B; thread = row. S is read from TMEM once, p = 2^(s - m) is
//               written as 16 bits over S's own columns and is the A operand of the second product straight from
//               TMEM, so P costs no shared-memory bandwidth (of which both products together need all there is when
//               P goes through it). The next S is issued after that product, in order, so it may overwrite P.
//               The running max m is raised, and O and l rescaled, only when a block exceeds it by more than 2^8.
//               m, l, O are f32; p is rounded to the operands' type because the tensor core takes one type for both
//               (its relative error, half an ulp, is that of the output's own rounding).
// Warps 2 and 3 only fill the first warpgroup: registers are moved between whole warpgroups.
// TMEM: S_A | S_B | O_A | O_B, 128 columns each. Shared memory: Q 2 x 128 x D, a ring of K and V blocks of 128 x D (4 of
// D = 128, 8 of 64), 32 KB through which outputs leave in whole lines.
// Measured (bf16, 16 heads over 8 of 128, one causal prompt, the causal half counted), in short replays of a graph with
// warm operands at 1.9 GHz: 4096 tokens 69 us, 990 TFLOP/s; 8191 tokens 233 us, 1180 TFLOP/s, 0.71 of a large matrix
// product's rate. The same call among others for a second, with other operands each time: 265 to 280 us, at the 1.7 GHz
// that the power limit leaves. A tile's own chain is about 2000 cycles of softmax and 1100 of its products per key block,
// with the other tile in antiphase: the tensor pipe and the unit of the exponentials are each busy half of the time, so
// neither is the limit by itself, and short prompts leave SMs idle at the end and between items (one Q buffer for both
// tiles). Tried on an earlier state of the kernel and left out: two threads per row (298 us against 289), an MMA thread
// per tile (their products interleave, so each chain gets longer: 336 against 298), the row's maximum overlapped with its
// loads (239 against 236).
//
// Keys that are masked for some rows of a tile but not for others carry p = 0; if their V holds an infinity or a NaN
// the product is NaN. So it is where a weight that a row does see is too small for 16 bits, and sums of values near the
// end of f32 overflow. A warp that has written non-finite results therefore looks at them again once it has done all its
// items (repair_rows), when no other role waits for it: the values of V that a row sees say which of its results
// stand, and the others are summed again over exactly its keys, in f32.
#include <algorithm>

#include "host_util.h"
#include "sm100.cuh"
#include "values.cuh"

namespace xdna {

// The larger magnitude of each of two 16-bit values, NaN where one is.
template <typename T>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __nv_bfloat162 r =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// 2^x of two values on the FMA pipe, to relieve the MUFU unit, whose rate (16 a clock and SM) is as tight here as the
// tensor core's: x = n + f with n whole and |f| <= 1/2, by adding and taking off 1.5 * 2^23; 2^f by the polynomial
// 1 + c1 f + ... of least largest relative error on [-1/2, 1/2] (a linear program over 4001 points): 1.0e-4 of degree
// 3, 2.8e-6 of degree 4, against roundings to 2^-9 (bf16) and 2^-12 (f16) that follow. x <= -126, and -inf with it,
// gives exactly 0 (2^-126 is taken off at the end, where it is otherwise lost), NaN gives NaN. x < 128.
template <int DEG>
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  constexpr float kC[4] = {DEG == 3 ? 0.6932829f : 0.6931242f, DEG == 3 ? 0.24221097f : 0.24024038f,
                           DEG == 3 ? 0.055008933f : 0.055906627f, 0.009585382f};
  auto both = [](float a) { return make_float2(a, a); };
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-126.f));
  const float2 t = __fadd2_rn(x, both(12582912.f)), n = __fadd2_rn(t, both(-12582912.f));
  const float2 f = __ffma2_rn(n, both(-1.f), x);
  float2 p = both(kC[DEG - 1]);
#pragma unroll
  for (int i = DEG - 2; i >= 0; --i) p = __ffma2_rn(p, f, both(kC[i]));
  p = __ffma2_rn(p, f, both(1.f));
  const float2 two_n = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                                   __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));
  return __ffma2_rn(p, two_n, both(-1.17549435e-38f));
}

// Of every four pairs of exponentials, those computed by exp2_fma. With heads of 64 the exponentials are twice as many
// per MMA: one of four 208 us, none 226, two 238 (one prompt of 8191, 16 heads of 64). With heads of 128 the issue
// slots it takes cost as much as it saves: 232, 229 and 249 us (16 heads over 8).
constexpr int ta_fma_of_4(int d) { return d == 64 ? 1 : 0; }

enum TileMode { PACKED = 0, PREFIX = 1 };

// What the plan of a packed call says (workspace): a header, then the tile pairs, those with the most key blocks
// first: {first token, first token of the sequence, end of the sequence, 0}.
struct PlanHeader {
  int n_pairs, first, end, pad;  // tokens [0, first) and [end, T) belong to no sequence
};

struct TileArgs {
  int hq, hkv, group, tok;  // tok: tokens per tile
  float scale_log2;
  int* err;
  void* out;
  // PACKED
  const PlanHeader* plan;  // null: at most 32 sequences, cu read here
  const int32_t* cu;
  int T, n_seqs;
  const void *q, *k, *v;  // repair_rows
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  // PREFIX
  int B, P, pairs, splits, blocks_per_split;
  float* part_o;   // [split][B * hq][D]
  float2* part_ml; // [split][B * hq]: m (log2 units), l
};

constexpr int kTaThreads = 384;  // three warpgroups: issue (TMA, MMA), softmax of tile A, of tile B
// Registers per thread after setmaxnreg: together what the launch gives, 384 x 168. 16 prompts of up to 1900 tokens, and
// one of 8191 with 16 heads of 64, with 56 for the issuing warps and 224 for the softmax: 125 and 248 us; 88 and 208: 111
// and 217; 120 and 192: 109 and 216; 152 and 176: 111 and 233.
constexpr int kTaRegsLaunch = 168, kTaRegsIssue = 120, kTaRegsSoftmax = 192;
static_assert(128 * kTaRegsIssue + 256 * kTaRegsSoftmax <= kTaThreads * kTaRegsLaunch, "more registers than the launch has");
constexpr int kTaBlock = 128;
constexpr float kTaRescale = 8.0f;
constexpr int kRepairRows = 8;  // rows that repair_rows sums together: the columns of a product

template <int D>
struct TaShape {
  static constexpr int kKB = D / 64;                    // 64-column k-blocks of a row
  static constexpr int kTile = 128 * D * 2;             // bytes of a Q tile, a K block or a V block
  static constexpr int kStages = D == 128 ? 4 : 8;      // K / V blocks in the ring (a fifth of 128 gained nothing)
  static constexpr int kStaging = 8 * 4096;             // a warp's 32 rows of 128 bytes on their way out
  static constexpr int kBars = 2 + 2 * kStages + 2 + 4 + 2 + 1;  // mbarriers
  static constexpr int kSmem = (2 + kStages) * kTile + kStaging + kBars * 8 + 16 /*TMEM address, abort flag, repair flags*/ + 1024 /*alignment*/;
  static_assert(kSmem <= 227 * 1024, "more shared memory than a CTA may have");
};

struct TileItem {
  int q_tok, kvh, kv_tok;  // first token of tile A, key head, first key (TMA coordinates)
  int nb[2];               // key blocks of tiles A and B
  int len, q_pos;          // PACKED: sequence length, tile A's first place in it
  int split;               // PREFIX
};

// N consecutive values of T as they are (N * 2 bytes, aligned to as many) and as floats.
template <int N>
struct Raw {
  uint32_t w[N / 2];
};
template <int N>
__device__ __forceinline__ Raw<N> load_raw(const void* p) {
  Raw<N> x;
  if constexpr (N == 8) {
    const uint4 u = *static_cast<const uint4*>(p);
    x.w[0] = u.x, x.w[1] = u.y, x.w[2] = u.z, x.w[3] = u.w;
  } else if constexpr (N == 4) {
    const uint2 u = *static_cast<const uint2*>(p);
    x.w[0] = u.x, x.w[1] = u.y;
  } else {
    x.w[0] = *static_cast<const uint32_t*>(p);
  }
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<N>& u, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint16_t h = static_cast<uint16_t>(u.w[i / 2] >> (16 * (i & 1)));
    x[i] = to_f32(*reinterpret_cast<const T*>(&h));
  }
}

// Looks again at a warp's rows of an item whose results, already in dst, hold an infinity or a NaN. Per lane: its row's
// place pos in the sequence (not falling from lane to lane), query q, result dst, and whether it has one (mine). k, v:
// the sequence's first key and value. A lane owns D / 32 dimensions. Per dimension, the sum of the non-finite values of V that the row sees is 0, an infinity or NaN:
//   NaN       so is the result, and it stands;
//   infinite  the result is that infinity where it stands, and NaN where a weight was lost to 16 bits or a masked value
//             came in: summed again. Where the row's scores are known to be sound, because another of its results is
//             finite, the keys between the first and the last non-finite value are enough;
//   0         the result is finite (a masked value came in, sums overflowed, or it was rounded past the type's end) or
//             a score is not: summed again over all keys.
// The sums over V's non-finite values run on from row to row, so a warp reads V once for all of its rows, and up to
// kRepairRows rows are summed again in one pass over K and V, 32 keys at a time, by running averages: with weights
// divided by the sum of the weights so far they stay within the range of V.
// One prompt of 8191 tokens (16 heads over 8 of 128, 235 us) with one NaN or infinity in V per head: 1.3 ms at its first
// token, 2.7 ms in the middle, 5.7 ms at the last one, whose tile's other rows are summed again over everything. The
// number of rows of V under way (kAhead) is what needs no spills here: with 16, and so with this called inside the loop
// over items, the kernel's own loops lost 1 to 8 % to the registers.
template <typename T, int D>
__device__ __noinline__ void repair_rows(bool mine, int pos, const T* q, T* dst, const T* k, int64_t k_st, const T* v,
                                         int64_t v_st, float sc) {
  constexpr bool kBf16 = !__is_same(T, __half);
  constexpr int kV = D / 32, kC = D / 32, kAhead = 8;  // rows of V under way
  constexpr unsigned kAll = 0xffffffffu;
  const int d0 = lane_id() * kV;
  auto of_lane = [](auto* p, int who) {
    return reinterpret_cast<decltype(p)>(__shfl_sync(kAll, reinterpret_cast<unsigned long long>(p), who));
  };
  const unsigned there = __ballot_sync(kAll, mine);
  unsigned again = 0;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    const T* row = of_lane(dst, r);
    bool odd = false;
    if (there >> r & 1) {
      float x[kV];
      unpack<T>(load_raw<kV>(row + d0), x);
#pragma unroll
      for (int i = 0; i < kV; ++i) odd |= !(fabsf(x[i]) < INFINITY);
    }
    if (__any_sync(kAll, odd)) again |= 1u << r;
  }
  float seen[kV];
  int scanned = 0, first = INT_MAX, last = -1;  // of the keys scanned, those with a non-finite value in these dimensions
#pragma unroll
  for (int i = 0; i < kV; ++i) seen[i] = 0.f;
  while (again) {
    // the next rows to sum again: their lanes and numbers of keys, and per lane the dimensions (bits)
    int count = 0, s0 = INT_MAX, s1 = 0, n_least = INT_MAX, lane_of[kRepairRows], n_of[kRepairRows];
    uint32_t redo[kRepairRows];
#pragma unroll
    for (int r = 0; r < kRepairRows; ++r) lane_of[r] = n_of[r] = 0, redo[r] = 0;
    while (again && count < kRepairRows) {
      const int who = __ffs(again) - 1;
      again &= again - 1;
      const int n = __shfl_sync(kAll, pos, who) + 1;
      const T* row_dst = of_lane(dst, who);
#pragma unroll 1
      for (; scanned < n; scanned = min(scanned + kAhead, n)) {
        Raw<kV> u[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) u[e] = load_raw<kV>(v + min(scanned + e, n - 1) * v_st + d0);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          float x[kV];
          unpack<T>(u[e], x);
          bool odd = false;
#pragma unroll
          for (int i = 0; i < kV; ++i) odd |= !(fabsf(x[i]) < INFINITY);
          if (odd && scanned + e < n) {
#pragma unroll
            for (int i = 0; i < kV; ++i)
              if (!(fabsf(x[i]) < INFINITY)) seen[i] += x[i];
            first = min(first, scanned + e);
            last = scanned + e;
          }
        }
      }
      float x[kV];
      unpack<T>(load_raw<kV>(row_dst + d0), x);
      uint32_t finite = 0, infinite = 0;
      bool sound = false;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        if (fabsf(x[i]) < INFINITY)
          sound = true;
        else if (seen[i] == 0.f)
          finite |= 1u << i;
        else if (!__isnanf(seen[i]) && x[i] != seen[i])
          infinite |= 1u << i;
      }
      if (!__any_sync(kAll, finite | infinite)) continue;
      sound = __any_sync(kAll, sound);
      if (__any_sync(kAll, finite) || !sound) {
        s0 = 0;
        s1 = max(s1, n);
      } else {
        s0 = min(s0, __reduce_min_sync(kAll, infinite ? first : INT_MAX));
        s1 = max(s1, __reduce_max_sync(kAll, infinite ? last : -1) + 1);
      }
      n_least = min(n_least, n);
#pragma unroll
      for (int r = 0; r < kRepairRows; ++r)
        if (r == count) lane_of[r] = who, n_of[r] = n, redo[r] = finite | infinite;
      ++count;
    }
    if (count == 0) return;
    // as in own_keys_kernel: the rows' queries are the columns of S^T = K Q^T, lane (g, t) holds the scores of keys g
    // and g + 8 against rows 2 t and 2 t + 1
    const int g = lane_id() >> 2, t = lane_id() & 3;
    Raw<8> qf[kC];
    int sees[2] = {0, 0};
    {
      int from = -1;
#pragma unroll
      for (int r = 0; r < kRepairRows; ++r) {
        if (r < count && r == g) from = lane_of[r];
        if (r == 2 * t) sees[0] = n_of[r];
        if (r == 2 * t + 1) sees[1] = n_of[r];
      }
      const T* row_q = of_lane(q, max(from, 0));
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        qf[c] = load_raw<8>(row_q + 32 * c + 8 * t);
        if (from < 0) qf[c].w[0] = qf[c].w[1] = qf[c].w[2] = qf[c].w[3] = 0;
      }
    }
    float o[kRepairRows][kV], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kRepairRows; ++r) {
#pragma unroll
      for (int i = 0; i < kV; ++i) o[r][i] = 0.f;
    }
    auto values = [&](Raw<kV>(&u)[8], int from) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = load_raw<kV>(v + min(from + e, s1 - 1) * v_st + d0);
    };
#pragma unroll 1
    for (; s0 < s1; s0 += 32) {
      Raw<kV> u[8];
      values(u, s0);
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        Raw<8> x[kC], y[kC];
        const T* kx = k + min(s0 + 16 * b + g, s1 - 1) * k_st + 8 * t;
        const T* ky = k + min(s0 + 16 * b + 8 + g, s1 - 1) * k_st + 8 * t;
#pragma unroll
        for (int c = 0; c < kC; ++c) x[c] = load_raw<8>(kx + 32 * c), y[c] = load_raw<8>(ky + 32 * c);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const uint32_t a0[4] = {x[c].w[0], y[c].w[0], x[c].w[1], y[c].w[1]};
          const uint32_t a1[4] = {x[c].w[2], y[c].w[2], x[c].w[3], y[c].w[3]};
          mma_16816<kBf16>(s[b], a0, qf[c].w[0], qf[c].w[1]);
          mma_16816<kBf16>(s[b], a1, qf[c].w[2], qf[c].w[3]);
        }
      }
      float keep[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows 2 t + h: scores of keys 16 b + 8 j + g, then weights
        float top = m[h], sum = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float& z = s[x >> 1][2 * (x & 1) + h];
          z = s0 + 8 * x + g < min(sees[h], s1) ? z * sc : -INFINITY;
          top = fmaxf(top, z);
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, x));
        const float base = top == -INFINITY ? 0.f : top;
        float p[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) sum += p[x] = exp2f(s[x >> 1][2 * (x & 1) + h] - base);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(kAll, sum, x);
        const bool any = l[h] > 0.f;
        const float before = l[h] * exp2f(m[h] - base);
        m[h] = top;
        l[h] = before + sum;
        const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
        keep[h] = before * inv;
        // a weight is zero for a score of -inf alone, which an infinity in V tells from one that is only small
        if (any && keep[h] < 1.4e-45f) keep[h] = 1.4e-45f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float& z = s[x >> 1][2 * (x & 1) + h];
          p[x] *= inv;
          z = z > -INFINITY && p[x] < 1.4e-45f ? 1.4e-45f : p[x];
        }
      }
#pragma unroll
      for (int r = 0; r < kRepairRows; ++r) {
        const float f = __shfl_sync(kAll, keep[r & 1], r >> 1);
#pragma unroll
        for (int i = 0; i < kV; ++i) o[r][i] *= f;
      }
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {
        const int at = s0 + 8 * x;
        const bool whole = at + 8 <= min(n_least, s1);
        float w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = x < 2 ? (x ? s[0][2 + h] : s[0][h]) : (x == 3 ? s[1][2 + h] : s[1][h]);
        Raw<kV> next[8];
        values(next, at + 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float f[kV];
          unpack<T>(u[e], f);
#pragma unroll
          for (int r = 0; r < kRepairRows; ++r) {
            const float p = __shfl_sync(kAll, w[r & 1], 4 * e + (r >> 1));
            if (whole || at + e < min(n_of[r], s1)) {  // a key that the row does not see may hold anything
#pragma unroll
              for (int i = 0; i < kV; ++i) o[r][i] = fmaf(p, f[i], o[r][i]);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = next[e];
      }
      bool open = false;  // what is NaN stays NaN
#pragma unroll
      for (int r = 0; r < kRepairRows; ++r) {
#pragma unroll
        for (int i = 0; i < kV; ++i) open |= (redo[r] >> i & 1) && !__isnanf(o[r][i]);
      }
      if (!__any_sync(kAll, open)) break;
    }
#pragma unroll
    for (int r = 0; r < kRepairRows; ++r) {
      T* row_dst = of_lane(dst, lane_of[r]);
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (redo[r] >> i & 1) row_dst[d0 + i] = from_f32<T>(fit<T>(o[r][i]));
    }
  }
}

template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kTaThreads, 1)
    tile_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const TileArgs args) {
  using Shape = TaShape<D>;
  constexpr int kStages = Shape::kStages, kKB = Shape::kKB, kTile = Shape::kTile, kBlk = 128 * 128;
  constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
  constexpr int kDeg = kBf16 ? 3 : 4;  // of exp2_fma
  constexpr uint32_t IDESC_S = idesc_half(kBf16, false, 128, 128);
  constexpr uint32_t IDESC_O = idesc_half(kBf16, true, 128, D);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smQ = smem;                       // [tile][k-block]
  uint8_t* smR = smQ + 2 * kTile;            // ring: [stage][k-block]
  uint8_t* smO = smR + kStages * kTile;      // staging
  uint64_t* bars = reinterpret_cast<uint64_t*>(smO + Shape::kStaging);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;              // the softmaxes have seen the item's last S: Q may be reloaded
  uint64_t* r_full = bars + 2;               // [kStages]
  uint64_t* r_empty = r_full + kStages;      // [kStages] likewise, 2 arrivals
  uint64_t* s_full = r_empty + kStages;      // [tile] S ready (and every earlier product of the tile done)
  uint64_t* p_full = s_full + 2;             // [tile][half] 64 columns of P written, and O rescaled
  uint64_t* o_full = p_full + 4;             // [tile] the item's last product done
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* repair = reinterpret_cast<uint8_t*>(tmem_slot + 2);  // [softmax warp] has written non-finite results

  if constexpr (MODE == PREFIX) asm volatile("griddepcontrol.launch_dependents;");
  const int warp = warp_id(), lane = lane_id();
  const int cta = static_cast<int>(blockIdx.x), G = static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(r_full + s, 1);
      mbar_init(r_empty + s, 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_full + 2 * t, 4);
      mbar_init(p_full + 2 * t + 1, 4);
      mbar_init(o_full + t, 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    for (int w = 0; w < 8; ++w) repair[w] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Items, heaviest first: round n of the G CTAs takes items nG .. nG + G - 1, alternately forwards and backwards,
  // which balances the CTAs' key blocks. Every warp walks the same items, all its lanes together.
  // PACKED, up to 32 sequences: no plan is made. Lane i holds sequence i, and an item's place in the order of falling
  // weight (key blocks) is found from counts: a sequence of len tokens has min(pairs, 128 w / (tokens of a pair)) pairs
  // of weight w or less (all of them where len <= 128 w), so walking the weights down and adding these up over the
  // lanes says which weight item number x has, and a scan over the lanes which sequence's and which pair.
  const int per_pair = 2 * args.tok;
  int n_items, one_first = 0, one_end = 0, seq_start = 0, seq_len = 0, level = 0, level_base = 0, level_count = 0;
  auto pairs_upto = [&](int w) { return seq_len <= kTaBlock * w ? (seq_len + per_pair - 1) / per_pair : kTaBlock * w / per_pair; };
  if constexpr (MODE == PACKED) {
    if (args.plan) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      n_items = args.plan->n_pairs * args.hkv;
      one_first = args.plan->first;
      one_end = args.plan->end;
    } else {
      auto clamp = [&](int x) { return min(max(x, 0), args.T); };
      one_first = clamp(args.cu[0]);
      int end = lane < args.n_seqs ? clamp(args.cu[lane + 1]) : 0;  // ascending whatever cu holds
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end = max(end, y);
      }
      end = max(end, one_first);
      seq_start = __shfl_up_sync(0xffffffffu, end, 1);
      if (lane == 0) seq_start = one_first;
      seq_len = end - seq_start;
      one_end = __shfl_sync(0xffffffffu, end, 31);
      n_items = __reduce_add_sync(0xffffffffu, (seq_len + per_pair - 1) / per_pair) * args.hkv;
    }
  } else {
    n_items = args.pairs * args.hkv * args.splits;
  }
  auto first_level = [&]() {
    level = __reduce_max_sync(0xffffffffu, (seq_len + kTaBlock - 1) / kTaBlock);
    level_base = 0;
    level_count = __reduce_add_sync(0xffffffffu, pairs_upto(level) - pairs_upto(level - 1));
  };
  if (MODE == PACKED && !args.plan) first_level();
  auto item = [&](int n, TileItem& it) -> bool {
    const int idx = n * G + ((n & 1) ? G - 1 - cta : cta);
    if (idx >= n_items) return false;
    it.kvh = idx % args.hkv;
    const int rest = idx / args.hkv;
    if constexpr (MODE == PACKED) {
      int begin, end;
      if (args.plan) {
        const int4 e = reinterpret_cast<const int4*>(args.plan + 1)[rest];
        it.q_tok = e.x;
        begin = e.y;
        end = e.z;
      } else {
        while (rest >= level_base + level_count) {  // weights down to 1 hold all pairs
          level_base += level_count;
          --level;
          level_count = __reduce_add_sync(0xffffffffu, pairs_upto(level) - pairs_upto(level - 1));
        }
        const int below = pairs_upto(level - 1), mine = pairs_upto(level) - below, at = rest - level_base;
        int upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        const int who = __ffs(__ballot_sync(0xffffffffu, upto > at)) - 1;
        begin = __shfl_sync(0xffffffffu, seq_start, who);
        end = begin + __shfl_sync(0xffffffffu, seq_len, who);
        it.q_tok = begin + __shfl_sync(0xffffffffu, below + at - (upto - mine), who) * per_pair;
      }
      it.kv_tok = begin;
      it.len = end - begin;
      it.q_pos = it.q_tok - begin;
      it.split = 0;
      for (int t = 0; t < 2; ++t) {  // a tile sees the keys up to its last token
        const int first = it.q_pos + t * args.tok, last = min(first + args.tok, it.len) - 1;
        it.nb[t] = last < first ? 0 : last / kTaBlock + 1;
      }
    } else {
      const int pair = rest % args.pairs;
      it.split = rest / args.pairs;
      it.q_tok = pair * per_pair;
      const int b0 = it.split * args.blocks_per_split;
      it.kv_tok = b0 * kTaBlock;
      const int nb = min(args.blocks_per_split, (args.P + kTaBlock - 1) / kTaBlock - b0);
      it.nb[0] = nb;
      it.nb[1] = it.q_tok + args.tok < args.B ? nb : 0;
      it.len = it.q_pos = 0;
    }
    return true;
  };

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTaRegsIssue));
  if (warp == 0) {
    // -------------------------------------------------------------------- TMA
    const bool leader = elect_one();
    int g = 0, q_loads = 0;  // ring blocks and Q loads so far
    bool ok = true;
    const uint32_t q_bytes = static_cast<uint32_t>(args.tok * args.group) * D * 2;
    auto load = [&](const CUtensorMap* map, int kvh, int tok) -> bool {
      const int st = g % kStages;
      if (!mbar_wait_warp(r_empty + st, ((g / kStages) & 1) ^ 1, abort_flag, args.err, 40)) return false;
      if (leader) {
        mbar_arrive_expect_tx(r_full + st, kTile);
        for (int kk = 0; kk < kKB; ++kk) tma_load_3d(smR + st * kTile + kk * kBlk, map, r_full + st, kk * 64, kvh, tok);
      }
      __syncwarp();
      ++g;
      return true;
    };
    TileItem it;
    for (int n = 0; ok && item(n, it); ++n) {
      const int tiles = it.nb[1] > 0 ? 2 : 1;
      if (!mbar_wait_warp(q_empty, (n & 1) ^ 1, abort_flag, args.err, 41)) break;
      if (leader) {
        mbar_arrive_expect_tx(q_full, tiles * q_bytes);
        for (int t = 0; t < tiles; ++t)
          for (int kk = 0; kk < kKB; ++kk)
            tma_load_4d(smQ + t * kTile + kk * kBlk, &tmQ, q_full, kk * 64, 0, it.kvh, it.q_tok + t * args.tok);
      }
      __syncwarp();
      ++q_loads;
      const int nb = max(it.nb[0], it.nb[1]);
      for (int j = 0; ok && j < nb; ++j)
        ok = load(&tmK, it.kvh, it.kv_tok + j * kTaBlock) && load(&tmV, it.kvh, it.kv_tok + j * kTaBlock);
    }
    // every load has landed before the CTA may exit
    volatile int never = 0;
    if (q_loads > 0) mbar_wait_warp(q_full, static_cast<uint32_t>((q_loads - 1) & 1), &never, args.err, 42);
    for (int s = 0; s < kStages && s < g; ++s) {
      const int last = (g - 1 - s) / kStages;  // the last use of stage s
      mbar_wait_warp(r_full + s, static_cast<uint32_t>(last & 1), &never, args.err, 42);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------------- MMA
    // The whole warp walks the loop, so that addresses and descriptors are warp-uniform values, and one elected lane
    // issues: from divergent code (lane 0 alone) an MMA went out every 85 to 90 cycles, and it takes 64.
    const bool leader = elect_one();
    bool ok = true, issued = false;
    int p_seen[2] = {0, 0};         // each tile's P so far
    uint32_t stage = 0, phase = 0;  // of the ring's next block
    const uint32_t ring0 = smem_u32(smR), q0 = smem_u32(smQ);
    // the stage i blocks on (i < kStages), and its phase
    auto stage_of = [&](uint32_t i) { return stage + i >= kStages ? stage + i - kStages : stage + i; };
    auto wait_ring = [&](uint32_t i) {
      const uint32_t st = stage_of(i);
      return mbar_wait_warp(r_full + st, phase ^ (stage + i >= kStages ? 1u : 0u), abort_flag, args.err, 43);
    };
    auto issue_s = [&](int t, uint32_t i) {
      tc_fence_after();
      if (leader) {
        const uint32_t tS = tmem + 128 * t;
        const uint64_t dQ = smem_desc_k_sw128(q0 + t * kTile), dK = smem_desc_k_sw128(ring0 + stage_of(i) * kTile);
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tS, dQ + (kk * (kBlk >> 4) + 2 * k), dK + (kk * (kBlk >> 4) + 2 * k), IDESC_S, (kk | k) != 0);
        }
        umma_commit(s_full + t);
      }
      __syncwarp();
      issued = true;
    };
    auto issue_pv = [&](int t, uint32_t i, bool first) -> bool {
      const uint32_t tO = tmem + 256 + 128 * t, tP = tmem + 128 * t;
      const uint64_t dV = smem_desc_mn_sw128(ring0 + stage_of(i) * kTile, kBlk);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!mbar_wait_warp(p_full + 2 * t + h, p_seen[t] & 1, abort_flag, args.err, 44)) return false;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ts(tO, tP + 32 * h + 8 * k, dV + (512 * h + 128 * k), IDESC_O, h || k ? 1u : first ? 0u : 1u);
        }
        __syncwarp();
      }
      ++p_seen[t];
      return true;
    };
    TileItem it;
    for (int n = 0; ok && item(n, it); ++n) {
      const int nb = max(it.nb[0], it.nb[1]);
      if (!mbar_wait_warp(q_full, n & 1, abort_flag, args.err, 45) || !wait_ring(0)) break;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (it.nb[t] > 0) issue_s(t, 0);
      for (int j = 0; ok && j < nb; ++j) {
        // the ring's next blocks: K_j, V_j, K_{j+1}
        ok = wait_ring(1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (ok && j < it.nb[t]) {
            ok = issue_pv(t, 1, j == 0);
            // K_{j+1} is waited for no earlier than it is used: its stage was released late
            if (ok && j + 1 < it.nb[t] && (ok = wait_ring(2))) issue_s(t, 2);
            if (ok && j + 1 == it.nb[t]) {
              if (leader) umma_commit(o_full + t);
              __syncwarp();
            }
          }
        }
        if (stage + 2 >= kStages) phase ^= 1;
        stage = stage_of(2);
      }
    }
    if (issued) {
      if (leader) umma_commit(drain);
      volatile int never = 0;
      mbar_wait_warp(drain, 0, &never, args.err, 46);
    }
  } else if (warp >= 4) {
    // -------------------------------------------------------------------- softmax (warps 4..11)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTaRegsSoftmax));
    const int t = (warp - 4) >> 2;           // tile
    const int qd = warp & 3;                 // TMEM lane quadrant = row block
    const int r = qd * 32 + lane;            // row of the tile
    const int r_tok = r / args.group, r_head = r - r_tok * args.group;
    const bool r_ok = r_tok < args.tok;      // rows past tok * group hold no query
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    const uint32_t tS = tmem + 128 * t + lane_off, tO = tmem + 256 + 128 * t + lane_off;
    const float sc = args.scale_log2;
    if constexpr (MODE == PACKED) {
      // tokens of no sequence
      const int64_t row = static_cast<int64_t>(args.hq) * D / 8;  // 16-byte pieces of a token
      const int64_t head = one_first * row, tail = (args.T - one_end) * row;
      uint4* o = static_cast<uint4*>(args.out);
      for (int64_t i = static_cast<int64_t>(cta) * 256 + threadIdx.x - 128; i < head + tail; i += static_cast<int64_t>(G) * 256)
        o[i < head ? i : one_end * row + i - head] = make_uint4(0, 0, 0, 0);
    }
    bool ok = true;
    int g = 0, items = 0, ring = 0;          // key blocks and items of this tile, ring blocks before this item
    TileItem it;
    for (int n = 0; ok && item(n, it); ring += 2 * max(it.nb[0], it.nb[1]), ++n) {
      const int nb = it.nb[t], other = it.nb[t ^ 1];
      if (nb == 0) continue;
      // one arrival of the two for this tile, both where the other tile has no part
      auto release = [&](uint64_t* bar, bool both) {
        if (qd == 0 && lane == 0) mbar_arrive_n(bar, both ? 2u : 1u);
      };
      auto stage = [&](int i) { return r_empty + (ring + i) % kStages; };
      const int pos = it.q_pos + t * args.tok + r_tok;  // PACKED: place in the sequence
      float m_use = -INFINITY, l = 0.f;
      for (int j = 0; j < nb; ++j, ++g) {
        if (!mbar_wait_warp(s_full + t, g & 1, abort_flag, args.err, 47)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // S(j) is done, and with it the product with V_{j-1}: K_j and V_{j-1} may be overwritten, after the last S Q too
        release(stage(2 * j), j >= other);
        if (j > 0) release(stage(2 * j - 1), j - 1 >= other);
        if (j + 1 == nb) release(q_empty, other == 0);
        // the last key of this block that the row sees
        const int last = MODE == PACKED ? pos - j * kTaBlock : args.P - 1 - it.kv_tok - j * kTaBlock;
        const bool masked = __any_sync(0xffffffffu, last < kTaBlock - 1);
        uint32_t v[4][32];                   // this row of S
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(tS + c * 32, v[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(v[c]);
        if (masked) {
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (e > last) v[e >> 5][e & 31] = __float_as_uint(-INFINITY);
        }
        // eight partial maxima, so that the reduction is not one long chain; two keys per instruction
        float m8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = __uint_as_float(v[0][i]);
#pragma unroll
        for (int e = 8; e + 16 <= 128; e += 16) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            m8[i] = fmax3(m8[i], __uint_as_float(v[(e + i) >> 5][(e + i) & 31]), __uint_as_float(v[(e + 8 + i) >> 5][(e + 8 + i) & 31]));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(m8[i], __uint_as_float(v[3][24 + i]));
        const float m_blk = fmaxf(fmax3(m8[0], m8[1], m8[2]), fmaxf(fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * sc;
        float alpha = 1.f;
        const bool raise = m_blk > m_use + kTaRescale;
        if (raise) {
          alpha = fast_exp2(m_use - m_blk);  // 0 while m_use is -inf
          m_use = m_blk;
        }
        if (j >= 1 && __any_sync(0xffffffffu, raise)) {
          // S(j) was issued after O += P(j-1) V(j-1), so O is complete
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld_32x32b_x16(tO + c * 16, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x32b_x16(tO + c * 16, o);
          }
        }
        l *= alpha;
        const float neg_m = m_use == -INFINITY ? 0.f : -m_use;
        float2 rs4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(neg_m, neg_m);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t(&x)[32] = v[c];
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 z = __ffma2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), sc2, nm2);
            const float2 pp = ((e >> 1) & 3) < ta_fma_of_4(D) ? exp2_fma<kDeg>(z) : make_float2(fast_exp2(z.x), fast_exp2(z.y));
            rs4[(e >> 1) & 3] = __fadd2_rn(rs4[(e >> 1) & 3], pp);
            w[e / 2] = pack2<T>(pp.x, pp.y);
          }
          __syncwarp();
          tmem_st_32x32b_x16(tS + c * 16, w);  // over columns of S already read
          if (c & 1) {
            // half of P is ready: its share of the product may start
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 2 * t + (c >> 1));
          }
        }
        l += ((rs4[0].x + rs4[0].y) + (rs4[1].x + rs4[1].y)) + ((rs4[2].x + rs4[2].y) + (rs4[3].x + rs4[3].y));
      }
      if (!ok || !mbar_wait_warp(o_full + t, items & 1, abort_flag, args.err, 48)) break;
      ++items;
      release(stage(2 * nb - 1), nb - 1 >= other);
      tc_fence_after();
      const int tok = it.q_tok + t * args.tok + r_tok;
      const int head = it.kvh * args.group + r_head;
      const bool mine = r_ok && (MODE == PACKED ? pos < it.len : tok < args.B);
      const int row = mine ? tok * args.hq + head : -1;
      // The rows go out through shared memory, 128 bytes of each at a time, so that a store of the warp writes four
      // whole lines; the threads' own rows, 16 bytes each, were 32 half sectors apart (128 us instead of 113 for 16
      // ragged prompts). put() takes 16-byte piece p of the thread's row, flush() writes the pieces to base + row * pitch.
      uint8_t* staging = smO + (warp - 4) * 4096;
      auto put = [&](int p, uint4 u) { *reinterpret_cast<uint4*>(staging + lane * 128 + ((p ^ lane) & 7) * 16) = u; };
      auto flush = [&](uint8_t* base, int pitch) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = i * 4 + (lane >> 3), to = __shfl_sync(0xffffffffu, row, from);
          const uint4 u = *reinterpret_cast<const uint4*>(staging + from * 128 + ((lane ^ from) & 7) * 16);
          if (to >= 0) *reinterpret_cast<uint4*>(base + static_cast<int64_t>(to) * pitch + (lane & 7) * 16) = u;
        }
        __syncwarp();
      };
      uint32_t o[32];
      if constexpr (MODE == PACKED) {
        const float inv = l > 0.f || __isnanf(l) ? 1.f / l : 0.f;
        uint32_t most = 0;  // the largest magnitude written, of even and of odd dimensions
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            __syncwarp();
            tmem_ld_32x32b_x32(tO + c * 64 + h * 32, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(o[e + i]) * inv;
              const uint4 u = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
              most = max_abs2<T>(max_abs2<T>(max_abs2<T>(max_abs2<T>(most, u.x), u.y), u.z), u.w);
              put(h * 4 + e / 8, u);
            }
          }
          flush(static_cast<uint8_t*>(args.out) + c * 128, D * 2);
        }
        Raw<2> w;
        float ends[2];
        w.w[0] = most;
        unpack<T>(w, ends);
        if (mine && !(ends[0] < INFINITY && ends[1] < INFINITY)) repair[warp - 4] = 1;
      } else {
        const int64_t part = static_cast<int64_t>(it.split) * args.B * args.hq;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          __syncwarp();
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; e += 4) put(e / 4, make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]));
          flush(reinterpret_cast<uint8_t*>(args.part_o + part * D) + c * 128, D * 4);
        }
        if (mine) args.part_ml[part + row] = make_float2(m_use, l);
      }
      // O has been read: the next item's first product (issued after this warp's next P) may overwrite it
      tc_fence_before();
    }
    if constexpr (MODE == PACKED) {
      __syncwarp();
      if (ok && repair[warp - 4]) {
        if (!args.plan) first_level();
        for (int n = 0; item(n, it); ++n) {
          if (it.nb[t] == 0) continue;
          const int pos = it.q_pos + t * args.tok + r_tok;
          const bool mine = r_ok && pos < it.len;
          const int64_t first = it.kv_tok, tok = mine ? it.q_tok + t * args.tok + r_tok : first, head = it.kvh * args.group + r_head;
          repair_rows<T, D>(mine, pos, static_cast<const T*>(args.q) + tok * args.q_st + head * args.q_sh,
                            static_cast<T*>(args.out) + (tok * args.hq + head) * D,
                            static_cast<const T*>(args.k) + first * args.k_st + it.kvh * args.k_sh, args.k_st,
                            static_cast<const T*>(args.v) + first * args.v_st + it.kvh * args.v_sh, args.v_st, sc);
        }
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------- the plan of a packed call
// One block: the sequences' bounds (the running maximum of the clamped words, so they ascend whatever cu holds), and
// their tile pairs sorted by key blocks, most first, by counting. The order among equals is left to the atomics: it
// changes which CTA takes a pair, never a result. The list has room for tokens / (2 tok) + n_seqs pairs, which the
// ascending bounds cannot exceed.
constexpr int kPlanFree = 32;  // up to so many sequences no plan is made (one lane each)
constexpr int kPlanThreads = 1024;
constexpr int kPlanBins = 2048;

__device__ __forceinline__ int warp_scan(int x, bool is_max) {
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane_id() >= o) x = is_max ? max(x, y) : x + y;
  }
  return x;
}

// Inclusive scan over the block; every thread calls it.
__device__ __forceinline__ int block_scan(int x, bool is_max, int* scratch) {
  x = warp_scan(x, is_max);
  if (lane_id() == 31) scratch[warp_id()] = x;
  __syncthreads();
  if (warp_id() == 0) scratch[lane_id()] = warp_scan(scratch[lane_id()], is_max);
  __syncthreads();
  if (warp_id() > 0) {
    const int y = scratch[warp_id() - 1];
    x = is_max ? max(x, y) : x + y;
  }
  __syncthreads();
  return x;
}

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const int32_t* cu, int n_seqs, int T, int per_pair,
                                                                   PlanHeader* plan) {
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ int scratch[32], starts[kPlanThreads], ends[kPlanThreads], upto[kPlanThreads], bins[kPlanBins];
  int4* list = reinterpret_cast<int4*>(plan + 1);
  auto clamp = [&](int x) { return min(max(x, 0), T); };
  const int first = clamp(cu[0]);
  for (int i = threadIdx.x; i < kPlanBins; i += kPlanThreads) bins[i] = 0;
  __syncthreads();
  int total = 0, reached = first;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      // bins[i] = pairs with more blocks than i: the place of the first pair of bin i
      const int a = bins[kPlanBins - 1 - 2 * threadIdx.x], b = bins[kPlanBins - 2 - 2 * threadIdx.x];
      __syncthreads();
      const int s = block_scan(a + b, false, scratch);
      bins[kPlanBins - 1 - 2 * threadIdx.x] = s - a - b;
      bins[kPlanBins - 2 - 2 * threadIdx.x] = s - b;
      __syncthreads();
    }
    reached = first;
    total = 0;
    for (int c = 0; c < n_seqs; c += kPlanThreads) {
      const int i = c + static_cast<int>(threadIdx.x);
      const int end = max(block_scan(i < n_seqs ? clamp(cu[i + 1]) : 0, true, scratch), reached);
      ends[threadIdx.x] = end;
      __syncthreads();
      const int start = threadIdx.x ? ends[threadIdx.x - 1] : reached;
      starts[threadIdx.x] = start;
      const int pairs = block_scan((end - start + per_pair - 1) / per_pair, false, scratch);
      upto[threadIdx.x] = pairs;
      __syncthreads();
      const int here = upto[kPlanThreads - 1];
      for (int p = threadIdx.x; p < here; p += kPlanThreads) {
        int lo = 0, hi = kPlanThreads - 1;  // the first sequence with upto > p
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (upto[mid] > p) hi = mid; else lo = mid + 1;
        }
        const int at = p - (lo ? upto[lo - 1] : 0), len = ends[lo] - starts[lo];
        const int blocks = (min(len, (at + 1) * per_pair) + kTaBlock - 1) / kTaBlock;
        const int bin = min(blocks, kPlanBins - 1);
        const int place = atomicAdd(&bins[bin], 1);
        if (pass == 1) list[place] = make_int4(starts[lo] + at * per_pair, starts[lo], ends[lo], 0);
      }
      total += here;
      reached = ends[kPlanThreads - 1];
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) *plan = PlanHeader{total, first, reached, 0};
}

// ---------------------------------------------------------------------------- the batch's own keys and the join
struct OwnArgs {
  const void *q, *ck, *cv, *pk, *pv;
  int64_t q_sb, q_sh, ck_sb, ck_st, ck_sh, cv_sb, cv_st, cv_sh, pk_st, pk_sh, pv_st, pv_sh;
  const int32_t* lens;
  int B, S, hq, hkv, group;
  int P;       // prefix keys read here, before the own ones (few sequences); else 0
  int parts;   // of the prefix: part_o / part_ml [parts + (splits > 1 ? splits : 0)][B * hq]
  int splits;  // of the own keys
  float scale_log2;
  float* part_o;
  float2* part_ml;
  void* out;
};

constexpr int kOwnWarps = 4;
constexpr int kOwnStep = 16;   // keys of a warp's step
constexpr int kOwnStages = 2;  // steps under way per warp
constexpr int kOwnMinSteps = 8;  // of a split, two per warp

// A sequence's own keys: few rows (the query heads that share a key head) against a cache of its own, so the time is
// the reading of the cache. One CTA per (sequence, key head, 8 query heads, split); its warps take steps of 16 keys in
// turn, two steps' copies under way each (cp.async: 16 KB per warp, 192 KB per SM), each with a running softmax of its
// own, joined at the end. The products are mma.sync 16 x 8 x 16 with keys, then dimensions, as rows and the query heads
// as columns (tcgen05's 128 rows would not be filled): S^T = K Q^T, O^T = V^T P^T. K and V are copied in 16-byte pieces
// that are fragments as they are: of K, lane (g, t) takes dimensions 32 c + 8 t .. + 7 of keys g and g + 8, which are A
// fragments when the queries' B fragments are read in the same order; of V, dimensions 64 e + 8 g .. + 7 of keys 2 t,
// 2 t + 1, 2 t + 8, 2 t + 9, which are, paired by a byte permute, A fragments of output rows in the order of dimensions
// 64 e + 8 g + 2 i (row g of product i) and 64 e + 8 g + 2 i + 1 (row g + 8). P^T is S^T's fragment, transposed by
// movmatrix. Every lane reads back just what it copied, so no barrier is needed.
// Keys past the length are not read and count as zeros with score -inf.
// 190 sequences of 300 keys, 16 heads over 8 of 128, alone: 58 us for 247 MB, 4.2 TB/s; the tensor pipe is busy 7 % of
// the time, the issue slots 25 %. 300 keys are 19 steps for four warps, so about five to a warp with two under way: the
// copies are off most of the time, between a start that waits for the length and two barriers and a join at the end.
// With one split the CTA also joins the prefix's parts and writes the output; else it leaves a part like theirs.
template <typename T, int D>
__global__ void __launch_bounds__(kOwnWarps * 32, 3) own_keys_kernel(const OwnArgs a) {
  constexpr bool kBf16 = !__is_same(T, __half);
  constexpr int kC = D / 32, kE = D / 64;
  constexpr int kStageBytes = 2 * kC * 2 * 512;  // a step's K and V, 16 bytes of each lane per piece
  extern __shared__ __align__(16) uint8_t own_smem[];
  uint8_t* ring = own_smem + warp_id() * (kOwnStages * kStageBytes);
  float(*so)[8][D + 4] = reinterpret_cast<float(*)[8][D + 4]>(own_smem);  // the warps' sums, once the ring is done
  __shared__ float2 sml[kOwnWarps][8];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int b = static_cast<int>(blockIdx.x) / a.hkv, kvh = static_cast<int>(blockIdx.x) % a.hkv;
  const int h0 = kvh * a.group + static_cast<int>(blockIdx.z) * 8;              // the tile's first query head
  const int rows = min(8, a.group - static_cast<int>(blockIdx.z) * 8);
  const int n = a.P + min(max(a.lens[b], 0), a.S);
  const int steps = (n + kOwnStep - 1) / kOwnStep;
  const int per = max((steps + a.splits - 1) / a.splits, kOwnMinSteps);
  const int s0 = min(steps, static_cast<int>(blockIdx.y) * per), s1 = min(steps, s0 + per);

  const T* kp = static_cast<const T*>(a.ck) + static_cast<int64_t>(b) * a.ck_sb + static_cast<int64_t>(kvh) * a.ck_sh + 8 * t;
  const T* vp = static_cast<const T*>(a.cv) + static_cast<int64_t>(b) * a.cv_sb + static_cast<int64_t>(kvh) * a.cv_sh + 8 * g;
  const T* pkp = static_cast<const T*>(a.pk) + static_cast<int64_t>(kvh) * a.pk_sh + 8 * t;
  const T* pvp = static_cast<const T*>(a.pv) + static_cast<int64_t>(kvh) * a.pv_sh + 8 * g;
  auto key_row = [&](int key) { return key < a.P ? pkp + key * a.pk_st : kp + (key - a.P) * a.ck_st; };
  auto value_row = [&](int key) { return key < a.P ? pvp + key * a.pv_st : vp + (key - a.P) * a.cv_st; };
  auto fetch = [&](int step, int st) {
    if (step < s1) {
      const uint32_t dst = smem_u32(ring + st * kStageBytes + lane * 16);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = step * kOwnStep + 8 * r + g;
        const T* src = key_row(min(key, n - 1));
#pragma unroll
        for (int c = 0; c < kC; ++c) cp_async_16(dst + (r * kC + c) * 512, src + 32 * c, key < n);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = step * kOwnStep + 2 * t + (x & 1) + 8 * (x >> 1);
        const T* src = value_row(min(key, n - 1));
#pragma unroll
        for (int e = 0; e < kE; ++e) cp_async_16(dst + (2 * kC + e * 4 + x) * 512, src + 64 * e, key < n);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kOwnStages; ++i) fetch(s0 + warp + i * kOwnWarps, i);

  uint4 q[kC];  // query head g, dimensions 32 c + 8 t .. + 7
#pragma unroll
  for (int c = 0; c < kC; ++c)
    q[c] = g < rows ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<int64_t>(b) * a.q_sb +
                                                      static_cast<int64_t>(h0 + g) * a.q_sh + 8 * t + 32 * c)
                    : make_uint4(0, 0, 0, 0);
  float o[kE][4][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // m, l: of query heads 2 t, 2 t + 1
#pragma unroll
  for (int e = 0; e < kE; ++e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[e][i][0] = o[e][i][1] = o[e][i][2] = o[e][i][3] = 0.f;
  }
  int st = 0;
  for (int step = s0 + warp; step < s1; step += kOwnWarps, st = st + 1 == kOwnStages ? 0 : st + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kOwnStages - 1) : "memory");
    const uint4* mine = reinterpret_cast<const uint4*>(ring + st * kStageBytes) + lane;
    float s2[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // two sums, so that the products are two chains
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const uint4 k0 = mine[c * 32], k1 = mine[(kC + c) * 32];
      const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
      mma_16816<kBf16>(s2[0], a0, q[c].x, q[c].y);
      mma_16816<kBf16>(s2[1], a1, q[c].z, q[c].w);
    }
    // s[e]: key g (g + 8 for e >= 2) of the step, query head 2 t + (e & 1)
    float s[4], f[2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[e] = step * kOwnStep + g + 8 * (e >> 1) < n ? (s2[0][e] + s2[1][e]) * a.scale_log2 : -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(s[h], s[2 + h]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float mn = fmaxf(m[h], mx);
      f[h] = mn == -INFINITY ? 1.f : fast_exp2(m[h] - mn);
      m[h] = mn;
      const float base = mn == -INFINITY ? 0.f : mn;
      s[h] = fast_exp2(s[h] - base);
      s[2 + h] = fast_exp2(s[2 + h] - base);
      l[h] = l[h] * f[h] + (s[h] + s[2 + h]);  // this lane's keys; the lanes' sums are added at the end
    }
    uint32_t p0, p1;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p0) : "r"(pack2<T>(s[0], s[1])));
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p1) : "r"(pack2<T>(s[2], s[3])));
    if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[e][i][0] *= f[0], o[e][i][1] *= f[1], o[e][i][2] *= f[0], o[e][i][3] *= f[1];
      }
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const uint4 u0 = mine[(2 * kC + e * 4) * 32], u1 = mine[(2 * kC + e * 4 + 1) * 32], u2 = mine[(2 * kC + e * 4 + 2) * 32],
                  u3 = mine[(2 * kC + e * 4 + 3) * 32];
      const uint32_t v0[4] = {u0.x, u0.y, u0.z, u0.w}, v1[4] = {u1.x, u1.y, u1.z, u1.w}, v2[4] = {u2.x, u2.y, u2.z, u2.w},
                     v3[4] = {u3.x, u3.y, u3.z, u3.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t av[4] = {__byte_perm(v0[i], v1[i], 0x5410), __byte_perm(v0[i], v1[i], 0x7632),
                                __byte_perm(v2[i], v3[i], 0x5410), __byte_perm(v2[i], v3[i], 0x7632)};
        mma_16816<kBf16>(o[e][i], av, p0, p1);
      }
    }
    fetch(step + kOwnStages * kOwnWarps, st);  // into the stage just read
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // the warp's part
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
    if (g == 0) sml[warp][2 * t + h] = make_float2(m[h], l[h]);
    if (2 * t + h < rows) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        float* dst = &so[warp][2 * t + h][64 * e + 8 * g];
        *reinterpret_cast<float4*>(dst) = make_float4(o[e][0][h], o[e][0][2 + h], o[e][1][h], o[e][1][2 + h]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(o[e][2][h], o[e][2][2 + h], o[e][3][h], o[e][3][2 + h]);
      }
    }
  }
  __syncthreads();
  // The prefix's parts, which are joined here with one split. With more, join_kernel reads them, and one CTA that waits
  // for the kernel that writes them is enough: this grid's end is then after its end, and the others leave their SMs.
  if (a.splits == 1 || (blockIdx.x + 1 == gridDim.x && blockIdx.y + 1 == gridDim.y && blockIdx.z + 1 == gridDim.z))
    asm volatile("griddepcontrol.wait;" ::: "memory");
  // four dimensions per thread
  const int64_t n_rows = static_cast<int64_t>(a.B) * a.hq;
  for (int i = threadIdx.x; i < rows * (D / 4); i += kOwnWarps * 32) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    const int64_t row = static_cast<int64_t>(b) * a.hq + h0 + r;
    const int parts = a.splits == 1 ? a.parts : 0;
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < kOwnWarps; ++w) mm = fmaxf(mm, sml[w][r].x);
#pragma unroll 8
    for (int s = 0; s < parts; ++s) mm = fmaxf(mm, a.part_ml[s * n_rows + row].x);
    const float base = mm == -INFINITY ? 0.f : mm;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 x) {
      const float f = fast_exp2(ml.x - base);
      ll = fmaf(f, ml.y, ll);
      acc.x = fmaf(f, x.x, acc.x), acc.y = fmaf(f, x.y, acc.y), acc.z = fmaf(f, x.z, acc.z), acc.w = fmaf(f, x.w, acc.w);
    };
    for (int w = 0; w < kOwnWarps; ++w) add(sml[w][r], *reinterpret_cast<const float4*>(&so[w][r][d]));
#pragma unroll 8
    for (int s = 0; s < parts; ++s)
      add(a.part_ml[s * n_rows + row], *reinterpret_cast<const float4*>(a.part_o + (s * n_rows + row) * D + d));
    if (a.splits == 1) {
      const float inv = ll > 0.f || __isnanf(ll) ? 1.f / ll : 0.f;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * D + d) =
          make_uint2(pack2<T>(fit<T>(acc.x * inv), fit<T>(acc.y * inv)), pack2<T>(fit<T>(acc.z * inv), fit<T>(acc.w * inv)));
    } else {
      const int64_t at = (a.parts + blockIdx.y) * n_rows + row;
      *reinterpret_cast<float4*>(a.part_o + at * D + d) = acc;
      if (d == 0) a.part_ml[at] = make_float2(mm, ll);
    }
  }
}

// One block per row, its warps with every fourth part each: the parts' sums brought to one maximum and added, in a
// fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const float* part_o, const float2* part_ml, int parts, int64_t n_rows, T* out) {
  const int64_t row = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kV = D / 32;  // dimensions of a lane
  __shared__ float sums[4][D];
  __shared__ float2 sml[4];
  float mm = -INFINITY, ll = 0.f, acc[kV];
  for (int s = lane_id(); s < parts; s += 32) mm = fmaxf(mm, part_ml[s * n_rows + row].x);
  for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
  const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
  for (int i = 0; i < kV; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = warp_id(); s < parts; s += 4) {
    const float2 ml = part_ml[s * n_rows + row];
    const float f = fast_exp2(ml.x - base);
    ll = fmaf(f, ml.y, ll);
    const float* x = part_o + (s * n_rows + row) * D + lane_id() * kV;
    if constexpr (kV == 4) {
      const float4 u = *reinterpret_cast<const float4*>(x);
      acc[0] = fmaf(f, u.x, acc[0]), acc[1] = fmaf(f, u.y, acc[1]), acc[2] = fmaf(f, u.z, acc[2]), acc[3] = fmaf(f, u.w, acc[3]);
    } else {
      const float2 u = *reinterpret_cast<const float2*>(x);
      acc[0] = fmaf(f, u.x, acc[0]), acc[1] = fmaf(f, u.y, acc[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) sums[warp_id()][lane_id() * kV + i] = acc[i];
  if (lane_id() == 0) sml[warp_id()].y = ll;
  __syncthreads();
  if (threadIdx.x < D / 2) {
    const int d = threadIdx.x * 2;
    float x = 0.f, y = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x += sums[w][d], y += sums[w][d + 1], l += sml[w].y;
    const float inv = l > 0.f || __isnanf(l) ? 1.f / l : 0.f;
    reinterpret_cast<uint32_t*>(out + row * D)[threadIdx.x] = pack2<T>(fit<T>(x * inv), fit<T>(y * inv));
  }
}

template <typename T, int D>
static int launch_own(const OwnArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.B * a.hkv), static_cast<unsigned>(a.splits), static_cast<unsigned>((a.group + 7) / 8));
  constexpr int kSmem = kOwnWarps * kOwnStages * (D / 32) * 2048;
  static_assert(kSmem >= kOwnWarps * 8 * (D + 4) * 4, "the sums lie where the ring was");
  auto kern = own_keys_kernel<T, D>;
  static std::atomic<bool> configured[64];  // setting the attribute twice from two threads is harmless
  int dev = 0;
  XDNA_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    XDNA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  // after the prefix's kernel it may start early; alone it is an ordinary launch
  int rc;
  if (a.parts > 0) {
    rc = launch_early("own_keys_kernel", kern, grid, kOwnWarps * 32, kSmem, s, a);
  } else {
    kern<<<grid, kOwnWarps * 32, kSmem, s>>>(a);
    rc = check_launch("own_keys_kernel");
  }
  if (rc != XDNA_OK || a.splits == 1) return rc;
  const int64_t n_rows = static_cast<int64_t>(a.B) * a.hq;
  return launch_early("join_kernel", join_kernel<T, D>, dim3(static_cast<unsigned>(n_rows)), 128, 0, s, a.part_o, a.part_ml,
                      a.parts + a.splits, n_rows, a.out);
}

// ---------------------------------------------------------------------------- host
static int check_heads(const char* what, int64_t hq, int64_t hkv, int64_t d, int dtype, float scale) {
  XDNA_CHECK_ARG(hq >= 1 && hkv >= 1 && hq % hkv == 0 && hq / hkv <= 128,
                 "%s: %lld query heads over %lld key heads", what, (long long)hq, (long long)hkv);
  XDNA_CHECK_ARG(dtype == XDNA_BF16 || dtype == XDNA_F16, "%s: bf16 or f16", what);
  XDNA_CHECK_ARG(scale > 0.f && scale * kLog2E < INFINITY, "%s: the scale must be positive and at most 2.3e38", what);
  if (d != 64 && d != 128) return fail(XDNA_ERR_UNSUPPORTED, "%s: head dimension %lld (64 or 128)", what, (long long)d);
  return XDNA_OK;
}

static bool row_ok(const void* p, int64_t a, int64_t b, int64_t c = 8) {
  return p != nullptr && aligned16(p) && a > 0 && b > 0 && c > 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

// q [n, hq, d] as (dimension, head of the group, key head, token): a box is a tile's 64 columns of all its rows.
static int q_map(CUtensorMap* m, const void* q, int64_t st, int64_t sh, int64_t n, int64_t hkv, int64_t group,
                 int64_t tok, int64_t d, int dtype) {
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)group, (uint64_t)hkv, (uint64_t)n};
  const uint64_t strides[3] = {(uint64_t)sh * 2, (uint64_t)(sh * group) * 2, (uint64_t)st * 2};
  const uint32_t box[4] = {64, (uint32_t)group, 1, (uint32_t)tok};
  return encode_tma(m, dtype == XDNA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, q, dims,
                    strides, box, "attention q");
}

static int kv_map(CUtensorMap* m, const void* k, int64_t st, int64_t sh, int64_t n, int64_t hkv, int64_t d, int dtype) {
  const uint64_t dims[3] = {(uint64_t)d, (uint64_t)hkv, (uint64_t)n};
  const uint64_t strides[2] = {(uint64_t)sh * 2, (uint64_t)st * 2};
  const uint32_t box[3] = {64, 1, kTaBlock};
  return encode_tma(m, dtype == XDNA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, k, dims,
                    strides, box, "attention k/v");
}

template <typename T, int D, int MODE>
static int launch_tiles_as(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileArgs& a, int grid,
                           cudaStream_t s) {
  static std::atomic<bool> configured[64];  // setting the attribute twice from two threads is harmless
  int dev = 0;
  XDNA_CUDA(cudaGetDevice(&dev));
  auto kern = tile_attention_kernel<T, D, MODE>;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    // setmaxnreg shares out the launch's registers: with fewer its warps would wait for good
    cudaFuncAttributes attr;
    XDNA_CUDA(cudaFuncGetAttributes(&attr, kern));
    if (attr.numRegs < kTaRegsLaunch) return fail(XDNA_ERR_UNSUPPORTED, "tile_attention_kernel: built with %d registers", attr.numRegs);
    XDNA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TaShape<D>::kSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  if (a.plan) {  // it may start while the plan is made
    return launch_early("tile_attention_kernel", kern, dim3(grid), kTaThreads, TaShape<D>::kSmem, s, q, k, v, a);
  }
  kern<<<grid, kTaThreads, TaShape<D>::kSmem, s>>>(q, k, v, a);
  return check_launch("tile_attention_kernel");
}

template <int MODE>
static int launch_tiles(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileArgs& a, int64_t d,
                        int dtype, int grid, cudaStream_t s) {
  if (dtype == XDNA_BF16)
    return d == 128 ? launch_tiles_as<__nv_bfloat16, 128, MODE>(q, k, v, a, grid, s)
                    : launch_tiles_as<__nv_bfloat16, 64, MODE>(q, k, v, a, grid, s);
  return d == 128 ? launch_tiles_as<__half, 128, MODE>(q, k, v, a, grid, s)
                  : launch_tiles_as<__half, 64, MODE>(q, k, v, a, grid, s);
}

static int64_t plan_pairs(int64_t n_seqs, int64_t tokens, int64_t group) { return tokens / (2 * (128 / group)) + n_seqs; }

// How a prefix call is split (times: graph replays with warm operands; a call among others takes a few us more). One
// sequence, and few with a short prefix, read the prefix themselves, before their own keys (direct). With 8 key heads of
// 128, direct against the tile kernel: 2 sequences and a prefix of 3000 10.9 us and
// 14.7, of 8000 22.1 and 17.1; 4 and 1000 8.7 and 9.2, and 2000 14.3 and 11.2; 8 and 500 8.7 and 10.4, and 1000 16.3 and
// 11.3; with 2 of 64, 8 and 1000 6.3 and 8.0, 16 and 1500 8.8 and 9.5.
// A sequence's keys, where the sequences and key heads alone are few CTAs for an SM, are split into pieces of at least
// 128 (a CTA's two steps per warp), at most 32: lengths differ, and the longest would be waited for.
// Else the prefix's blocks are split over at most one CTA per SM. The own keys' kernel runs beside this one on the SMs
// that it leaves, as long as its CTAs need not wait for it (where the own keys are split too, or the CTAs all fit
// there, three to an SM). Then the number of parts is a balance: of a part's time, 10 us and 1.4 per block (2 where
// its items have two tiles), against the work of both kernels, 8 us per part's CTA and those blocks and the own keys,
// half the cache, at 20 KB per us and SM, spread over all SMs. Else the two follow each other, or, where that is
// shorter, caches of two pieces or more are split too, for a join's 3 us. (32 sequences, prefix 4096, caches of 600:
// 16 parts of 2 blocks 26.5 us, 8 parts 24.2, 6 parts 22.1; 64 and caches of 300: 28.9, 25.7, 24.1; 8 sequences,
// prefix 8192, caches of 300: 16 parts of 4 blocks 18.2, 8 parts 23.2; 16 sequences, prefix 2000, caches of 64: 16
// parts of one block 14.0, 8 parts 12.1; 100 sequences, prefix 1000, caches of 200: 8 parts of one block 26.3, 4 parts
// 28.0. Split caches against whole ones: 300 sequences, prefix 9000, caches of 300: 81 us against 100; 190 and 16381:
// 69 against 73; 190 and 4096: 49 against 51.)
// The lengths are on the device, so half the cache stands for them. A cache with much more room than it holds makes the
// parts too few: 32 sequences, prefix 4096, up to 600 keys of their own take 25 us in caches of 600, 31 of 1200, 64 of
// 2400 and more; 190, prefix 16381, up to 301 keys: 71 in caches of 301, 93 of 602, 130 of 1204, 241 of 4096 and more. A
// caller with long caches passes views of them that are about as long as the longest sequence.
struct PrefixSplit {
  bool direct;
  int64_t pairs, parts, blocks_per_part, own;
  PrefixSplit(int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d, int sms) {
    direct = B == 1 || B * P * hkv * d <= 6 << 20;
    const int64_t tok = 128 / (hq / hkv), blocks = direct ? 0 : (P + kTaBlock - 1) / kTaBlock;
    const int64_t ctas = B * hkv * ((hq / hkv + 7) / 8), keys = S + (direct ? P : 0);
    own = std::max<int64_t>(1, std::min<int64_t>({(keys + 127) / 128, 8 * sms / ctas, 32}));
    pairs = (B + 2 * tok - 1) / (2 * tok);
    const int64_t units = pairs * hkv;
    const double block = B > tok ? 2.0 : 1.4, keys_work = 0.5 * B * S * hkv * d * 4 / 20e3;
    double best = 1e30;
    blocks_per_part = 0;
    const int64_t most = std::max<int64_t>(1, std::min(blocks, sms / units)), whole = own;
    for (int64_t per = (blocks + most - 1) / most; per >= 1 && per <= blocks && 10 + block * per < best; ++per) {
      const int64_t c = units * ((blocks + per - 1) / per);
      const double part = 10 + block * per, beside = std::max(part, (keys_work + 8.0 * c + block * units * blocks) / sms);
      const bool fits = whole > 1 || ctas <= 3 * (sms - c);
      const double time = fits ? beside : part + 3 + keys_work / sms;
      if (time < best) best = time, blocks_per_part = per, own = whole;
      if (!fits && S >= 256 && beside + 3 < best) best = beside + 3, blocks_per_part = per, own = 2;
    }
    parts = blocks ? (blocks + blocks_per_part - 1) / blocks_per_part : 0;
  }
  int64_t all() const { return parts + (own > 1 ? own : 0); }
};

}  // namespace xdna

using namespace xdna;

extern "C" {

size_t xdna_packed_attention_workspace(int64_t n_seqs, int64_t tokens, int64_t hq, int64_t hkv) {
  if (n_seqs <= kPlanFree || tokens < 0 || hkv < 1 || hq < hkv || hq / hkv > 128) return 0;
  return sizeof(PlanHeader) + 16 * static_cast<size_t>(plan_pairs(n_seqs, tokens, hq / hkv));
}

int xdna_packed_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                          const void* v, int64_t v_st, int64_t v_sh, const int32_t* cu_seqlens, int64_t n_seqs,
                          int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int dtype, float scale, void* out,
                          void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_heads("packed_attention", hq, hkv, d, dtype, scale);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(tokens >= 0 && n_seqs >= 0 && tokens < (1ll << 31) / hq && n_seqs < (1 << 24),
                 "packed_attention: bad sizes");
  int sms = 0;
  if ((rc = check_device(&sms)) != XDNA_OK) return rc;
  if (tokens == 0) return XDNA_OK;
  XDNA_CHECK_ARG(row_ok(q, q_st, q_sh) && row_ok(k, k_st, k_sh) && row_ok(v, v_st, v_sh) && cu_seqlens && out &&
                     aligned16(out),
                 "packed_attention: operands must be 16-byte aligned with strides that are positive multiples of 8");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_seqs == 0) {
    XDNA_CUDA(cudaMemsetAsync(out, 0, static_cast<size_t>(tokens * hq * d * 2), s));
    return XDNA_OK;
  }
  const int64_t group = hq / hkv, tok = 128 / group;
  TileArgs a{};
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.group = static_cast<int>(group);
  a.tok = static_cast<int>(tok);
  a.scale_log2 = scale * kLog2E;
  a.err = device_error_word();
  a.out = out;
  a.cu = cu_seqlens;
  a.T = static_cast<int>(tokens);
  a.n_seqs = static_cast<int>(n_seqs);
  a.q = q, a.k = k, a.v = v;
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  CUtensorMap tq, tk, tv;
  if ((rc = q_map(&tq, q, q_st, q_sh, tokens, hkv, group, tok, d, dtype)) != XDNA_OK ||
      (rc = kv_map(&tk, k, k_st, k_sh, tokens, hkv, d, dtype)) != XDNA_OK ||
      (rc = kv_map(&tv, v, v_st, v_sh, tokens, hkv, d, dtype)) != XDNA_OK)
    return rc;
  const int64_t pairs = plan_pairs(n_seqs, tokens, group);
  if (n_seqs > kPlanFree) {
    XDNA_CHECK_ARG(workspace && aligned16(workspace) &&
                       workspace_bytes >= xdna_packed_attention_workspace(n_seqs, tokens, hq, hkv),
                   "packed_attention: workspace too small or unaligned");
    auto* plan = static_cast<PlanHeader*>(workspace);
    packed_plan_kernel<<<1, kPlanThreads, 0, s>>>(cu_seqlens, static_cast<int>(n_seqs), a.T, static_cast<int>(2 * tok), plan);
    if ((rc = check_launch("packed_plan_kernel")) != XDNA_OK) return rc;
    a.plan = plan;
  }
  XDNA_CHECK_ARG(pairs < (1ll << 31) / hkv, "packed_attention: bad sizes");
  return launch_tiles<PACKED>(tq, tk, tv, a, d, dtype, static_cast<int>(std::min<int64_t>(pairs * hkv, sms)), s);
}

size_t xdna_prefix_attention_workspace(int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d) {
  if (B < 1 || P < 0 || S < 0 || hkv < 1 || hq < hkv || hq / hkv > 128) return 0;
  int sms = 0;
  if (check_device(&sms) != XDNA_OK) return 0;
  return static_cast<size_t>(PrefixSplit(B, P, S, hq, hkv, d, sms).all() * B * hq) * (sizeof(float2) + d * sizeof(float));
}

int xdna_prefix_attention(const void* q, int64_t q_sb, int64_t q_sh, const void* pk, int64_t pk_st, int64_t pk_sh,
                          const void* pv, int64_t pv_st, int64_t pv_sh, const void* ck, int64_t ck_sb, int64_t ck_st,
                          int64_t ck_sh, const void* cv, int64_t cv_sb, int64_t cv_st, int64_t cv_sh,
                          const int32_t* lens, int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d,
                          int dtype, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_heads("prefix_attention", hq, hkv, d, dtype, scale);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(B >= 0 && P >= 0 && S >= 0 && B < (1ll << 24) / hq && P < (1ll << 30) && S < (1ll << 30),
                 "prefix_attention: bad sizes");
  int sms = 0;
  if ((rc = check_device(&sms)) != XDNA_OK) return rc;
  if (B == 0) return XDNA_OK;
  XDNA_CHECK_ARG(row_ok(q, q_sb, q_sh) && (P == 0 || (row_ok(pk, pk_st, pk_sh) && row_ok(pv, pv_st, pv_sh))) &&
                     (S == 0 || (row_ok(ck, ck_sb, ck_st, ck_sh) && row_ok(cv, cv_sb, cv_st, cv_sh))) && lens && out &&
                     aligned16(out),
                 "prefix_attention: operands must be 16-byte aligned with strides that are positive multiples of 8");
  const size_t need = xdna_prefix_attention_workspace(B, P, S, hq, hkv, d);
  XDNA_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
                 "prefix_attention: workspace too small or unaligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t group = hq / hkv, tok = 128 / group;
  const PrefixSplit split(B, P, S, hq, hkv, d, sms);
  float* part_o = static_cast<float*>(workspace);
  float2* part_ml = reinterpret_cast<float2*>(part_o + split.all() * B * hq * d);
  if (split.parts > 0) {
    TileArgs a{};
    a.hq = static_cast<int>(hq);
    a.hkv = static_cast<int>(hkv);
    a.group = static_cast<int>(group);
    a.tok = static_cast<int>(tok);
    a.scale_log2 = scale * kLog2E;
    a.err = device_error_word();
    a.B = static_cast<int>(B);
    a.P = static_cast<int>(P);
    a.pairs = static_cast<int>(split.pairs);
    a.splits = static_cast<int>(split.parts);
    a.blocks_per_split = static_cast<int>(split.blocks_per_part);
    a.part_o = part_o;
    a.part_ml = part_ml;
    CUtensorMap tq, tk, tv;
    if ((rc = q_map(&tq, q, q_sb, q_sh, B, hkv, group, tok, d, dtype)) != XDNA_OK ||
        (rc = kv_map(&tk, pk, pk_st, pk_sh, P, hkv, d, dtype)) != XDNA_OK ||
        (rc = kv_map(&tv, pv, pv_st, pv_sh, P, hkv, d, dtype)) != XDNA_OK)
      return rc;
    const int64_t items = split.pairs * hkv * split.parts;
    if ((rc = launch_tiles<PREFIX>(tq, tk, tv, a, d, dtype, static_cast<int>(std::min<int64_t>(items, sms)), s)) != XDNA_OK)
      return rc;
  }
  OwnArgs o{};
  o.q = q, o.ck = ck, o.cv = cv;
  o.q_sb = q_sb, o.q_sh = q_sh;
  o.ck_sb = ck_sb, o.ck_st = ck_st, o.ck_sh = ck_sh, o.cv_sb = cv_sb, o.cv_st = cv_st, o.cv_sh = cv_sh;
  if (split.direct) {
    o.P = static_cast<int>(P);
    o.pk = pk, o.pv = pv;
    o.pk_st = pk_st, o.pk_sh = pk_sh, o.pv_st = pv_st, o.pv_sh = pv_sh;
  }
  o.lens = lens;
  o.B = static_cast<int>(B);
  o.S = static_cast<int>(S);
  o.hq = static_cast<int>(hq);
  o.hkv = static_cast<int>(hkv);
  o.group = static_cast<int>(group);
  o.parts = static_cast<int>(split.parts);
  o.splits = static_cast<int>(split.own);
  o.scale_log2 = scale * kLog2E;
  o.part_o = part_o;
  o.part_ml = part_ml;
  o.out = out;
  if (dtype == XDNA_BF16) return d == 128 ? launch_own<__nv_bfloat16, 128>(o, s) : launch_own<__nv_bfloat16, 64>(o, s);
  return d == 128 ? launch_own<__half, 128>(o, s) : launch_own<__half, 64>(o, s);
}

}  // extern "C"
