// One head of one token, spread over the lanes of a part of a warp, with its norm and its rotation.
//
//   u = x / sqrt(mean of x^2 over the head + eps) * w      (w: the norm's weights; without them u = x)
//   pairs p = 0 .. R / 2 - 1 of u's first R entries, (p, p + R / 2) or interleaved (2 p, 2 p + 1), turned by
//   the angle position * inv_freq[p]:   (a cos - b sin, b cos + a sin) * factor;   the entries from R on stay.
//
// A lane has V first and V second entries of pairs (of the entries past R: 2 V that follow one another), so that no
// value crosses lanes; with interleaved pairs these are 2 V neighbouring entries.
#pragma once

#include "values.cuh"

namespace xdna {

// N values of T as they are; loads and stores take addresses aligned to the smaller of N * sizeof(T) and 16 bytes.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * static_cast<int>(sizeof(T));
  uint32_t w[kBytes >= 4 ? kBytes / 4 : 1];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> x;
  if constexpr (Pack<T, N>::kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < Pack<T, N>::kBytes / 16; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      x.w[4 * i] = u.x, x.w[4 * i + 1] = u.y, x.w[4 * i + 2] = u.z, x.w[4 * i + 3] = u.w;
    }
  } else if constexpr (Pack<T, N>::kBytes == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    x.w[0] = u.x, x.w[1] = u.y;
  } else if constexpr (Pack<T, N>::kBytes == 4) {
    x.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    x.w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  if constexpr (Pack<T, N>::kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < Pack<T, N>::kBytes / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(x.w[4 * i], x.w[4 * i + 1], x.w[4 * i + 2], x.w[4 * i + 3]);
  } else if constexpr (Pack<T, N>::kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(x.w[0], x.w[1]);
  } else if constexpr (Pack<T, N>::kBytes == 4) {
    *reinterpret_cast<uint32_t*>(p) = x.w[0];
  } else {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(x.w[0]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void to_floats(const Pack<T, N>& u, float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(u.w[i]);
    } else if constexpr (__is_same(T, __half)) {
      const uint16_t h = static_cast<uint16_t>(u.w[i / 2] >> (16 * (i & 1)));
      x[i] = __half2float(*reinterpret_cast<const __half*>(&h));
    } else {
      x[i] = __uint_as_float(i & 1 ? u.w[i / 2] & 0xffff0000u : u.w[i / 2] << 16);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> from_floats(const float* x) {
  Pack<T, N> u;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) u.w[i] = __float_as_uint(x[i]);
  } else if constexpr (N == 1) {
    u.w[0] = pack2<T>(x[0], 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) u.w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  }
  return u;
}

// N weights from place `at` on as floats, of any of the three types.
template <int N>
__device__ __forceinline__ void load_weights(const void* w, int dtype, int64_t at, float* x) {
  if (dtype == XDNA_F32)
    to_floats<float, N>(load_pack<float, N>(static_cast<const float*>(w) + at), x);
  else if (dtype == XDNA_BF16)
    to_floats<__nv_bfloat16, N>(load_pack<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(w) + at), x);
  else
    to_floats<__half, N>(load_pack<__half, N>(static_cast<const __half*>(w) + at), x);
}

// Angles in turns, as 64-bit fractions: a frequency's turns per position, to 2^-64 (1 / (2 pi) in two parts, and the first
// product's rounding), times the position leaves the part within a turn, off by no more than position * 2^-64: 2^-24 radians
// at 2^37. cos and sin of it, times factor: of its upper 24 bits in 32 bits, turned on by what is left (below 2^-24 of half a
// turn, so to first order).
__device__ __forceinline__ uint64_t turns_of(float inv_freq) {
  constexpr double kHigh = 0.15915494309189535, kLow = -9.839338337591243e-18;
  const double f = inv_freq, turns = __dmul_rn(f, kHigh), rest = fma(f, kLow, fma(f, kHigh, -turns));
  return static_cast<uint64_t>(__double2ll_rn((turns - rint(turns)) * 18446744073709551616.0)) +
         static_cast<uint64_t>(__double2ll_rn(rest * 18446744073709551616.0));
}
__device__ __forceinline__ float2 turn_of(uint64_t turns, float factor) {
  const int32_t high = static_cast<int32_t>(turns >> 32), upper = high & ~0xff;
  float s, c;
  sincospif(static_cast<float>(upper) * 4.656612873e-10f, &s, &c);  // 2^-31: half turns
  const float rest = (static_cast<float>(high & 0xff) + 0.5f) * 1.4629180792671596e-9f;  // to 2^-32, times pi 2^-31
  return make_float2(fmaf(-s, rest, c) * factor, fmaf(c, rest, s) * factor);
}

// Where a lane's unit j of a head lies and which of its pairs turn: V entries from lo and V from hi on, pairs
// V j .. V j + turning - 1. n_freq = R / 2, a multiple of V where pairs are not interleaved.
struct UnitAt {
  int lo, hi, turning;
};
template <int V, bool INTER>
__device__ __forceinline__ UnitAt unit_at(int j, int n_freq) {
  const int turning = min(max(n_freq - V * j, 0), V);
  if (!INTER && turning > 0) return {V * j, V * j + n_freq, V};
  return {2 * V * j, 2 * V * j + V, turning};
}

// x: the unit's 2 V values, first those of lo, then those of hi. Pairs that are not interleaved turn all or none, two at a
// time.
template <int V, bool INTER>
__device__ __forceinline__ void turn_unit(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], int turning) {
  if (!INTER && turning == 0) return;
  if constexpr (INTER || V == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float &a = x[INTER ? 2 * i : i], &b = x[INTER ? 2 * i + 1 : i + V];
      if (!INTER || i < turning) {
        const float t = fmaf(a, c[i], -b * s[i]);
        b = fmaf(b, c[i], a * s[i]);
        a = t;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 a = make_float2(x[i], x[i + 1]), b = make_float2(x[i + V], x[i + 1 + V]);
      const float2 cc = make_float2(c[i], c[i + 1]), ss = make_float2(s[i], s[i + 1]), minus = make_float2(-s[i], -s[i + 1]);
      const float2 t = __ffma2_rn(a, cc, __fmul2_rn(b, minus)), y = __ffma2_rn(b, cc, __fmul2_rn(a, ss));
      x[i] = t.x, x[i + 1] = t.y, x[i + V] = y.x, x[i + 1 + V] = y.y;
    }
  }
}

// x *= by * w, and the sum of squares. (Two at a time, as in turn_unit, the registers cost more than the instructions saved:
// cache_append of 12968 tokens 40.7 us instead of 32.3.)
template <int N>
__device__ __forceinline__ void scale_by(float* x, float by, const float* w) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] *= by * w[i];
}
template <int N>
__device__ __forceinline__ float squares(const float* x) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
  return s;
}

// 1 / sqrt(x): rsqrtf (2 ulp) and one step of Newton's method, y + y / 2 * (1 - x y^2), which leaves about one ulp.
__device__ __forceinline__ float inverse_root(float x) {
  const float y = rsqrtf(x);
  return x > 1e-37f && x < 3e38f ? fmaf(0.5f * y, fmaf(-x * y, y, 1.f), y) : y;
}

// The sum over LANES neighbouring lanes, from a multiple of LANES on, on all of them. All lanes of the warp.
template <int LANES>
__device__ __forceinline__ float sum_of_lanes(float x) {
  if constexpr ((LANES & (LANES - 1)) == 0) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  } else {
    const int first = lane_id() / LANES * LANES;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < LANES; ++i) sum += __shfl_sync(0xffffffffu, x, (first + i) & 31);
    return sum;
  }
}

}  // namespace xdna
