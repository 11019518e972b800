// What lies between the products of a decoder layer: rotary positions (with the norm of queries and keys before them)
// and the norms around a block.
#include <algorithm>
#include <type_traits>

#include "host_util.h"
#include "rotary.cuh"
#include "rotary.h"

namespace xdna {

constexpr int kRotaryWarps = 4;

// A warp has one token (wpt > 1: one of the wpt warps that share a token) and goes over its heads, 32 / LANES at a time; the
// next heads are asked for before those at hand are worked on, and the first ones before the angles are known. The token's
// cosines and sines are worked out once, each by one lane, and handed round by shuffles; they then stay in registers. U
// units of 2 V values per lane, U > 1 with V = 1 alone.
// 16384 tokens of 24 heads of 128 in bf16 with norms of their own: 43.6 us, 4.6 TB/s (37.9 without the norm; 8192 in f32,
// the same bytes: 38.5). 70 % of the issue slots are busy, 270 to 320 instructions for four heads of a token, of which the
// norm, the turn and the 16-bit values take about 150; the norms' weights come through L1 for each token; and the 72
// registers of seven blocks spill 8 to 28 bytes a thread in the 8-wide variants of 16 bits, 36 to 56 in those of f32.
// Blocks of four warps, seven to an SM; of eight: 45.6 us; two rounds asked for ahead: 52, three: 51 (registers); several
// tokens per warp, so that the start of one hides behind another: 47.
template <typename T, int V, int LANES, int U, bool INTER>
__global__ void __launch_bounds__(kRotaryWarps * 32, 7) rotary_kernel(const RotaryArgs a) {
  static_assert(U == 1 || (V == 1 && LANES == 32), "more units only where a lane has all of a warp's row");
  // heads of a round (32 % LANES lanes are left over), angles of a lane
  constexpr int kRows = 32 / LANES, kPer = (V + kRows - 1) / kRows;
  const int lane = lane_id(), r = lane / LANES, j0 = lane % LANES;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kRotaryWarps + warp_id(), token = w / a.wpt;
  if (token >= a.T) return;
  const T* x = static_cast<const T*>(a.x) + token * a.x_st;
  T* out = static_cast<T*>(a.out) + token * a.H * a.D;
  const int units = r < kRows ? a.D / (2 * V) : 0, stride = a.wpt * kRows;
  UnitAt u[U];
#pragma unroll
  for (int k = 0; k < U; ++k) u[k] = unit_at<V, INTER>(j0 + k * LANES, a.n_freq);
  Pack<T, V> later[U][2];
  auto load = [&](int h) {
    const T* p = x + h * a.x_sh;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      later[k][0] = later[k][1] = Pack<T, V>{};
      if (h < a.H && j0 + k * LANES < units) later[k][0] = load_pack<T, V>(p + u[k].lo), later[k][1] = load_pack<T, V>(p + u[k].hi);
    }
  };
  const float inv_d = 1.f / static_cast<float>(a.D);
  int h = static_cast<int>(w % a.wpt) * kRows + r;
  load(h);
  const Place at = place_of(a, token);
  float cos_[U][V], sin_[U][V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float2 mine[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = (j0 + k * LANES) * V + r * kPer + i;
      mine[i] = p < a.n_freq ? turn_of(turns_of(a.inv_freq[p]) * static_cast<uint64_t>(at.position), a.factor) : make_float2(1.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int src = (i / kPer) * LANES + j0;
      cos_[k][i] = __shfl_sync(0xffffffffu, mine[i % kPer].x, src);
      sin_[k][i] = __shfl_sync(0xffffffffu, mine[i % kPer].y, src);
    }
  }
  for (; h - r < a.H; h += stride) {
    float f[U][2 * V];
#pragma unroll
    for (int k = 0; k < U; ++k) to_floats<T, V>(later[k][0], f[k]), to_floats<T, V>(later[k][1], f[k] + V);
    load(h + stride);
    float inv = 1.f;
    if (a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < U; ++k) ss += squares<2 * V>(f[k]);
      inv = inverse_root(fmaf(sum_of_lanes<LANES>(ss), inv_d, a.eps));
    }
    if (h >= a.H) continue;
    T* p = out + static_cast<int64_t>(h) * a.D;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (j0 + k * LANES >= units) continue;
      if (a.norm) {
        float g[2 * V];
        load_weights<V>(a.norm, a.norm_dtype, h * a.norm_sh + u[k].lo, g);
        load_weights<V>(a.norm, a.norm_dtype, h * a.norm_sh + u[k].hi, g + V);
        scale_by<2 * V>(f[k], inv, g);
      }
      turn_unit<V, INTER>(f[k], cos_[k], sin_[k], u[k].turning);
      store_pack<T, V>(p + u[k].lo, at.there ? from_floats<T, V>(f[k]) : Pack<T, V>{});
      store_pack<T, V>(p + u[k].hi, at.there ? from_floats<T, V>(f[k] + V) : Pack<T, V>{});
    }
  }
}

template <typename T, int V, int LANES, int U, bool INTER>
static int launch_rotary_as(RotaryArgs a, int sms, cudaStream_t s) {
  // warps of a token: more than one where there are too few tokens to fill the SMs, up to one for each of its rounds
  constexpr int kRows = 32 / LANES;
  a.wpt = 1;
  while (a.wpt < 8 && a.T * a.wpt < 32 * sms && a.wpt * kRows < a.H) a.wpt *= 2;
  const int64_t blocks = (a.T * a.wpt + kRotaryWarps - 1) / kRotaryWarps;
  rotary_kernel<T, V, LANES, U, INTER><<<static_cast<unsigned>(blocks), kRotaryWarps * 32, 0, s>>>(a);
  return check_launch("rotary_kernel");
}

template <typename T, bool INTER>
static int launch_rotary_t(const RotaryArgs& a, int sms, cudaStream_t s) {
  // the widest loads that keep both entries of a pair on one lane, and as many heads to a round as their lanes let in. 24
  // heads of 64, 80 and 96 with eight lanes each, as 128 has, took 39.0, 40.8 and 41.8 us; with four, five and six 25.1, 34.6
  // and 39.9
  if (a.D % 16 == 0 && (INTER || a.n_freq % 8 == 0)) {
    if (a.D <= 64) return launch_rotary_as<T, 8, 4, 1, INTER>(a, sms, s);
    if (a.D == 80) return launch_rotary_as<T, 8, 5, 1, INTER>(a, sms, s);
    if (a.D == 96) return launch_rotary_as<T, 8, 6, 1, INTER>(a, sms, s);
    return a.D <= 128 ? launch_rotary_as<T, 8, 8, 1, INTER>(a, sms, s) : launch_rotary_as<T, 8, 16, 1, INTER>(a, sms, s);
  }
  if (INTER || a.n_freq % 4 == 0)
    return a.D <= 128 ? launch_rotary_as<T, 4, 16, 1, INTER>(a, sms, s) : launch_rotary_as<T, 4, 32, 1, INTER>(a, sms, s);
  if constexpr (!INTER) return launch_rotary_as<T, 1, 32, 4, false>(a, sms, s);
  return XDNA_OK;
}

int launch_rotary(const RotaryArgs& a, int dtype, bool interleaved, int sms, cudaStream_t s) {
  if (a.T == 0 || a.H == 0) return XDNA_OK;
  switch (dtype) {
    case XDNA_F32:
      return interleaved ? launch_rotary_t<float, true>(a, sms, s) : launch_rotary_t<float, false>(a, sms, s);
    case XDNA_BF16:
      return interleaved ? launch_rotary_t<__nv_bfloat16, true>(a, sms, s) : launch_rotary_t<__nv_bfloat16, false>(a, sms, s);
    default:
      return interleaved ? launch_rotary_t<__half, true>(a, sms, s) : launch_rotary_t<__half, false>(a, sms, s);
  }
}

// ---------------------------------------------------------------------------- norms around a block
//   z = post ? y / sqrt(mean y^2 + eps) * post : y;   x' = x + scale * gate * z;   h = x' / sqrt(mean x'^2 + eps) * weight
struct AddNormArgs {
  const void *x, *y;
  int64_t ldx, ldy;
  const void *weight, *post, *gate;
  int weight_dtype, post_dtype, gate_dtype;
  int64_t ld_gate;  // 0: one for all rows
  float scale, eps;
  void *x_out, *h;
  int64_t rows;
  int D;
};

// Sums over a row's threads (threadIdx.x of blockDim.x); the barrier also ends the reading of an earlier sum.
__device__ __forceinline__ float sum_of_row(float x, float* parts) {
  x = sum_of_lanes<32>(x);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return x;
  if (lane_id() == 0) parts[warp_id()] = x;
  __syncthreads();
  x = lane_id() < warps ? parts[lane_id()] : 0.f;
  return sum_of_lanes<32>(x);
}

// Eight weights from place `at` on, which need not be a multiple of eight (the same remainder for the whole row): whole
// pieces around them, shifted in registers. n: weights in all; 0 <= at, at + 8 <= n.
__device__ __forceinline__ void load_shifted(const void* w, int dtype, int at, int n, float (&x)[8]) {
  if (dtype == XDNA_F32) {
    const int r = at & 3, from = at - r;
    const float* p = static_cast<const float*>(w) + from;
    float y[12];
    if (from + 12 <= n) {
      to_floats<float, 12>(load_pack<float, 12>(p), y);
    } else {
#pragma unroll
      for (int i = 0; i < 12; ++i) y[i] = from + i < n ? p[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 10; ++i) y[i] = r & 2 ? y[i + 2] : y[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r & 1 ? y[i + 1] : y[i];
  } else {
    const int r = at & 7, from = at - r;
    const uint16_t* p = static_cast<const uint16_t*>(w) + from;
    Pack<__half, 16> u;
    if (from + 16 <= n) {
      u = load_pack<__half, 16>(reinterpret_cast<const __half*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        u.w[i] = (from + 2 * i < n ? p[2 * i] : 0u) | (from + 2 * i + 1 < n ? static_cast<uint32_t>(p[2 * i + 1]) << 16 : 0u);
    }
#pragma unroll
    for (int i = 0; i < 6; ++i) u.w[i] = r & 4 ? u.w[i + 2] : u.w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) u.w[i] = r & 2 ? u.w[i + 1] : u.w[i];
    Pack<__half, 8> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = __funnelshift_r(u.w[i], u.w[i + 1], r & 1 ? 16 : 0);
    if (dtype == XDNA_F16)
      to_floats<__half, 8>(v, x);
    else
      to_floats<__nv_bfloat16, 8>(*reinterpret_cast<const Pack<__nv_bfloat16, 8>*>(&v), x);
  }
}

// A row lies in the registers of blockDim.x threads, C pieces of V values each, and is read and written once; with one
// warp to a row, blockDim.y rows to a block. SHIFT: rows whose length is no multiple of V, in arrays that start at a
// boundary of 16 bytes and whose pitches leave the same remainder. Pieces then begin at boundaries, `shift` entries before
// the row's, and its ends are taken entry by entry. 8191 rows of 5003 in bf16 with a norm behind the block and a gate of
// their own: 111 us (3.7 TB/s); entry by entry 436. Rows of 4096: 57.2 us (5.9 TB/s); with the gate in f32, which is read
// behind the first sum, 74.7 (5.4). The inverse roots are rsqrtf's, off by 2 ulp at most, which is less than the
// sums of a row's squares are off by.
template <typename TX, typename TY, int V, int C, bool SHIFT>
__global__ void __launch_bounds__(1024) add_norm_kernel(const AddNormArgs a) {
  __shared__ float parts[2][32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // a whole warp; blocks of several warps to a row have one row
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TY* y = static_cast<const TY*>(a.y) + row * a.ldy;
  TX* x_out = static_cast<TX*>(a.x_out) + row * a.D;
  TY* h = static_cast<TY*>(a.h) + row * a.D;
  const int shift = SHIFT ? static_cast<int>(row * a.D % V) : 0;
  const int step = blockDim.x * V, first = static_cast<int>(threadIdx.x) * V - shift;
  auto whole = [&](int at) { return SHIFT ? at >= 0 && at + V <= a.D : at < a.D; };
  auto any = [&](int at) { return at + V > 0 && at < a.D; };  // SHIFT: the ends
  // V values of a row's array, or of weights, from `at` on; zeros where there are none
  auto row_values = [&](auto* p, int at, float (&f)[V]) {
    using E = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
    if (whole(at)) {
      to_floats<E, V>(load_pack<E, V>(p + at), f);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = 0.f;
        if (SHIFT && at + i >= 0 && at + i < a.D) to_floats<E, 1>(load_pack<E, 1>(p + at + i), f + i);
      }
    }
  };
  auto weights = [&](const void* w, int dtype, int at, float (&f)[V]) {
    if constexpr (SHIFT) {
      if (whole(at)) {
        load_shifted(w, dtype, at, a.D, f);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          f[i] = 0.f;
          if (at + i >= 0 && at + i < a.D) load_weights<1>(w, dtype, at + i, f + i);
        }
      }
    } else {
      load_weights<V>(w, dtype, at, f);
    }
  };
  auto store = [&](auto* p, int at, const float (&f)[V]) {
    using E = std::remove_reference_t<decltype(*p)>;
    if (whole(at)) {
      store_pack<E, V>(p + at, from_floats<E, V>(f));
    } else if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at + i >= 0 && at + i < a.D) store_pack<E, 1>(p + at + i, from_floats<E, 1>(f + i));
    }
  };
  Pack<TX, V> rx[C];
  Pack<TY, V> ry[C];
  // a gate of 16 bits for each entry, with the others, not behind the first sum
  const bool gated = V == 8 && a.gate && a.ld_gate > 0 && a.gate_dtype != XDNA_F32;
  Pack<__half, V> rg[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    rx[c] = Pack<TX, V>{};
    ry[c] = Pack<TY, V>{};
    rg[c] = Pack<__half, V>{};
    if (whole(at)) {
      ry[c] = load_pack<TY, V>(y + at);
      rx[c] = load_pack<TX, V>(x + at);
      if (gated) rg[c] = load_pack<__half, V>(static_cast<const __half*>(a.gate) + row * a.ld_gate + at);
    } else if constexpr (SHIFT) {
      if (any(at)) {
        float f[V];
        row_values(y, at, f);
        ry[c] = from_floats<TY, V>(f);  // exact
        row_values(x, at, f);
        rx[c] = from_floats<TX, V>(f);
      }
    }
  }
  float by = a.scale;
  const float inv_d = 1.f / static_cast<float>(a.D);
  if (a.post) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f[V];
      to_floats<TY, V>(ry[c], f);
      ss += squares<V>(f);
    }
    by *= rsqrtf(sum_of_row(ss, parts[0]) * inv_d + a.eps);
  }
  float z[C][V], ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    to_floats<TX, V>(rx[c], z[c]);
    if (!(SHIFT ? any(at) : whole(at))) continue;
    float f[V], g[V];
    to_floats<TY, V>(ry[c], f);
    if (a.post) {
      weights(a.post, a.post_dtype, at, g);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= g[i];
    }
    if (gated && whole(at)) {
      if (a.gate_dtype == XDNA_F16)
        to_floats<__half, V>(rg[c], g);
      else
        to_floats<__nv_bfloat16, V>(*reinterpret_cast<const Pack<__nv_bfloat16, V>*>(&rg[c]), g);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= g[i];
    } else if (a.gate) {
      if (SHIFT && a.ld_gate > 0) {
        if (a.gate_dtype == XDNA_F32)
          row_values(static_cast<const float*>(a.gate) + row * a.ld_gate, at, g);
        else if (a.gate_dtype == XDNA_BF16)
          row_values(static_cast<const __nv_bfloat16*>(a.gate) + row * a.ld_gate, at, g);
        else
          row_values(static_cast<const __half*>(a.gate) + row * a.ld_gate, at, g);
      } else if constexpr (SHIFT) {
        weights(a.gate, a.gate_dtype, at, g);
      } else {
        load_weights<V>(a.gate, a.gate_dtype, row * a.ld_gate + at, g);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) z[c][i] = fmaf(f[i], by, z[c][i]);
    store(x_out, at, z[c]);
    ss += squares<V>(z[c]);
  }
  const float inv = rsqrtf(sum_of_row(ss, parts[1]) * inv_d + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    if (!(SHIFT ? any(at) : whole(at))) continue;
    float g[V];
    weights(a.weight, a.weight_dtype, at, g);
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] *= z[c][i] * inv;
    store(h, at, g);
  }
}

constexpr int kNormMost = 16384;  // entries of a row: 1024 threads of 16

template <typename TX, typename TY, int V, int C, bool SHIFT>
static int launch_add_norm_as(const AddNormArgs& a, cudaStream_t s) {
  const int entries = a.D + (SHIFT ? V - 1 : 0), threads = (entries + V * C * 32 - 1) / (V * C * 32) * 32, rows = threads == 32 ? 4 : 1;
  add_norm_kernel<TX, TY, V, C, SHIFT><<<static_cast<unsigned>((a.rows + rows - 1) / rows), dim3(threads, rows), 0, s>>>(a);
  return check_launch("add_norm_kernel");
}

enum { NORM_SINGLE, NORM_SHIFT, NORM_WIDE };  // how rows lie: anyhow, with the same remainders, at boundaries of 16 bytes

template <typename TX, typename TY>
static int launch_add_norm(const AddNormArgs& a, int lie, int sms, cudaStream_t s) {
  // few rows: one piece per thread, for the latency; many: two, so that more is under way. 8191 rows of 4096 in bf16 with a
  // gate of their own: 75.9 us with one, 65.8 with two, 67.8 with four.
  if (lie == NORM_WIDE)
    return a.rows < 2 * sms && a.D <= 8 * 1024 ? launch_add_norm_as<TX, TY, 8, 1, false>(a, s) : launch_add_norm_as<TX, TY, 8, 2, false>(a, s);
  if (lie == NORM_SHIFT && a.D <= kNormMost - 8) return launch_add_norm_as<TX, TY, 8, 2, true>(a, s);
  return a.D <= 4 * 1024 ? launch_add_norm_as<TX, TY, 1, 4, false>(a, s) : launch_add_norm_as<TX, TY, 1, 16, false>(a, s);
}

template <typename TX>
static int launch_add_norm(const AddNormArgs& a, int y_dtype, int lie, int sms, cudaStream_t s) {
  if (y_dtype == XDNA_F32) return launch_add_norm<TX, float>(a, lie, sms, s);
  if (y_dtype == XDNA_BF16) return launch_add_norm<TX, __nv_bfloat16>(a, lie, sms, s);
  return launch_add_norm<TX, __half>(a, lie, sms, s);
}

}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_rotary(const void* x, int dtype, int64_t T, int64_t H, int64_t D, int64_t x_st, int64_t x_sh,
                const void* positions, int position_bytes, const float* inv_freq, int64_t n_freq, float factor,
                int interleaved, const void* norm, int norm_dtype, int64_t norm_sh, float eps, void* out, void* stream) {
  XDNA_CHECK_ARG(T >= 0 && H >= 0 && T < (1ll << 31) && H < (1ll << 20), "rotary: bad sizes");
  XDNA_CHECK_ARG(is_float_dtype(dtype), "rotary: f32, bf16 or f16");
  if (D < 8 || D > 256 || D % 8 != 0)
    return fail(XDNA_ERR_UNSUPPORTED, "rotary: head dimension %lld (multiples of 8 up to 256)", (long long)D);
  XDNA_CHECK_ARG(n_freq >= 0 && 2 * n_freq <= D, "rotary: %lld frequencies for heads of %lld", (long long)n_freq, (long long)D);
  XDNA_CHECK_ARG(position_bytes == 4 || position_bytes == 8, "rotary: 32 or 64-bit positions");
  int sms = 0;
  int rc = check_device(&sms);
  if (rc != XDNA_OK) return rc;
  if (T == 0 || H == 0) return XDNA_OK;
  XDNA_CHECK_ARG(x && out && positions && (n_freq == 0 || inv_freq) && aligned16(x) && aligned16(out) && x_st > 0 && x_sh > 0 &&
                     x_st % 8 == 0 && x_sh % 8 == 0,
                 "rotary: null pointer, unaligned rows or bad strides");
  XDNA_CHECK_ARG(norm == nullptr || (is_float_dtype(norm_dtype) && norm_sh >= 0 && norm_sh % 8 == 0 && aligned16(norm)),
                 "rotary: the norm's weights are f32, bf16 or f16, aligned");
  RotaryArgs a{};
  a.x = x, a.out = out, a.x_st = x_st, a.x_sh = x_sh;
  a.positions = positions, a.position_bytes = position_bytes;
  a.inv_freq = inv_freq, a.n_freq = static_cast<int>(n_freq), a.factor = factor;
  a.norm = norm, a.norm_dtype = norm_dtype, a.norm_sh = norm_sh, a.eps = eps;
  a.T = T, a.H = static_cast<int>(H), a.D = static_cast<int>(D);
  return launch_rotary(a, dtype, interleaved != 0, sms, static_cast<cudaStream_t>(stream));
}

int xdna_add_norm(const void* x, int x_dtype, int64_t ldx, const void* y, int y_dtype, int64_t ldy, int64_t rows,
                  int64_t D, const void* weight, int weight_dtype, const void* post, int post_dtype, const void* gate,
                  int gate_dtype, int64_t ld_gate, float scale, float eps, void* x_out, void* h, void* stream) {
  XDNA_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "add_norm: bad sizes");
  if (D < 1 || D > kNormMost)
    return fail(XDNA_ERR_UNSUPPORTED, "add_norm: rows of %lld entries (1 to %d)", (long long)D, kNormMost);
  XDNA_CHECK_ARG(is_float_dtype(x_dtype) && is_float_dtype(y_dtype), "add_norm: f32, bf16 or f16");
  int sms = 0;
  int rc = check_device(&sms);
  if (rc != XDNA_OK) return rc;
  if (rows == 0) return XDNA_OK;
  XDNA_CHECK_ARG(x && y && weight && x_out && h && is_float_dtype(weight_dtype) && (!post || is_float_dtype(post_dtype)) &&
                     (!gate || (is_float_dtype(gate_dtype) && ld_gate >= 0)) && ldx >= 0 && ldy >= 0,
                 "add_norm: null pointer, bad type or pitch");
  const AddNormArgs a{x, y, ldx, ldy, weight, post, gate, weight_dtype, post_dtype, gate_dtype, ld_gate, scale, eps, x_out, h,
                      rows, static_cast<int>(D)};
  bool aligned = true;
  for (const void* p : {x, y, weight, post, gate, static_cast<const void*>(x_out), static_cast<const void*>(h)}) aligned = aligned && aligned16(p);
  const bool alike = aligned && ldx % 8 == D % 8 && ldy % 8 == D % 8 && (!gate || ld_gate == 0 || ld_gate % 8 == D % 8);
  const int lie = !alike ? NORM_SINGLE : D % 8 == 0 ? NORM_WIDE : NORM_SHIFT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == XDNA_F32) return launch_add_norm<float>(a, y_dtype, lie, sms, s);
  if (x_dtype == XDNA_BF16) return launch_add_norm<__nv_bfloat16>(a, y_dtype, lie, sms, s);
  return launch_add_norm<__half>(a, y_dtype, lie, sms, s);
}

}  // extern "C"
