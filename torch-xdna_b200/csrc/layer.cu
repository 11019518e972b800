// What lies between the products of a decoder layer: rotary positions (with the norm of queries and keys before them)
// and the norms around a block.
#include <algorithm>

#include "host_util.h"
#include "rotary.cuh"
#include "rotary.h"

namespace xdna {

constexpr int kRotaryWarps = 8;

// A warp has one token (wpt > 1: one of the wpt warps that share a token) and goes over its heads, 32 / LANES at a time.
// The token's cosines and sines are worked out once, each by one lane, and handed round by shuffles; they then stay in
// registers. U units of 2 V values per lane, U > 1 with V = 1 alone.
template <typename T, int V, int LANES, int U, bool INTER>
__global__ void __launch_bounds__(kRotaryWarps * 32) rotary_kernel(const RotaryArgs a) {
  static_assert(U == 1 || (V == 1 && LANES == 32), "more units only where a lane has all of a warp's row");
  constexpr int kRows = 32 / LANES, kAhead = U > 1 ? 1 : 2;  // heads of a warp at a time, of these under way
  const int lane = lane_id(), r = lane / LANES, j0 = lane % LANES;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kRotaryWarps + warp_id(), token = w / a.wpt;
  if (token >= a.T) return;
  const Place at = place_of(a, token);
  UnitAt u[U];
  float2 cs[U][V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    u[k] = unit_at<V, INTER>(j0 + k * LANES, a.n_freq);
    if constexpr (V >= kRows) {
      constexpr int kPer = V / kRows;  // angles of a lane
      float2 mine[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int p = (j0 + k * LANES) * V + r * kPer + i;
        mine[i] = p < a.n_freq ? turn_of(at.position, a.inv_freq[p], a.factor) : make_float2(1.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int src = (i / kPer) * LANES + j0;
        cs[k][i].x = __shfl_sync(0xffffffffu, mine[i % kPer].x, src);
        cs[k][i].y = __shfl_sync(0xffffffffu, mine[i % kPer].y, src);
      }
    }
  }
  const T* x = static_cast<const T*>(a.x) + token * a.x_st;
  T* out = static_cast<T*>(a.out) + token * a.H * a.D;
  const int units = a.D / (2 * V), stride = a.wpt * kRows;
  const int first = static_cast<int>(w % a.wpt) * kRows;
  for (int h0 = first; h0 < a.H; h0 += kAhead * stride) {
    Pack<T, V> raw[kAhead][U][2];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int h = h0 + n * stride + r;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (h < a.H && j0 + k * LANES < units) {
          const T* p = x + h * a.x_sh;
          raw[n][k][0] = load_pack<T, V>(p + u[k].lo), raw[n][k][1] = load_pack<T, V>(p + u[k].hi);
        } else {
          raw[n][k][0] = raw[n][k][1] = Pack<T, V>{};
        }
      }
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int h = h0 + n * stride + r;
      float f[U][2 * V];
#pragma unroll
      for (int k = 0; k < U; ++k) to_floats<T, V>(raw[n][k][0], f[k]), to_floats<T, V>(raw[n][k][1], f[k] + V);
      if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) ss = fmaf(f[k][i], f[k][i], ss);
        }
        ss = sum_of_lanes<LANES>(ss);
        const float inv = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (h < a.H && j0 + k * LANES < units) {
            float g[2 * V];
            load_weights<V>(a.norm, a.norm_dtype, h * a.norm_sh + u[k].lo, g);
            load_weights<V>(a.norm, a.norm_dtype, h * a.norm_sh + u[k].hi, g + V);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[k][i] *= inv * g[i];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (h >= a.H || j0 + k * LANES >= units) continue;
        turn_unit<V, INTER>(f[k], cs[k], u[k].turning);
        if (!at.there) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) f[k][i] = 0.f;
        }
        T* p = out + static_cast<int64_t>(h) * a.D;
        store_pack<T, V>(p + u[k].lo, from_floats<T, V>(f[k]));
        store_pack<T, V>(p + u[k].hi, from_floats<T, V>(f[k] + V));
      }
    }
  }
}

template <typename T, int V, int LANES, int U, bool INTER>
static int launch_rotary_as(RotaryArgs a, int sms, cudaStream_t s) {
  // warps of a token: more than one where there are too few tokens to fill the SMs, up to one for each of its rounds
  constexpr int kRows = 32 / LANES;
  a.wpt = 1;
  while (a.wpt < kRotaryWarps && a.T * a.wpt < 32 * sms && a.wpt * kRows < a.H) a.wpt *= 2;
  const int64_t blocks = (a.T * a.wpt + kRotaryWarps - 1) / kRotaryWarps;
  rotary_kernel<T, V, LANES, U, INTER><<<static_cast<unsigned>(blocks), kRotaryWarps * 32, 0, s>>>(a);
  return check_launch("rotary_kernel");
}

template <typename T, bool INTER>
static int launch_rotary_t(const RotaryArgs& a, int sms, cudaStream_t s) {
  // the widest loads that keep both entries of a pair on one lane
  if (a.D % 16 == 0 && (INTER || a.n_freq % 8 == 0))
    return a.D <= 128 ? launch_rotary_as<T, 8, 8, 1, INTER>(a, sms, s) : launch_rotary_as<T, 8, 16, 1, INTER>(a, sms, s);
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

// A row lies in the registers of blockDim.x threads, C pieces of V values each, and is read and written once; with one
// warp to a row, blockDim.y rows to a block.
template <typename TX, typename TY, int V, int C>
__global__ void __launch_bounds__(V == 8 && C == 4 ? 512 : 1024) add_norm_kernel(const AddNormArgs a) {
  __shared__ float parts[2][32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // a whole warp; blocks of several warps to a row have one row
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TY* y = static_cast<const TY*>(a.y) + row * a.ldy;
  const int step = blockDim.x * V, first = threadIdx.x * V;
  Pack<TX, V> rx[C];
  Pack<TY, V> ry[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    if (at < a.D) {
      ry[c] = load_pack<TY, V>(y + at);
      rx[c] = load_pack<TX, V>(x + at);
    } else {
      ry[c] = Pack<TY, V>{};
      rx[c] = Pack<TX, V>{};
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
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(f[i], f[i], ss);
    }
    by *= rsqrtf(sum_of_row(ss, parts[0]) * inv_d + a.eps);
  }
  float z[C][V], ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    to_floats<TX, V>(rx[c], z[c]);
    if (at < a.D) {
      float f[V], g[V];
      to_floats<TY, V>(ry[c], f);
      if (a.post) {
        load_weights<V>(a.post, a.post_dtype, at, g);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] *= g[i];
      }
      if (a.gate) {
        load_weights<V>(a.gate, a.gate_dtype, row * a.ld_gate + at, g);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) z[c][i] = fmaf(f[i], by, z[c][i]);
      store_pack<TX, V>(static_cast<TX*>(a.x_out) + row * a.D + at, from_floats<TX, V>(z[c]));
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(z[c][i], z[c][i], ss);
    }
  }
  const float inv = rsqrtf(sum_of_row(ss, parts[1]) * inv_d + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = first + c * step;
    if (at < a.D) {
      float g[V];
      load_weights<V>(a.weight, a.weight_dtype, at, g);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] *= z[c][i] * inv;
      store_pack<TY, V>(static_cast<TY*>(a.h) + row * a.D + at, from_floats<TY, V>(g));
    }
  }
}

constexpr int kNormMost = 16384;  // entries of a row: 512 threads of 32, or 1024 of 16

template <typename TX, typename TY, int V, int C>
static int launch_add_norm_as(const AddNormArgs& a, cudaStream_t s) {
  const int threads = (a.D + V * C * 32 - 1) / (V * C * 32) * 32, rows = threads == 32 ? 4 : 1;
  add_norm_kernel<TX, TY, V, C><<<static_cast<unsigned>((a.rows + rows - 1) / rows), dim3(threads, rows), 0, s>>>(a);
  return check_launch("add_norm_kernel");
}

template <typename TX, typename TY>
static int launch_add_norm(const AddNormArgs& a, bool wide, int sms, cudaStream_t s) {
  // few rows: short ones per thread, for the latency; many: as much under way per thread as its registers hold
  const bool few = a.rows < 2 * sms;
  if (wide) return few && a.D <= 8 * 1024 ? launch_add_norm_as<TX, TY, 8, 1>(a, s) : launch_add_norm_as<TX, TY, 8, 4>(a, s);
  return a.D <= 4 * 1024 ? launch_add_norm_as<TX, TY, 1, 4>(a, s) : launch_add_norm_as<TX, TY, 1, 16>(a, s);
}

template <typename TX>
static int launch_add_norm(const AddNormArgs& a, int y_dtype, bool wide, int sms, cudaStream_t s) {
  if (y_dtype == XDNA_F32) return launch_add_norm<TX, float>(a, wide, sms, s);
  if (y_dtype == XDNA_BF16) return launch_add_norm<TX, __nv_bfloat16>(a, wide, sms, s);
  return launch_add_norm<TX, __half>(a, wide, sms, s);
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
  // pieces of eight where every row starts on a boundary of 16 bytes
  bool wide = D % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && ld_gate % 8 == 0;
  for (const void* p : {x, y, weight, post, gate, static_cast<const void*>(x_out), static_cast<const void*>(h)}) wide = wide && aligned16(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == XDNA_F32) return launch_add_norm<float>(a, y_dtype, wide, sms, s);
  if (x_dtype == XDNA_BF16) return launch_add_norm<__nv_bfloat16>(a, y_dtype, wide, sms, s);
  return launch_add_norm<__half>(a, y_dtype, wide, sms, s);
}

}  // extern "C"
