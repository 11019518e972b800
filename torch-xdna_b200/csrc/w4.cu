// Linears with 4-bit weights and group scales for the few rows of a decode step:
//   y[m, n] = sum over groups g of s[n, g] * sum_{k in g} (c[n, k] - 8) x[m, k]  (+ bias[n]),  c in 0..15.
//
// Codes are stored in blocks of 128 columns (64 bytes, K padded with code 8 to whole blocks): the block's runs of
// eight columns r = 4 w + t lie as 32-bit words at place 4 t + w, and in a word the eight codes lie in the column
// order 0, 2, 4, 6, 1, 3, 5, 7 from the lowest bits.
#include "host_util.h"
#include "sm100.cuh"

namespace xdna {

constexpr int kW4Block = 128;

__device__ __forceinline__ float load_f32(const void* p, int dt, int64_t i) {
  if (dt == XDNA_F32) return static_cast<const float*>(p)[i];
  if (dt == XDNA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_f32(void* p, int dt, int64_t i, float x) {
  if (dt == XDNA_F32)
    static_cast<float*>(p)[i] = x;
  else if (dt == XDNA_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// bit position of column c (0..7) in its run's word
__host__ __device__ constexpr int w4_shift(int c) { return 4 * ((c >> 1) + 4 * (c & 1)); }

struct W4Args {
  const void* x;
  int64_t ldx;
  const uint8_t* codes;
  const void* scales;
  const void* bias;
  void* y;
  int64_t ldy, M, N, K, row_bytes, n_groups;
  int x_dtype, scale_dtype, bias_dtype, group;
};

// One warp per output: lane l takes the words l, l + 32, ... of the row.
__global__ void __launch_bounds__(256) w4_kernel(const W4Args a) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + warp_id(), m = blockIdx.y;
  if (n >= a.N) return;
  const uint32_t* row = reinterpret_cast<const uint32_t*>(a.codes + n * a.row_bytes);
  float acc = 0.f;
  for (int64_t i = lane_id(); i < a.row_bytes / 4; i += 32) {
    const int place = static_cast<int>(i & 15);
    const int64_t col = (i >> 4) * kW4Block + ((place & 3) * 4 + (place >> 2)) * 8;
    if (col >= a.K) continue;
    const uint32_t word = row[i];
    float part = 0.f;
    for (int c = 0; c < 8 && col + c < a.K; ++c)
      part += (static_cast<float>((word >> w4_shift(c)) & 15u) - 8.f) * load_f32(a.x, a.x_dtype, m * a.ldx + col + c);
    acc += part * load_f32(a.scales, a.scale_dtype, n * a.n_groups + col / a.group);
  }
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane_id() == 0) {
    if (a.bias) acc += load_f32(a.bias, a.bias_dtype, n);
    store_f32(a.y, a.x_dtype, m * a.ldy + n, acc);
  }
}

// s = max |w| / 7 over the group, rounded to the scales' type; code = clamp(rint(w / s), -8, 7) + 8, 8 where s is 0.
// One warp per block of 128 columns: lane l takes columns 4 l .. 4 l + 3, so a group is group / 4 lanes.
__global__ void __launch_bounds__(256) w4_pack_kernel(const void* w, int dt, int64_t N, int64_t K, int64_t ldw,
                                                      int group, uint8_t* codes, int64_t row_bytes, void* scales,
                                                      int sdt, int64_t n_groups) {
  const int64_t blocks = row_bytes / 64;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (i >= N * blocks) return;
  const int64_t n = i / blocks, col = (i % blocks) * kW4Block + 4 * lane_id();
  float x[4], top = 0.f;
  for (int c = 0; c < 4; ++c) {
    x[c] = col + c < K ? load_f32(w, dt, n * ldw + col + c) : 0.f;
    top = fmaxf(top, fabsf(x[c]));
  }
  for (int o = group / 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float s = top / 7.f;
  s = sdt == XDNA_BF16 ? __bfloat162float(__float2bfloat16_rn(s)) : __half2float(__float2half_rn(s));
  const int64_t g = col / group;
  if (lane_id() % (group / 4) == 0 && g < n_groups) store_f32(scales, sdt, n * n_groups + g, s);
  // the run of eight columns is two lanes' four
  const int first = (lane_id() & 1) * 4;
  uint32_t word = 0;
  for (int c = 0; c < 4; ++c) {
    const float r = s > 0.f ? fminf(fmaxf(rintf(x[c] / s), -8.f), 7.f) : 0.f;
    word |= static_cast<uint32_t>(static_cast<int>(r) + 8) << w4_shift(first + c);
  }
  word |= __shfl_xor_sync(0xffffffffu, word, 1);
  if ((lane_id() & 1) == 0) {
    const int run = lane_id() >> 1;
    reinterpret_cast<uint32_t*>(codes + n * row_bytes + (i % blocks) * 64)[(run & 3) * 4 + (run >> 2)] = word;
  }
}

static int check_w4(const char* what, int64_t N, int64_t K, int group, int scale_dtype) {
  XDNA_CHECK_ARG(N >= 0 && N < (1ll << 31) && K >= 1 && K < (1ll << 31), "%s: bad sizes", what);
  XDNA_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: groups of 32, 64 or 128 columns", what);
  XDNA_CHECK_ARG(scale_dtype == XDNA_BF16 || scale_dtype == XDNA_F16, "%s: scales in bf16 or f16", what);
  return XDNA_OK;
}

}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_w4_pack(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ldw, int group, uint8_t* codes,
                 void* scales, int scale_dtype, void* stream) {
  int rc = check_w4("w4_pack", N, K, group, scale_dtype);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(is_float_dtype(w_dtype) && ldw >= K, "w4_pack: bad weight type or row pitch");
  if ((rc = check_device(nullptr)) != XDNA_OK) return rc;
  if (N == 0) return XDNA_OK;
  XDNA_CHECK_ARG(w && codes && scales && aligned16(codes), "w4_pack: null pointer or unaligned codes");
  const int64_t row_bytes = (K + kW4Block - 1) / kW4Block * 64, warps = N * (row_bytes / 64);
  XDNA_CHECK_ARG(warps / 8 < (1ll << 31) - 1, "w4_pack: too many blocks");
  w4_pack_kernel<<<static_cast<unsigned>((warps + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      w, w_dtype, N, K, ldw, group, codes, row_bytes, scales, scale_dtype, (K + group - 1) / group);
  return check_launch("w4_pack_kernel");
}

int xdna_linear_w4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* codes,
                   const void* scales, int scale_dtype, int group, int64_t N, const void* bias, int bias_dtype,
                   void* y, int64_t ldy, void* stream) {
  int rc = check_w4("linear_w4", N, K, group, scale_dtype);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(M >= 0 && M < 65536 && ldx >= K && ldy >= N && is_float_dtype(x_dtype), "linear_w4: bad x or y");
  XDNA_CHECK_ARG(bias == nullptr || is_float_dtype(bias_dtype), "linear_w4: bad bias type");
  if ((rc = check_device(nullptr)) != XDNA_OK) return rc;
  if (M == 0 || N == 0) return XDNA_OK;
  XDNA_CHECK_ARG(x && codes && scales && y && aligned16(codes), "linear_w4: null pointer or unaligned codes");
  const W4Args a{x, ldx, codes, scales, bias, y, ldy, M, N, K, (K + kW4Block - 1) / kW4Block * 64,
                 (K + group - 1) / group, x_dtype, scale_dtype, bias_dtype, group};
  w4_kernel<<<dim3(static_cast<unsigned>((N + 7) / 8), static_cast<unsigned>(M)), 256, 0,
              static_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("w4_kernel");
}

}  // extern "C"
