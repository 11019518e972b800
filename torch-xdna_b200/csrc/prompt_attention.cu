// Attention of the generation path: causal attention over packed prompts of different lengths
// (xdna_packed_attention) and the decode attention of a batch that shares a prefix (xdna_prefix_attention).
//
//   packed   o[t, h] = sum_s p_s v[s, h / G],  p = softmax over the keys s <= t of t's own sequence of
//            scale * q[t, h] . k[s, h / G]                                  (G = Hq / Hkv query heads per key head)
//   prefix   o[b, h]: the same softmax over all P prefix keys and the first lens[b] keys of b's own cache
//
// A row with no keys at all is zero.
#include "host_util.h"
#include "sm100.cuh"

namespace xdna {

struct PackedArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides of a token and of a head, in elements
  const int32_t* cu;
  int n_seqs, T, hq, hkv;
  float scale_log2;
  void* out;
};

struct PrefixArgs {
  const void *q, *pk, *pv, *ck, *cv;
  int64_t q_sb, q_sh, pk_st, pk_sh, pv_st, pv_sh, ck_sb, ck_st, ck_sh, cv_sb, cv_st, cv_sh;
  const int32_t* lens;
  int B, P, S, hq, hkv;
  float scale_log2;
  void* out;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// One row's running softmax, D / 32 dimensions per lane.
template <typename T, int D>
struct Row {
  float q[D / 32], o[D / 32], m, l;
  __device__ void init(const T* qp, float sc) {
    for (int i = 0; i < D / 32; ++i) {
      q[i] = to_f32(qp[i * 32 + lane_id()]) * sc;
      o[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
  }
  __device__ void key(const T* kp, const T* vp) {
    float s = 0.f;
    for (int i = 0; i < D / 32; ++i) s += q[i] * to_f32(kp[i * 32 + lane_id()]);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float a = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * a + p;
    for (int i = 0; i < D / 32; ++i) o[i] = o[i] * a + p * to_f32(vp[i * 32 + lane_id()]);
  }
  __device__ void store(T* dst) const {
    for (int i = 0; i < D / 32; ++i) dst[i * 32 + lane_id()] = from_f32<T>(l > 0.f ? o[i] / l : 0.f);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(256) packed_kernel(const PackedArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (row >= static_cast<int64_t>(a.T) * a.hq) return;
  const int t = static_cast<int>(row / a.hq), h = static_cast<int>(row % a.hq), hk = h / (a.hq / a.hkv);
  int lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (mid < a.n_seqs && a.cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  Row<T, D> r;
  r.init(static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh, a.scale_log2);
  if (a.n_seqs > 0 && t < a.cu[lo + 1])
    for (int s = max(a.cu[lo], 0); s <= t; ++s)
      r.key(static_cast<const T*>(a.k) + s * a.k_st + hk * a.k_sh, static_cast<const T*>(a.v) + s * a.v_st + hk * a.v_sh);
  r.store(static_cast<T*>(a.out) + row * D);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) prefix_kernel(const PrefixArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (row >= static_cast<int64_t>(a.B) * a.hq) return;
  const int b = static_cast<int>(row / a.hq), h = static_cast<int>(row % a.hq), hk = h / (a.hq / a.hkv);
  Row<T, D> r;
  r.init(static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh, a.scale_log2);
  for (int s = 0; s < a.P; ++s)
    r.key(static_cast<const T*>(a.pk) + s * a.pk_st + hk * a.pk_sh, static_cast<const T*>(a.pv) + s * a.pv_st + hk * a.pv_sh);
  const int n = min(max(a.lens[b], 0), a.S);
  for (int s = 0; s < n; ++s)
    r.key(static_cast<const T*>(a.ck) + b * a.ck_sb + s * a.ck_st + hk * a.ck_sh,
          static_cast<const T*>(a.cv) + b * a.cv_sb + s * a.cv_st + hk * a.cv_sh);
  r.store(static_cast<T*>(a.out) + row * D);
}

static int check_heads(const char* what, int64_t hq, int64_t hkv, int64_t d, int dtype, float scale) {
  XDNA_CHECK_ARG(hq >= 1 && hkv >= 1 && hq % hkv == 0 && hq / hkv <= 128,
                 "%s: %lld query heads over %lld key heads", what, (long long)hq, (long long)hkv);
  XDNA_CHECK_ARG(dtype == XDNA_BF16 || dtype == XDNA_F16, "%s: bf16 or f16", what);
  XDNA_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", what);
  if (d != 64 && d != 128) return fail(XDNA_ERR_UNSUPPORTED, "%s: head dimension %lld (64 or 128)", what, (long long)d);
  return XDNA_OK;
}

static bool row_ok(const void* p, int64_t a, int64_t b, int64_t c = 8) {
  return p != nullptr && aligned16(p) && a > 0 && b > 0 && c > 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

}  // namespace xdna

using namespace xdna;

extern "C" {

size_t xdna_packed_attention_workspace(int64_t n_seqs, int64_t tokens, int64_t hq, int64_t hkv) {
  return 0;
}

int xdna_packed_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                          const void* v, int64_t v_st, int64_t v_sh, const int32_t* cu_seqlens, int64_t n_seqs,
                          int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int dtype, float scale, void* out,
                          void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_heads("packed_attention", hq, hkv, d, dtype, scale);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(tokens >= 0 && n_seqs >= 0 && tokens < (1ll << 31) / hq && n_seqs < (1 << 24),
                 "packed_attention: bad sizes");
  if ((rc = check_device(nullptr)) != XDNA_OK) return rc;
  if (tokens == 0) return XDNA_OK;
  XDNA_CHECK_ARG(row_ok(q, q_st, q_sh) && row_ok(k, k_st, k_sh) && row_ok(v, v_st, v_sh) && cu_seqlens && out &&
                     aligned16(out),
                 "packed_attention: operands must be 16-byte aligned with strides that are positive multiples of 8");
  const PackedArgs a{q, k, v, q_st, q_sh, k_st, k_sh, v_st, v_sh, cu_seqlens, (int)n_seqs, (int)tokens, (int)hq,
                     (int)hkv, scale * 1.4426950408889634f, out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned g = static_cast<unsigned>((tokens * hq + 7) / 8);
  if (dtype == XDNA_BF16)
    d == 128 ? packed_kernel<__nv_bfloat16, 128><<<g, 256, 0, s>>>(a) : packed_kernel<__nv_bfloat16, 64><<<g, 256, 0, s>>>(a);
  else
    d == 128 ? packed_kernel<__half, 128><<<g, 256, 0, s>>>(a) : packed_kernel<__half, 64><<<g, 256, 0, s>>>(a);
  return check_launch("packed_kernel");
}

size_t xdna_prefix_attention_workspace(int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d) {
  return 0;
}

int xdna_prefix_attention(const void* q, int64_t q_sb, int64_t q_sh, const void* pk, int64_t pk_st, int64_t pk_sh,
                          const void* pv, int64_t pv_st, int64_t pv_sh, const void* ck, int64_t ck_sb, int64_t ck_st,
                          int64_t ck_sh, const void* cv, int64_t cv_sb, int64_t cv_st, int64_t cv_sh,
                          const int32_t* lens, int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d,
                          int dtype, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_heads("prefix_attention", hq, hkv, d, dtype, scale);
  if (rc != XDNA_OK) return rc;
  XDNA_CHECK_ARG(B >= 0 && P >= 0 && S >= 0 && B < (1ll << 31) / hq && P < (1ll << 31) && S < (1ll << 31),
                 "prefix_attention: bad sizes");
  if ((rc = check_device(nullptr)) != XDNA_OK) return rc;
  if (B == 0) return XDNA_OK;
  XDNA_CHECK_ARG(row_ok(q, q_sb, q_sh) && (P == 0 || (row_ok(pk, pk_st, pk_sh) && row_ok(pv, pv_st, pv_sh))) &&
                     (S == 0 || (row_ok(ck, ck_sb, ck_st, ck_sh) && row_ok(cv, cv_sb, cv_st, cv_sh))) && lens && out &&
                     aligned16(out),
                 "prefix_attention: operands must be 16-byte aligned with strides that are positive multiples of 8");
  const PrefixArgs a{q, pk, pv, ck, cv, q_sb, q_sh, pk_st, pk_sh, pv_st, pv_sh, ck_sb, ck_st, ck_sh, cv_sb, cv_st,
                     cv_sh, lens, (int)B, (int)P, (int)S, (int)hq, (int)hkv, scale * 1.4426950408889634f, out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned g = static_cast<unsigned>((B * hq + 7) / 8);
  if (dtype == XDNA_BF16)
    d == 128 ? prefix_kernel<__nv_bfloat16, 128><<<g, 256, 0, s>>>(a) : prefix_kernel<__nv_bfloat16, 64><<<g, 256, 0, s>>>(a);
  else
    d == 128 ? prefix_kernel<__half, 128><<<g, 256, 0, s>>>(a) : prefix_kernel<__half, 64><<<g, 256, 0, s>>>(a);
  return check_launch("prefix_kernel");
}

}  // extern "C"
