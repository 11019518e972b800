// The logits of the next token before it is chosen: penalties for the tokens so far, a bias and a grammar mask,
// in one pass over [B, V]. For row b and token v, with `seen` = v is among the row's first lens[b] tokens and c =
// how often it is among those after the first prompt_lens[b]:
//   l = seen ? (l > 0 ? l / rep[b] : l * rep[b]) : l
//   l = l - freq[b] * c - (c > 0 ? pres[b] : 0)
//   l = l + bias[v]
//   l = mask bit v ? l : -inf          (a select: what stands in a masked place does not matter)
#include "host_util.h"
#include "sm100.cuh"

namespace xdna {

struct LogitsArgs {
  const void* in;
  void* out;
  int64_t ld_in, ld_out, V;
  const void* tokens;
  int64_t T, ld_tokens;
  const int32_t *lens, *prompt_lens;
  const float *rep, *pres, *freq, *bias;
  int64_t ld_bias;
  const uint32_t* mask;
  int64_t ld_mask;
};

constexpr int kLogitsChunk = 4096;       // vocabulary entries of a block
constexpr uint32_t kSeen = 0x80000000u;  // in the counter of an entry: it is among the row's tokens

__device__ __forceinline__ float logit_in(const float* p) { return *p; }
__device__ __forceinline__ float logit_in(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit_in(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void logit_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void logit_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void logit_out(__half* p, float x) { *p = __float2half_rn(x); }

// A block takes kLogitsChunk entries of one row: it counts the row's tokens that fall into them in shared memory
// (integer sums, so their order does not matter), then makes one pass over the entries.
template <typename T, typename Tok>
__global__ void __launch_bounds__(256) logits_kernel(const LogitsArgs a) {
  __shared__ uint32_t count[kLogitsChunk];
  const int64_t row = blockIdx.y, base = static_cast<int64_t>(blockIdx.x) * kLogitsChunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(kLogitsChunk), a.V - base));
  if (a.tokens) {
    for (int i = threadIdx.x; i < kLogitsChunk; i += 256) count[i] = 0;
    __syncthreads();
    const int64_t len = a.lens ? min(static_cast<int64_t>(max(a.lens[row], 0)), a.T) : a.T;
    const int64_t prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
    const Tok* tok = static_cast<const Tok*>(a.tokens) + row * a.ld_tokens;
    for (int64_t i = threadIdx.x; i < len; i += 256) {
      const int64_t at = static_cast<int64_t>(tok[i]) - base;
      if (at < 0 || at >= n) continue;
      atomicOr(&count[at], kSeen);
      if (i >= prompt) atomicAdd(&count[at], 1u);
    }
    __syncthreads();
  }
  const float rep = a.rep ? a.rep[row] : 1.f, pres = a.pres ? a.pres[row] : 0.f, freq = a.freq ? a.freq[row] : 0.f;
  const T* in = static_cast<const T*>(a.in) + row * a.ld_in + base;
  T* out = static_cast<T*>(a.out) + row * a.ld_out + base;
  for (int i = threadIdx.x; i < n; i += 256) {
    float l = logit_in(in + i);
    const uint32_t c = a.tokens ? count[i] : 0u;
    if (c) {
      l = l > 0.f ? l / rep : l * rep;
      const uint32_t k = c & ~kSeen;
      if (k) l = l - freq * static_cast<float>(k) - pres;
    }
    if (a.bias) l += a.bias[row * a.ld_bias + base + i];
    if (a.mask && !((a.mask[row * a.ld_mask + ((base + i) >> 5)] >> ((base + i) & 31)) & 1u)) l = -INFINITY;
    logit_out(out + i, l);
  }
}

template <typename T>
static void launch_logits(const LogitsArgs& a, int token_bytes, dim3 grid, cudaStream_t s) {
  if (token_bytes == 8)
    logits_kernel<T, int64_t><<<grid, 256, 0, s>>>(a);
  else
    logits_kernel<T, int32_t><<<grid, 256, 0, s>>>(a);
}

}  // namespace xdna

using namespace xdna;

extern "C" int xdna_process_logits(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld_in,
                                   const void* tokens, int token_bytes, int64_t T, int64_t ld_tokens,
                                   const int32_t* lens, const int32_t* prompt_lens, const float* repetition,
                                   const float* presence, const float* frequency, const float* bias, int64_t ld_bias,
                                   const uint32_t* mask, int64_t ld_mask, void* out, int64_t ld_out, void* stream) {
  XDNA_CHECK_ARG(B >= 0 && B < 65536 && V >= 0 && V < (1ll << 31) && T >= 0 && T < (1ll << 31),
                 "process_logits: bad sizes (at most 65535 rows)");
  XDNA_CHECK_ARG(is_float_dtype(dtype), "process_logits: f32, bf16 or f16 logits");
  XDNA_CHECK_ARG(tokens == nullptr || token_bytes == 4 || token_bytes == 8, "process_logits: 32 or 64-bit tokens");
  int rc = check_device(nullptr);
  if (rc != XDNA_OK) return rc;
  if (B == 0 || V == 0) return XDNA_OK;
  XDNA_CHECK_ARG(logits && out && ld_in >= 0 && ld_out >= V, "process_logits: null pointer or bad row pitch");
  const LogitsArgs a{logits, out, ld_in, ld_out, V, tokens, T, ld_tokens, lens, prompt_lens, repetition, presence,
                     frequency, bias, ld_bias, mask, ld_mask};
  const dim3 grid(static_cast<unsigned>((V + kLogitsChunk - 1) / kLogitsChunk), static_cast<unsigned>(B));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == XDNA_F32)
    launch_logits<float>(a, token_bytes, grid, s);
  else if (dtype == XDNA_BF16)
    launch_logits<__nv_bfloat16>(a, token_bytes, grid, s);
  else
    launch_logits<__half>(a, token_bytes, grid, s);
  return check_launch("logits_kernel");
}
