// The logits of the next token before it is chosen: penalties for the tokens so far, a bias and a grammar mask,
// in one pass over [B, V]. For row b and token v, with `seen` = v is among the row's first lens[b] tokens and c =
// how often it is among those after the first prompt_lens[b]:
//   l = seen ? (l > 0 ? l / rep[b] : l * rep[b]) : l      (the quotient as l times 1 / rep[b]: 1 ulp of f32)
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

constexpr int kLogitsThreads = 512;
constexpr int kLogitsCtas = 4;  // per SM, all its threads: what covers a block's two barriers is other blocks

template <typename T>
struct LogitVec;  // 16 bytes of logits
template <>
struct LogitVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
};
template <>
struct LogitVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};
template <>
struct LogitVec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float x) { *p = __float2half_rn(x); }
};

// A block takes VECS x 512 pieces of 16 bytes of one row. The loads go out first: the thread's first tokens, its
// logits and mask words. While they are on their way the block clears a bitmap and its counters; then it marks
// and counts the row's tokens that fall into its entries (integer sums in shared memory, so their order does not
// matter), and each piece is worked on in registers and written; only pieces with a marked entry look at the counters.
// The row is cut at 16-byte boundaries of its own address, so rows of any pitch are read and written in whole pieces
// except at their two ends.
// The history is read once per block, from the L2. 128 rows of 151936 in bf16 with a mask each, a shared bias and 2048
// tokens each: 26 us (82 MB, 3.1 TB/s); without tokens 16 us. Of the difference about 4 us are the atomics and the
// penalised entries, 2 the reading of the history and 1 the clearing; six blocks of 256 an SM took 27.4 us, longer
// ones, fewer to an SM, 28 to 33, and a pass of its own for the penalised entries 30 (their scattered stores).
template <typename T, typename Tok, int VECS>
__global__ void __launch_bounds__(kLogitsThreads, kLogitsCtas) logits_kernel(const LogitsArgs a) {
  using Vec = LogitVec<T>;
  constexpr int N = Vec::N, kChunk = VECS * kLogitsThreads * N;
  constexpr int M = 16 / sizeof(Tok), kAhead = 1;    // tokens of a piece, pieces of the history loaded ahead
  extern __shared__ __align__(16) uint32_t count[];  // [kChunk] (with tokens)
  __shared__ uint32_t marked[kChunk / 32];
  const int64_t row = blockIdx.y;
  const T* in = static_cast<const T*>(a.in) + row * a.ld_in;
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const int V = static_cast<int>(a.V), tid = threadIdx.x;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  // entries [base, base + kChunk) of the row, those outside [0, V) left out; in + base is on a 16-byte boundary
  const int base = static_cast<int>(blockIdx.x) * kChunk - shift;
  const bool pieces = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(in)) & 15) == 0;

  // the history up to T, whatever the row's length: it is cut when counting
  const Tok* tok = static_cast<const Tok*>(a.tokens) + row * a.ld_tokens;
  const int T_ = static_cast<int>(a.T);
  const int head = min(T_, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(tok) & 15)) % 16 / sizeof(Tok)));
  uint4 ahead[kAhead];
  int len = T_, prompt = 0;
  if (a.tokens) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = head + (i * kLogitsThreads + tid) * M;
      if (at + M <= T_) ahead[i] = *reinterpret_cast<const uint4*>(tok + at);
    }
    if (a.lens) len = min(max(a.lens[row], 0), T_);
    if (a.prompt_lens) prompt = a.prompt_lens[row];
  }
  const float rep = a.rep ? a.rep[row] : 1.f, inv_rep = 1.f / rep, pres = a.pres ? a.pres[row] : 0.f, freq = a.freq ? a.freq[row] : 0.f;
  auto whole = [&](int at) { return pieces && at >= 0 && at + N <= V; };
  uint4 raw[VECS];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int at = base + (v * kLogitsThreads + tid) * N;
    if (whole(at)) raw[v] = __ldcs(reinterpret_cast<const uint4*>(in + at));
  }
  const float* bias = a.bias ? a.bias + row * a.ld_bias : nullptr;
  const bool wide_bias = bias && (reinterpret_cast<uintptr_t>(bias + base) & 15) == 0;
  const uint32_t* mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
  uint32_t allowed[VECS];
  if (mask) {
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = base + (v * kLogitsThreads + tid) * N, sh = at & 31;
      if (whole(at)) {
        allowed[v] = mask[at >> 5] >> sh;
        if (sh + N > 32) allowed[v] |= mask[(at >> 5) + 1] << (32 - sh);
      }
    }
  }
  if (a.tokens) {
#pragma unroll
    for (int i = 0; i < kChunk / 4 / kLogitsThreads; ++i) reinterpret_cast<uint4*>(count)[i * kLogitsThreads + tid] = make_uint4(0, 0, 0, 0);
    if (tid < kChunk / 32) marked[tid] = 0;
    __syncthreads();
    // entries [first, first + range) of the row are this block's: one subtraction and one comparison per token
    const uint32_t first = static_cast<uint32_t>(max(base, 0));
    const uint32_t range = static_cast<uint32_t>(max(min(base + kChunk, V) - max(base, 0), 0));  // 0 in a block past V
    auto here = [&](Tok id) {
      if constexpr (sizeof(Tok) == 8)
        return static_cast<uint64_t>(id) - first < range;
      else
        return static_cast<uint32_t>(id) - first < range;
    };
    auto put = [&](int i, Tok id) {
      if (!here(id) || i >= len) return;
      const int at = static_cast<int>(id) - base;
      atomicOr(&marked[at >> 5], 1u << (at & 31));
      if (i >= prompt) atomicAdd(&count[at], 1u);
    };
    auto put_piece = [&](int at, const uint4& u) {
      Tok id[M];
      *reinterpret_cast<uint4*>(id) = u;
      bool any = false;
#pragma unroll
      for (int e = 0; e < M; ++e) any |= here(id[e]);
      if (any) {
#pragma unroll
        for (int e = 0; e < M; ++e) put(at + e, id[e]);
      }
    };
    if (tid < head) put(tid, tok[tid]);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = head + (i * kLogitsThreads + tid) * M;
      if (at + M <= T_) put_piece(at, ahead[i]);
    }
    const int rest = head + (T_ - head) / M * M;
    for (int at = head + (kAhead * kLogitsThreads + tid) * M; at < min(len, rest); at += kLogitsThreads * M)
      put_piece(at, *reinterpret_cast<const uint4*>(tok + at));
    if (rest + tid < T_) put(rest + tid, tok[rest + tid]);  // fewer than M
    __syncthreads();
  }
  auto penalise = [&](float l, int at) {
    l *= l > 0.f ? inv_rep : rep;
    const uint32_t c = count[at];
    return c ? l - freq * static_cast<float>(c) - pres : l;
  };
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int in_chunk = (v * kLogitsThreads + tid) * N, at = base + in_chunk;
    const uint32_t hit = a.tokens ? marked[in_chunk >> 5] >> (in_chunk & 31) & ((1u << N) - 1) : 0;
    if (whole(at)) {
      float x[N];
      Vec::unpack(raw[v], x);
      if (hit) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (hit >> e & 1) x[e] = penalise(x[e], in_chunk + e);
      }
      if (wide_bias) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const float4 f = *reinterpret_cast<const float4*>(bias + at + e);
          x[e] += f.x, x[e + 1] += f.y, x[e + 2] += f.z, x[e + 3] += f.w;
        }
      } else if (bias) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] += bias[at + e];
      }
      if (mask) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (!(allowed[v] >> e & 1)) x[e] = -INFINITY;
      }
      __stcs(reinterpret_cast<uint4*>(out + at), Vec::pack(x));
    } else {
      for (int e = 0; e < N; ++e) {
        const int i = at + e;
        if (i < 0 || i >= V) continue;
        float l = Vec::load(in + i);
        if (hit >> e & 1) l = penalise(l, in_chunk + e);
        if (bias) l += bias[i];
        if (mask && !((mask[i >> 5] >> (i & 31)) & 1u)) l = -INFINITY;
        Vec::store(out + i, l);
      }
    }
  }
}

template <typename T, typename Tok, int VECS>
static void launch_logits(const LogitsArgs& a, int64_t B, cudaStream_t s) {
  constexpr int N = LogitVec<T>::N, kChunk = VECS * kLogitsThreads * N;
  // a row that starts off a 16-byte boundary reaches up to N - 1 entries further
  const dim3 grid(static_cast<unsigned>((a.V + N - 1 + kChunk - 1) / kChunk), static_cast<unsigned>(B));
  logits_kernel<T, Tok, VECS><<<grid, kLogitsThreads, a.tokens ? kChunk * 4 : 0, s>>>(a);
}

// Two pieces a thread, or one where that leaves SMs without enough blocks.
template <typename T>
static void run_logits(const LogitsArgs& a, int64_t B, int token_bytes, int sms, cudaStream_t s) {
  const int64_t pieces = B * ((a.V + LogitVec<T>::N - 1) / LogitVec<T>::N + kLogitsThreads - 1) / kLogitsThreads;
  const bool two = pieces >= 4 * sms;
  if (token_bytes == 8)
    two ? launch_logits<T, int64_t, 2>(a, B, s) : launch_logits<T, int64_t, 1>(a, B, s);
  else
    two ? launch_logits<T, int32_t, 2>(a, B, s) : launch_logits<T, int32_t, 1>(a, B, s);
}

}  // namespace xdna

using namespace xdna;

extern "C" int xdna_process_logits(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld_in,
                                   const void* tokens, int token_bytes, int64_t T, int64_t ld_tokens,
                                   const int32_t* lens, const int32_t* prompt_lens, const float* repetition,
                                   const float* presence, const float* frequency, const float* bias, int64_t ld_bias,
                                   const uint32_t* mask, int64_t ld_mask, void* out, int64_t ld_out, void* stream) {
  XDNA_CHECK_ARG(B >= 0 && B < 65536 && V >= 0 && V < (1ll << 30) && T >= 0 && T < (1ll << 30),
                 "process_logits: bad sizes (at most 65535 rows)");
  XDNA_CHECK_ARG(is_float_dtype(dtype), "process_logits: f32, bf16 or f16 logits");
  XDNA_CHECK_ARG(tokens == nullptr || token_bytes == 4 || token_bytes == 8, "process_logits: 32 or 64-bit tokens");
  int sms = 0;
  int rc = check_device(&sms);
  if (rc != XDNA_OK) return rc;
  if (B == 0 || V == 0) return XDNA_OK;
  XDNA_CHECK_ARG(logits && out && ld_in >= 0 && ld_out >= V && reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0, "process_logits: null pointer or bad row pitch");
  const LogitsArgs a{logits, out, ld_in, ld_out, V, tokens, T, ld_tokens, lens, prompt_lens, repetition, presence,
                     frequency, bias, ld_bias, mask, ld_mask};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == XDNA_F32)
    run_logits<float>(a, B, token_bytes, sms, s);
  else if (dtype == XDNA_BF16)
    run_logits<__nv_bfloat16>(a, B, token_bytes, sms, s);
  else
    run_logits<__half>(a, B, token_bytes, sms, s);
  return check_launch("logits_kernel");
}
