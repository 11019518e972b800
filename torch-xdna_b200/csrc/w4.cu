// Linears with 4-bit weights and group scales for the few rows of a decode step:
//   y[m, n] = sum over groups g of s[n, g] * sum_{k in g} (c[n, k] - 8) x[m, k]  (+ bias[n]),  c in 0..15.
//
// Codes are stored in blocks of 128 columns (64 bytes, K padded with code 8 to whole blocks): the block's runs of
// eight columns r = 4 w + t lie as 32-bit words at place 4 t + w, and in a word the eight codes lie in the column
// order 0, 2, 4, 6, 1, 3, 5, 7 from the lowest bits.
#include <algorithm>

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
  int64_t ldy;
  int M, N, K, blocks, n_groups;  // blocks of 128 columns
  int x_dtype, scale_dtype, bias_dtype;
  int rows;     // x rows of a pass (blockIdx.y)
  int chunk;    // blocks of x in shared memory at a time
};

// The linear as tensor-core products of 16 weight rows by 8 (NT times) x rows, with the weights as the A operand: a
// decode step has few x rows, so its time is the reading of the codes, and what has to be kept small is the work per
// code. A warp takes tiles of 16 weight rows. Each lane copies its codes (16 bytes, 32 codes, of each block of the rows
// g and g + 8) and its share of the scales into the warp's ring in shared memory, kW4Blocks blocks to a stage and
// kW4Stages stages ahead (cp.async), so that the addresses are worked out once per stage. Every 32-bit word of the
// codes is, after a shift, a mask-and-or and a subtraction per pair, two registers of A fragments: codes are stored so
// that a word's pairs are neighbouring columns and the four lanes of a fragment row hold one group of 32.
// (code - 8) is exact in bf16 and f16, so the products are exact; they are summed in f32 over a group, and then
// multiplied by the group's scale into the f32 accumulators.
// f32 x: each value is the exact sum of three bf16 numbers (truncated high, middle and low 8 bits), which take three
// of the x rows of a product and are added at the end; so the result has the accuracy of f32 sums.
// x lies in shared memory, 64 bytes off a multiple of 128 per row, which makes the B fragments' loads free of conflicts.
// A CTA has an equal share of the tiles, to one, eight at a time; where fewer are left, or there are fewer from the
// start, 2, 4 or 8 warps share one, each with a run of its blocks, and add their sums in shared memory in a fixed order.
// (Whole rounds of eight alone left the 9496 tiles of a 151936-row head at 4.01 rounds: a fifth with three CTAs.)
// 151936 x 1024, 8 x rows, groups of 128: 23 us for 82 MB, 3.6 TB/s. The copies alone take 19 us (16 warps to an SM, each
// with two stages under way), and taking codes apart (11 operations for the 8 codes of a word; the issue slots are busy 59
// % of the time) is not wholly hidden behind them. 4096 x 1024, one x row: 3.5 us, of which a kernel that does next to
// nothing takes 1.5. (Short replays of a graph.)
// A group's products are summed before its scale: |x| above 4e37 / group can overflow f32 there.
// K split over the CTAs of a cluster, to give few tiles more SMs, was left out: 24.7 us became 18.3 where x is long (30
// rows of 5001), but 4.1 became 6.0 for 1024 x 2048 (the cluster's launch and its two barriers).
constexpr int kW4Blocks = 4;
constexpr int kW4Stages = 2;
constexpr int kW4Threads = 256;
constexpr int kW4Smem = 227 * 1024;  // what a CTA may have; two on an SM lose 1 KB each of its 228
// a warp's codes and scales: of each row four lanes' words as often as the stage's groups need
constexpr int w4_scale_words(int group) { return (kW4Blocks * (kW4Block / group) + 3) / 4; }
constexpr int w4_stage_bytes(int group) { return kW4Blocks * 1024 + w4_scale_words(group) * 256; }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// 16 bytes, of which the first n are read and the others are zeros.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// 4 bytes, of which the first n (2 or 4) are read and the others are zeros.
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The codes at bits 0..3 and 16..19 of w as two exact values code - 8: 128 + code (bf16: ulp 1 at 128) or 1024 + code
// (f16) by setting the exponent, minus 136 or 1032.
template <bool BF16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t u, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(u) : "r"(w), "r"(0x000f000fu), "r"(BF16 ? 0x43004300u : 0x64006400u));  // (w & mask) | exponent
  if constexpr (BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0x3f803f80u), "r"(0xc308c308u));  // u * 1 - 136
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0x3c003c00u), "r"(0xe408e408u));  // u * 1 - 1032
  return r;
}

// XT: x's type (XDNA_F32 as three bf16 parts per value).
template <int XT, int NT, int GROUP>
__global__ void __launch_bounds__(kW4Threads) w4_kernel(const W4Args a) {
  constexpr bool kBf16 = XT != XDNA_F16;
  constexpr int kParts = XT == XDNA_F32 ? 3 : 1, kPer = kW4Block / GROUP;  // groups per block
  constexpr int kStageBytes = w4_stage_bytes(GROUP), kWords = w4_scale_words(GROUP);
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * a.rows, m_rows = min(a.rows, a.M - m0), v_rows = m_rows * kParts;
  const int pitch = a.chunk * kW4Block * 2 + 64;
  uint8_t* ring = smem + warp * (kW4Stages * kStageBytes);
  uint8_t* smx = smem + 8 * kW4Stages * kStageBytes;
  float* red = reinterpret_cast<float*>(smx + ((a.rows * kParts * pitch + 127) & ~127));  // [warp][16][NT * 8]
  const int64_t n_tiles = (a.N + 15) / 16;
  const int tile0 = static_cast<int>(n_tiles * blockIdx.x / gridDim.x), tile1 = static_cast<int>(n_tiles * (blockIdx.x + 1) / gridDim.x);
  const int64_t row_bytes = static_cast<int64_t>(a.blocks) * 64;

  // What a warp does, in order: its tile of each round, of it its run of each chunk of blocks, of it stages of kW4Blocks
  // blocks. prefetch() walks this order kW4Stages ahead of the use.
  struct Round {
    int tile, ks, slice, run;  // tile -1: no part in it
  };
  auto round_of = [&](int i) -> Round {
    const int left = tile1 - tile0 - 8 * i;
    int log2 = left >= 5 ? 0 : left >= 3 ? 1 : left == 2 ? 2 : 3;
    while ((1 << log2) > a.blocks) --log2;
    Round r;
    r.ks = 1 << log2;
    r.slice = warp & (r.ks - 1);
    r.run = (a.chunk + r.ks - 1) >> log2;
    r.tile = (warp >> log2) < left ? tile0 + 8 * i + (warp >> log2) : -1;
    return r;
  };
  const int n_rounds = (tile1 - tile0 + 7) / 8;
  Round p = n_rounds > 0 ? round_of(0) : Round{-1, 1, 0, 0};
  int p_round = 0, p_b0 = 0, p_blk = 0, p_end = 0, p_stage = 0;  // of the run under way, blocks p_blk .. p_end - 1 are left
  // where its next stage's codes of rows g and g + 8 lie, and the aligned 4 bytes that hold their scales: lane t copies
  // every fourth scale of a row (a stage's scales are an even number, so they stay aligned)
  const uint8_t *p_lo = nullptr, *p_hi = nullptr;
  const uint16_t *p_slo = nullptr, *p_shi = nullptr;
  bool p_inner = false;  // there are rows after these
  static_assert(kW4Blocks * kPer % 2 == 0, "a stage's scales are an even number");
  // the next run with blocks, if there is one
  auto next_run = [&](bool first) {
    while (p_round < n_rounds) {
      if (!first) {
        p_b0 += a.chunk;
        if (p_b0 >= a.blocks || p.tile < 0) {
          p_b0 = 0;
          if (++p_round < n_rounds) p = round_of(p_round);
        }
      }
      first = false;
      if (p_round >= n_rounds || p.tile < 0) continue;
      p_blk = p_b0 + p.slice * p.run;
      p_end = min(a.blocks, p_b0 + min(a.chunk, (p.slice + 1) * p.run));
      if (p_blk >= p_end) continue;
      // rows past N repeat the last one: their results are not used
      const int n = min(p.tile * 16 + g, a.N - 1), n8 = min(n + 8, a.N - 1);
      p_lo = a.codes + n * row_bytes + p_blk * 64 + t * 16;
      p_hi = a.codes + n8 * row_bytes + p_blk * 64 + t * 16;
      const uint16_t* sc = static_cast<const uint16_t*>(a.scales);
      p_slo = sc + ((static_cast<int64_t>(n) * a.n_groups + p_blk * kPer + t) & ~int64_t(1));
      p_shi = sc + ((static_cast<int64_t>(n8) * a.n_groups + p_blk * kPer + t) & ~int64_t(1));
      p_inner = n8 < a.N - 1;
      return;
    }
  };
  next_run(true);
  const uint32_t ring_lane = smem_u32(ring) + lane * 16, ring_scale = smem_u32(ring) + kW4Blocks * 1024 + lane * 4;
  auto prefetch = [&]() {
    if (p_round < n_rounds) {
      const uint32_t dst = ring_lane + p_stage * kStageBytes, dst_s = ring_scale + p_stage * kStageBytes;
      if (p_blk + kW4Blocks <= p_end && (p_inner || p_blk + std::max(kW4Blocks, 4 / kPer) < a.blocks)) {
#pragma unroll
        for (int u = 0; u < kW4Blocks; ++u) {
          cp_async_16(dst + u * 1024, p_lo + u * 64);
          cp_async_16(dst + u * 1024 + 512, p_hi + u * 64);
        }
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          cp_async_4(dst_s + j * 256, p_slo + 4 * j, 4);
          cp_async_4(dst_s + j * 256 + 128, p_shi + 4 * j, 4);
        }
      } else {
#pragma unroll
        for (int u = 0; u < kW4Blocks; ++u) {
          if (p_blk + u < p_end) {
            cp_async_16(dst + u * 1024, p_lo + u * 64);
            cp_async_16(dst + u * 1024 + 512, p_hi + u * 64);
          }
        }
        const uint16_t* sc_last = static_cast<const uint16_t*>(a.scales) + (static_cast<int64_t>(a.N) * a.n_groups - 1);
        const int groups = min(a.n_groups, p_end * kPer);
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          if (p_blk * kPer + 4 * j + t < groups) {  // the array's last scale may stand alone in its word
            cp_async_4(dst_s + j * 256, p_slo + 4 * j, p_slo + 4 * j < sc_last ? 4 : 2);
            cp_async_4(dst_s + j * 256 + 128, p_shi + 4 * j, p_shi + 4 * j < sc_last ? 4 : 2);
          }
        }
      }
      p_blk += kW4Blocks;
      p_lo += kW4Blocks * 64;
      p_hi += kW4Blocks * 64;
      p_slo += kW4Blocks * kPer;
      p_shi += kW4Blocks * kPer;
      if (p_blk >= p_end) next_run(false);
    }
    p_stage = p_stage + 1 == kW4Stages ? 0 : p_stage + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // x of 16 bits on 16-byte boundaries is copied as the codes are, and before the first of them; else it is read value
  // by value after they are on their way.
  const bool copy_x = kParts == 1 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ldx % 8 == 0;
  auto stage_x = [&](int b0) {
    const int cols = min(a.blocks - b0, a.chunk) * kW4Block, k0 = b0 * kW4Block;
    if (kParts == 1 && copy_x) {
      const uint16_t* x = static_cast<const uint16_t*>(a.x) + static_cast<int64_t>(m0) * a.ldx + k0;
      const int per = cols / 8;
      for (int i = threadIdx.x; i < m_rows * per; i += kW4Threads) {
        const int r = i / per, c = (i - r * per) * 8, n = min(max(a.K - k0 - c, 0), 8) * 2;  // zeros past K
        cp_async_16(smem_u32(smx) + r * pitch + c * 2, n ? x + r * a.ldx + c : x, n);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      return;
    }
    // single values: a warp takes runs of 512 columns of a row, 16 loads per lane under way together
    const int runs = (cols + 511) / 512;
    for (int job = warp; job < m_rows * runs; job += kW4Threads / 32) {
      const int r = job / runs, c0 = (job - r * runs) * 512 + lane;
      if constexpr (kParts == 1) {
        const uint16_t* x = static_cast<const uint16_t*>(a.x) + static_cast<int64_t>(m0 + r) * a.ldx + k0;
        uint16_t v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = c0 + 32 * e < cols && k0 + c0 + 32 * e < a.K ? x[c0 + 32 * e] : uint16_t(0);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (c0 + 32 * e < cols) *reinterpret_cast<uint16_t*>(smx + r * pitch + (c0 + 32 * e) * 2) = v[e];
      } else {
        const float* x = static_cast<const float*>(a.x) + static_cast<int64_t>(m0 + r) * a.ldx + k0;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = c0 + 32 * e < cols && k0 + c0 + 32 * e < a.K ? x[c0 + 32 * e] : 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (c0 + 32 * e >= cols) break;
          const bool fin = fabsf(v[e]) < INFINITY;
          const __nv_bfloat16 hi = fin ? __float2bfloat16_rz(v[e]) : __float2bfloat16_rn(v[e]);
          const float r1 = fin ? v[e] - __bfloat162float(hi) : 0.f;
          const __nv_bfloat16 mid = __float2bfloat16_rz(r1);
          const __nv_bfloat16 lo = __float2bfloat16_rn(r1 - __bfloat162float(mid));
          __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(smx + 3 * r * pitch + (c0 + 32 * e) * 2);
          d[0] = hi;
          d[pitch / 2] = mid;
          d[pitch] = lo;
        }
      }
    }
  };
  if (copy_x) stage_x(0);
#pragma unroll
  for (int i = 0; i < kW4Stages; ++i) prefetch();
  if (!copy_x) stage_x(0);
  asm volatile("cp.async.wait_group %0;" ::"n"(kW4Stages) : "memory");  // x, where it is copied
  __syncthreads();
  int stage = 0;

  auto scale_of = [&](uint32_t word, uint32_t selector) {
    const uint32_t top = __byte_perm(word, 0, selector);  // the scale in the upper half
    return a.scale_dtype == XDNA_BF16 ? __uint_as_float(top) : __half2float(__ushort_as_half(static_cast<unsigned short>(top >> 16)));
  };
  auto finish = [&](int m, int n, float v) {
    if (a.bias) v += load_f32(a.bias, a.bias_dtype, n);
    store_f32(a.y, XT, (m0 + m) * a.ldy + n, v);
  };

  int x_row[NT];  // columns of a product past the last x row repeat it: their sums are not used
#pragma unroll
  for (int i = 0; i < NT; ++i) x_row[i] = min(i * 8 + g, v_rows - 1) * pitch;
  for (int round = 0; round < n_rounds; ++round) {
    const Round now = round_of(round);
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    // a scale is the upper half of its word where it stands at an odd place of the array
    const int row_lo = min(max(now.tile, 0) * 16 + g, a.N - 1);
    const uint32_t odd_lo = row_lo & a.n_groups & 1, odd_hi = min(row_lo + 8, a.N - 1) & a.n_groups & 1;
    for (int b0 = 0; b0 < a.blocks; b0 += a.chunk) {
      if (a.chunk < a.blocks && (b0 > 0 || round > 0)) {
        __syncthreads();
        stage_x(b0);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
      }
      const int first = b0 + now.slice * now.run;
      const int last = now.tile < 0 ? 0 : min(a.blocks, b0 + min(a.chunk, (now.slice + 1) * now.run));
      for (int blk = first; blk < last; blk += kW4Blocks) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kW4Stages - 1) : "memory");
        __syncwarp();  // a fragment row's scales come from its four lanes
        const uint8_t* mine = ring + stage * kStageBytes + lane * 16;
        const uint8_t* scales = ring + stage * kStageBytes + kW4Blocks * 1024 + g * 16;
        const uint8_t* xb = smx + (blk - b0) * (kW4Block * 2) + t * 16;
        // byte selectors that bring a word's scale to the upper half: of the scales of even and of odd lanes
        const bool up_lo = (odd_lo ^ (blk * kPer)) & 1, up_hi = (odd_hi ^ (blk * kPer)) & 1;
        const uint32_t sel_lo[2] = {up_lo ? 0x3244u : 0x1044u, up_lo ? 0x1044u : 0x3244u};
        const uint32_t sel_hi[2] = {up_hi ? 0x3244u : 0x1044u, up_hi ? 0x1044u : 0x3244u};
#pragma unroll
        for (int u = 0; u < kW4Blocks; ++u) {
          if (blk + u >= last) break;
          const uint4 lo4 = *reinterpret_cast<const uint4*>(mine + u * 1024), hi4 = *reinterpret_cast<const uint4*>(mine + u * 1024 + 512);
          const uint32_t wl[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, wh[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
          float part[NT][4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if ((w * 32) % GROUP == 0) {
#pragma unroll
              for (int i = 0; i < NT; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
            }
            const uint32_t a0[4] = {code_pair<kBf16>(wl[w]), code_pair<kBf16>(wh[w]), code_pair<kBf16>(wl[w] >> 4),
                                    code_pair<kBf16>(wh[w] >> 4)};
            const uint32_t a1[4] = {code_pair<kBf16>(wl[w] >> 8), code_pair<kBf16>(wh[w] >> 8),
                                    code_pair<kBf16>(wl[w] >> 12), code_pair<kBf16>(wh[w] >> 12)};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const uint4 b = *reinterpret_cast<const uint4*>(xb + x_row[i] + u * (kW4Block * 2) + w * 64);
              mma_16816<kBf16>(part[i], a0, b.x, b.y);
              mma_16816<kBf16>(part[i], a1, b.z, b.w);
            }
            if ((w * 32 + 32) % GROUP == 0) {
              const int idx = u * kPer + w * 32 / GROUP, j = idx >> 2, lane_t = idx & 3;
              // groups past the last hold padding columns alone
              const bool there = kPer == 1 || (blk + u) * kPer + w * 32 / GROUP < a.n_groups;
              const uint32_t s_lo = *reinterpret_cast<const uint32_t*>(scales + j * 256 + lane_t * 4);
              const uint32_t s_hi = *reinterpret_cast<const uint32_t*>(scales + j * 256 + 128 + lane_t * 4);
              const float sl = there ? scale_of(s_lo, sel_lo[lane_t & 1]) : 0.f;
              const float sh = there ? scale_of(s_hi, sel_hi[lane_t & 1]) : 0.f;
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                acc[i][0] = fmaf(part[i][0], sl, acc[i][0]);
                acc[i][1] = fmaf(part[i][1], sl, acc[i][1]);
                acc[i][2] = fmaf(part[i][2], sh, acc[i][2]);
                acc[i][3] = fmaf(part[i][3], sh, acc[i][3]);
              }
            }
          }
        }
        __syncwarp();
        prefetch();  // into the stage just read
        stage = stage + 1 == kW4Stages ? 0 : stage + 1;
      }
    }
    if (kParts == 1 && now.ks == 1) {
      if (now.tile >= 0) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int m = i * 8 + 2 * t + (e & 1), n = now.tile * 16 + g + (e >> 1) * 8;
            if (m < m_rows && n < a.N) finish(m, n, acc[i][e]);
          }
        }
      }
      continue;
    }
    float* mine = red + warp * (16 * NT * 8);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(g + (e >> 1) * 8) * (NT * 8) + i * 8 + 2 * t + (e & 1)] = acc[i][e];
    }
    const bool alone = now.ks == 1;
    if (alone) __syncwarp(); else __syncthreads();
    // outputs: those of the round's tiles, or of this warp's alone
    const int here = alone ? now.tile >= 0 : min(8 / now.ks, tile1 - tile0 - 8 * round);
    const int n_out = here * 16, step = alone ? 32 : kW4Threads;
    for (int i = alone ? lane : threadIdx.x; i < n_out * m_rows; i += step) {
      const int r = i % n_out, m = i / n_out;
      const int n = (alone ? now.tile : tile0 + 8 * round + (r >> 4)) * 16 + (r & 15);
      if (n >= a.N) continue;
      const float* sums = red + ((alone ? warp : (r >> 4) * now.ks) * 16 + (r & 15)) * (NT * 8) + m * kParts;
      float v = 0.f;
      for (int q = kParts - 1; q >= 0; --q)  // small parts first
        for (int k = 0; k < now.ks; ++k) v += sums[k * 16 * (NT * 8) + q];
      finish(m, n, v);
    }
    if (alone) __syncwarp(); else __syncthreads();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int XT, int NT>
static int launch_w4(W4Args& a, int group, dim3 grid, int smem, cudaStream_t s) {
  auto kern = group == 32 ? w4_kernel<XT, NT, 32> : group == 64 ? w4_kernel<XT, NT, 64> : w4_kernel<XT, NT, 128>;
  static std::atomic<bool> configured[3][64];  // setting the attribute twice from two threads is harmless
  const int gi = group / 64;
  int dev = 0;
  XDNA_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[gi][dev].load(std::memory_order_acquire)) {
    XDNA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem));
    if (dev >= 0 && dev < 64) configured[gi][dev].store(true, std::memory_order_release);
  }
  kern<<<grid, kW4Threads, smem, s>>>(a);
  return check_launch("w4_kernel");
}

template <int XT>
static int run_w4(W4Args& a, int group, int sms, cudaStream_t s) {
  constexpr int kParts = XT == XDNA_F32 ? 3 : 1;
  // a pass takes up to 32 x rows (10 of f32); more run as further passes over the codes, which the L2 then holds
  const int passes = (a.M + 32 / kParts - 1) / (32 / kParts);
  a.rows = (a.M + passes - 1) / passes;
  const int v_rows = a.rows * kParts, nt = v_rows <= 8 ? 1 : v_rows <= 16 ? 2 : 4;
  // x in shared memory, whole where it fits beside the ring and the sums, else in runs of blocks
  const int others = 8 * kW4Stages * w4_stage_bytes(group) + 8 * 16 * nt * 8 * 4;
  a.chunk = std::min(a.blocks, ((kW4Smem - others - 128) / v_rows - 64) / (kW4Block * 2));
  const int smem = others + (v_rows * (a.chunk * kW4Block * 2 + 64) + 127) / 128 * 128;
  // One wave: the CTAs of all passes together are as many as run at a time, two per SM where the shared memory allows it,
  // so x is copied once per CTA and pass. (Two per SM of each pass whatever the shared memory, 20000 rows of 4096: 79 us
  // for 32 x rows, 44 for 16, against 52 and 24; 6144 rows of 1024 and 40 x rows 24.9 against 8.1; x in shorter runs so
  // that two CTAs always fit took 134 and 31.)
  const int at_once = sms * (smem <= kW4Smem / 2 - 512 ? 2 : 1);
  // Many passes may leave SMs idle: another wave where it fills a fifth more of them (4096 rows of 1024: 2400 x rows 142
  // us in one wave, 102 in two; 3300: 142 and 114; 1800, a quarter more: 73 and 70; but 1000, a ninth more: 39 and 44).
  const int tiles = (a.N + 15) / 16;
  int across = 1;
  double best = 0;
  for (int waves = 1; waves <= 4; ++waves) {
    const int x = std::min(tiles, waves * at_once / passes);
    const double filled = static_cast<double>(x) * passes / (waves * at_once);
    if (filled > 1.2 * best) best = filled, across = std::max(1, x);
  }
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(passes));
  return nt == 1 ? launch_w4<XT, 1>(a, group, grid, smem, s)
                 : nt == 2 ? launch_w4<XT, 2>(a, group, grid, smem, s) : launch_w4<XT, 4>(a, group, grid, smem, s);
}

// s = max |w| / 7 over the group, rounded to the scales' type, NaN where a weight of it is not finite, which then shows
// in the results; code = clamp(rint(w / s), -8, 7) + 8, 8 where s is 0 or NaN.
// One warp per block of 128 columns: lane l takes columns 4 l .. 4 l + 3, so a group is group / 4 lanes.
__global__ void __launch_bounds__(256) w4_pack_kernel(const void* w, int dt, int64_t N, int64_t K, int64_t ldw,
                                                      int group, uint8_t* codes, int64_t row_bytes, void* scales,
                                                      int sdt, int64_t n_groups) {
  const int64_t blocks = row_bytes / 64;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (i >= N * blocks) return;
  const int64_t n = i / blocks, col = (i % blocks) * kW4Block + 4 * lane_id();
  float x[4], top = 0.f;
  int odd = 0;
  for (int c = 0; c < 4; ++c) {
    x[c] = col + c < K ? load_f32(w, dt, n * ldw + col + c) : 0.f;
    top = fmaxf(top, fabsf(x[c]));
    odd |= !(fabsf(x[c]) < INFINITY);
  }
  for (int o = group / 8; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    odd |= __shfl_xor_sync(0xffffffffu, odd, o);
  }
  float s = odd ? NAN : top / 7.f;
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
  XDNA_CHECK_ARG(N >= 0 && N < (1ll << 30) && K >= 1 && K < (1ll << 24), "%s: bad sizes", what);
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
  XDNA_CHECK_ARG(M >= 0 && ldx >= K && ldy >= N && is_float_dtype(x_dtype), "linear_w4: bad x or y");
  XDNA_CHECK_ARG(bias == nullptr || is_float_dtype(bias_dtype), "linear_w4: bad bias type");
  int sms = 0;
  if ((rc = check_device(&sms)) != XDNA_OK) return rc;
  if (M == 0 || N == 0) return XDNA_OK;
  XDNA_CHECK_ARG(x && codes && scales && y && aligned16(codes) && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                 "linear_w4: null pointer or unaligned codes or scales");
  W4Args a{};
  a.ldx = ldx;
  a.codes = codes;
  a.scales = scales;
  a.bias = bias;
  a.ldy = ldy;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.blocks = static_cast<int>((K + kW4Block - 1) / kW4Block);
  a.n_groups = static_cast<int>((K + group - 1) / group);
  a.x_dtype = x_dtype;
  a.scale_dtype = scale_dtype;
  a.bias_dtype = bias_dtype;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  constexpr int64_t kRows = 1 << 19;  // of a launch: 52429 passes of f32, and a grid may have 65535
  for (int64_t m = 0; m < M && rc == XDNA_OK; m += kRows) {
    a.x = static_cast<const uint8_t*>(x) + m * ldx * dtype_size(x_dtype);
    a.y = static_cast<uint8_t*>(y) + m * ldy * dtype_size(x_dtype);
    a.M = static_cast<int>(std::min(kRows, M - m));
    rc = x_dtype == XDNA_F32 ? run_w4<XDNA_F32>(a, group, sms, s)
                             : x_dtype == XDNA_BF16 ? run_w4<XDNA_BF16>(a, group, sms, s) : run_w4<XDNA_F16>(a, group, sms, s);
  }
  return rc;
}

}  // extern "C"
