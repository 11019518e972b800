/* xdna_b200.h -- C ABI of libxdna_b200.so, the B200 (sm_100a) kernels behind torch_xdna's custom ops.
 *
 * Conventions (every entry point):
 *   - returns XDNA_OK (0) or a negative XDNA_ERR_* code; xdna_last_error() then describes the
 *     failure (thread-local, valid until the next call on the same thread);
 *   - every pointer is caller-owned device memory on the current CUDA device, except where a
 *     comment says "host";
 *   - `stream` is a cudaStream_t (NULL = legacy default stream); calls only enqueue work and
 *     never synchronise, except xdna_take_device_error();
 *   - no entry point allocates device memory except xdna_ipc_alloc (the shareable buffer a caller
 *     asks for); scratch is passed in by the caller;
 *   - leading dimensions (`ld*`) are in elements; int8 operands read by TMA need their row
 *     pitch in bytes to be a multiple of 16 and their base 16-byte aligned;
 *   - the library caches, per device, the device addresses of its own globals (the error word,
 *     the no-allocation scratch) on first use: it must not be used on a device after a
 *     cudaDeviceReset of that device (the cached addresses would point into the destroyed
 *     context); load the library again in a new process instead.
 *
 * The reference (AyaSakura-comp/torch-xdna) reaches its device through Python calls into
 * Triton-XDNA; each entry point below names the reference call it replaces.
 */
#ifndef XDNA_B200_H
#define XDNA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ status codes */
#define XDNA_OK 0
#define XDNA_ERR_INVALID (-1)     /* bad argument: shape, stride, alignment, dtype, mode */
#define XDNA_ERR_UNSUPPORTED (-2) /* a valid request this build does not implement */
#define XDNA_ERR_CUDA (-3)        /* a CUDA runtime or driver call failed */
#define XDNA_ERR_TIMEOUT (-4)     /* a bounded device-side wait gave up; the kernel returned early */
#define XDNA_ERR_DEVICE (-5)      /* the current device is not an sm_100 (B200-class) GPU */

/* ------------------------------------------------------------------ element types */
#define XDNA_F32 0
#define XDNA_BF16 1
#define XDNA_F16 2
#define XDNA_I32 3
#define XDNA_I8 4
#define XDNA_U8 5
#define XDNA_E4M3 6

/* ------------------------------------------------------------------ conv3x3 modes */
#define XDNA_CONV_Q 0         /* q = sat((acc + 2^(shift-1)) >> shift) as int8, or uint8 [0,255] with relu, NCHW */
#define XDNA_CONV_DEQUANT 1   /* y = float(q) * (scale[co] * sx[n]) (+ bias[co]) in out_dtype, channels-last
                                 memory [N, H, W, Co] (torch's channels_last layout of an [N, Co, H, W] tensor) */
#define XDNA_CONV_CALIBRATE 2 /* *acc_max = max over the sums of image 0 of (relu ? max(acc,0) : |acc|) */
#define XDNA_CONV_Q_NHWC 3    /* q as XDNA_CONV_Q, written channels-last [N, H, W, Co]: the int8 form in which
                                 one conv's output feeds the next (xdna_conv_quant_codes) */
/* Or'ed into a mode: one tap at offset 0 instead of the 3x3 stencil's nine, i.e. a 1x1 conv over the
 * bordered input with weights wp [Co, 1, Cp]. With the input from xdna_conv_quant_taps (the nine taps of
 * a few channels packed into each pixel's row) and the weights packed the same way, it is the 3x3 conv
 * of a layer with <= 7 input channels in one K block instead of nine. */
#define XDNA_CONV_SINGLE_TAP 16
/* Or'ed into a mode: a stride-2 conv (3x3 with padding 1, or with XDNA_CONV_SINGLE_TAP the 1x1 conv with no
 * padding). xp is then the input split into its stride phases by xdna_conv_quant_phases,
 * [planes, N, Ho+2, Wo+2, Cp] with planes = 4 (3x3) or 1 (1x1), and H, W are the OUTPUT's height and width
 * (Ho = ceil(H_in / 2), Wo = ceil(W_in / 2)). Plane 2 * ry + rx at bordered pixel (Y, X) holds input pixel
 * (2 (Y - 1) + ry, 2 (X - 1) + rx), zero outside the input; tap (ky, kx) of output pixel (y, x) reads plane
 * ((ky != 1), (kx != 1)) at bordered row y + (ky != 0), column x + (kx != 0), so every tap is a constant row
 * offset as in the stride-1 conv. Extends the reference's conv route (which offloads only 3x3 stride-1 convs,
 * R:torch_xdna/backend.py:130-174) to the ResNet-style layers it lists as missing
 * (R:results/conv3x3_cascade.md:222-223): same quantise, calibration and requantise. */
#define XDNA_CONV_STRIDE2 32
/* Or'ed into XDNA_CONV_Q_NHWC: the next layer's per-image maxima, so that its quantise from these codes
 * (xdna_conv_quant_codes_given_amax) needs no pass of its own over them. acc_max then holds N words, cleared by
 * this call, that receive per image the f32 bit pattern of max |y| over the output pixels, where
 * y = float(q) * (scale[c] * sx[n]) (+ bias[c], f32) is computed with the f32 operations of
 * xdna_conv_quant_codes; with XDNA_CONV_NEXT_RELU y is max(y, 0) first; with XDNA_CONV_NEXT_POOL only the
 * rows and columns a 2x2 / stride-2 pool keeps (an odd last one is left out) count, which is the pooled
 * image's max when y >= 0 (so it needs XDNA_CONV_NEXT_RELU, or relu = 1 and no bias). Needs scale, sx
 * (this conv's input scales) and bias (f32 or NULL; with XDNA_CONV_BIAS_INT32 the bias is in the codes and y
 * has no float bias term). */
#define XDNA_CONV_NEXT_AMAX 64
#define XDNA_CONV_NEXT_RELU 128
#define XDNA_CONV_NEXT_POOL 256
/* Or'ed into any conv mode: the bias inside the int32 sums, before the requantise (an option the reference
 * names as future work; its own route adds the bias to the dequantised floats, R:results/conv3x3_cascade.md:224).
 * `bias` is then int32 [N, Co] (bias_dtype XDNA_I32, one row per image: the units of the sums depend on the
 * image's sx), from xdna_conv_bias_int32; the sums become acc + bias[n][co] in every mode (the calibration's
 * max included), and DEQUANT adds no float bias. |acc| must stay below 2^31 - 3 * 2^29 (K * 127^2 < 5.3e8). */
#define XDNA_CONV_BIAS_INT32 512
/* Or'ed into XDNA_CONV_Q_NHWC for a stride-1 3x3 conv with Cp = 64, Co <= 128 and an even N: xp holds the
 * images in pairs, [N/2, H+2, W+2, 128] (bytes 0..63 of a row: image 2i's channels, 64..127: image 2i+1's;
 * xdna_conv_quant_codes_pairs writes it), which halves the TMA row requests of the conv's loads. */
#define XDNA_CONV_PAIRS 1024
/* `relu` of xdna_conv3x3_i8: 0 none; 1 fused into the requantise ([0,255] uint8, the reference's ReLU of
 * a bias-free conv); XDNA_RELU_AFTER_BIAS (DEQUANT only) applied to the dequantised output after the
 * bias, the requantise saturating to int8 — the same values as torch.relu on the DEQUANT output. */
#define XDNA_RELU_AFTER_BIAS 2

/* Last error of this thread, as text. */
const char* xdna_last_error(void);

/* ABI version of this library (bumped when a signature changes). */
int xdna_abi_version(void);

/* Kernels of this library that the calling thread has enqueued so far. */
int64_t xdna_launch_count(void);

/* XDNA_OK when `device` is an sm_100 GPU this library's kernels run on. */
int xdna_device_check(int device);

/* Reads and clears the device-side error word that bounded waits write (code, site). Synchronises
 * `stream`. *code is XDNA_OK when no kernel recorded an error since the last call. */
int xdna_take_device_error(int* code, int* site, void* stream);

/* Self-test of the bounded device waits (no reference counterpart): launches one block whose wait on an
 * mbarrier that nothing arrives at gives up after limit_ns (1 us .. 2 s) of device time, exactly as the
 * waits inside every kernel of the library do, records XDNA_ERR_TIMEOUT at site 99 in the device error word
 * and returns; xdna_take_device_error then reports it. The GPU context stays usable. */
int xdna_selftest_wait_timeout(uint64_t limit_ns, void* stream);

/* ------------------------------------------------------------------ W8A8 linear
 * Per-row symmetric int8 quantisation: for each row r of x [rows, cols] (leading dim ldx, dtype
 * f32 / bf16 / f16): scale[r] = max(max_c |x[r,c]|, 1e-8) / 127 (the max taken in x's dtype),
 * xq[r,c] = clamp(round_half_even(float(x[r,c]) / scale[r]), -127, 127). IEEE division, no FMA.
 * Replaces R:torch_xdna/runtime.py:145-148 (_quant_rows), the quantise ops of
 * R:torch_xdna/runtime.py:366-368 (linear_int8) and the weight quantisation of QWeight
 * R:torch_xdna/runtime.py:59-66 (a weight is quantised as rows of [N, K]). */
int xdna_quant_rows_i8(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* xq,
                       int64_t ldq, float* scale, void* stream);

/* acc[M,N] = xq[M,K] . wq[N,K]^T in int32 on the tcgen05 tensor cores (both operands K-major).
 * y_dtype XDNA_I32: y receives acc (sx, sw, bias ignored).
 * y_dtype XDNA_F32 / XDNA_BF16 / XDNA_F16: y = (float(acc) * sx[m]) * sw[n] (+ float(bias[n])),
 *   rounded once to y_dtype (round to nearest even) -- the reference's dequantise order.
 * bias may be NULL; bias_dtype is its element type.
 * Replaces kernels.mm_i8 R:torch_xdna/kernels.py:172-192 as called by _npu_acc
 * R:torch_xdna/runtime.py:191-209 (and the CPU route torch._int_mm, R:torch_xdna/runtime.py:162-163),
 * fused with the dequantisation of R:torch_xdna/runtime.py:350-353, :370-374 and :429-432. */
int xdna_gemm_i8(const int8_t* xq, int64_t ldx, const int8_t* wq, int64_t ldw, int64_t M, int64_t N, int64_t K,
                 const float* sx, const float* sw, const void* bias, int bias_dtype, void* y, int y_dtype,
                 int64_t ldy, void* stream);

/* The kernel configuration xdna_gemm_i8 launches for an M x N output on the current device: *tile_n output
 * columns per tile (64, 128 or 256) and *pair = 1 when 256 x 256 tiles run on CTA pairs. Callers that
 * verify one launch per configuration (the reference's verify="first", R:torch_xdna/runtime.py:191-209)
 * key their checks with it. */
int xdna_gemm_i8_config(int64_t M, int64_t N, int* tile_n, int* pair);

/* ------------------------------------------------------------------ conv3x3
 * The implicit-GEMM conv reads activations as a zero-bordered NHWC int8 tensor
 * xp [N, H+2, W+2, Cp] (Cp = channels rounded up to a multiple of 16, pad channels zero), and
 * weights as wp [Co, 9, Cp] int8 (tap = 3*ky + kx, pad channels zero). */

/* Per-image quantisation fused with the layout change: for image n of x [N, C, H, W] (NCHW,
 * contiguous, f32 / bf16 / f16): sx[n] = max(max |x[n]|, 1e-8) / 127, and xp gets
 * clamp(round_half_even(float(x) / sx[n]), -127, 127) inside a zero border.
 * amax_scratch: N uint32 words of scratch this call clears and uses.
 * Replaces the quantise ops of conv3x3_int8, R:torch_xdna/conv.py:45-46, and the host-side
 * NCHW -> NPU layout packing of Triton-XDNA's conv3x3 host code. */
int xdna_conv_quant_nhwc(const void* x, int x_dtype, int64_t N, int64_t C, int64_t H, int64_t W, int8_t* xp,
                         int64_t Cp, float* sx, uint32_t* amax_scratch, void* stream);

/* The same quantisation for x in channels-last memory ([N, H, W, C], torch's channels_last layout of
 * an [N, C, H, W] tensor; 16-byte aligned): a streaming copy with no transpose. This is the layout the
 * XDNA_CONV_DEQUANT epilogue writes, so one conv's output feeds the next conv's quantise directly. */
int xdna_conv_quant_channels_last(const void* x, int x_dtype, int64_t N, int64_t C, int64_t H, int64_t W,
                                  int8_t* xp, int64_t Cp, float* sx, uint32_t* amax_scratch, void* stream);

/* The next conv's input straight from a conv's int8 output, with no float tensor in between: q [N, H, W, C]
 * (XDNA_CONV_Q_NHWC; uint8 when q_unsigned, else int8; C a multiple of 4) stands for the dequantised
 * y = float(q) * (scale[c] * sx_in[n]) (+ bias[c]) (then max(y, 0) when relu_after), computed with the
 * same f32 roundings as XDNA_CONV_DEQUANT. With pool, y is max-pooled 2x2 / stride 2 first (output
 * H / 2 x W / 2, rounded down: torch's max_pool2d(2)); pooling the codes is exact because y grows with q.
 * Then y is quantised per image exactly as xdna_conv_quant_nhwc does (sx_out[n] = max(amax, 1e-8) / 127,
 * round half even, saturate to +-127) into the bordered xp [N, H'+2, W'+2, Cp]. amax_scratch: N words.
 * Replaces the dequantise at the end of conv3x3_int8 R:torch_xdna/conv.py:47-50, the graph's relu and
 * max_pool2d, and the next conv3x3_int8's quantise R:torch_xdna/conv.py:45-46, for a chain of convs whose
 * intermediate activations have no other use (the int8 NHWC chaining the reference names as its largest
 * remaining cost). */
/* xdna_conv_quant_nhwc for a layer of C <= 7 input channels with the 3x3 stencil's taps packed into each
 * pixel's row: xp [N, H+2, W+2, Kp] (Kp = round_up(9 C, 16)), byte t * C + c of bordered pixel (yb, xb) is
 * the quantised x[n, c, yb - 2 + t / 3, xb - 2 + t % 3] (0 outside the image), the rest zeros. The same
 * per-image scale and quantised values as xdna_conv_quant_nhwc; the conv then runs with
 * XDNA_CONV_SINGLE_TAP and weights wp [Co, 1, Kp], byte t * C + c of row co = wq[co, c, t / 3, t % 3]. */
int xdna_conv_quant_taps(const void* x, int x_dtype, int64_t N, int64_t C, int64_t H, int64_t W, int8_t* xp,
                         int64_t Kp, float* sx, uint32_t* amax_scratch, void* stream);

/* The per-image quantisation of xdna_conv_quant_nhwc (same sx, same values) written as the stride phases a
 * stride-2 conv reads (XDNA_CONV_STRIDE2): xp [planes, N, Ho+2, Wo+2, Cp], Ho = ceil(H / 2), Wo = ceil(W / 2),
 * planes 4 (all phases, for the 3x3 conv) or 1 (the even-even phase, for the 1x1 conv). x [N, C, H, W] in
 * NCHW memory (x_channels_last 0) or channels-last memory (1). Every byte of xp is written (borders and pixels
 * past the input are zeros). amax_scratch: N words. */
int xdna_conv_quant_phases(const void* x, int x_dtype, int x_channels_last, int64_t N, int64_t C, int64_t H,
                           int64_t W, int planes, int8_t* xp, int64_t Cp, float* sx, uint32_t* amax_scratch,
                           void* stream);

/* The two halves of xdna_conv_quant_nhwc / xdna_conv_quant_channels_last, for an image split into strips of
 * rows over several GPUs, whose scale needs the max over every strip (combined between the two calls, e.g.
 * by an all-reduce of the words): xdna_conv_image_amax writes each image's max |x| as its f32 bit pattern
 * (amax [N], cleared first; per_image = C * H * W contiguous elements, NaN propagates); xdna_conv_quant_given_amax
 * quantises x [N, C, H, W] (NCHW, or channels-last memory with x_channels_last) into the bordered xp with
 * sx[n] = max(amax[n], 1e-8) / 127 from the given words. A strip's border rows are written as zeros: the
 * halo rows from its neighbours are copied over them afterwards. No reference counterpart (the reference
 * runs on one device); the arithmetic is that of R:torch_xdna/conv.py:45-46. */
int xdna_conv_image_amax(const void* x, int x_dtype, int64_t N, int64_t per_image, uint32_t* amax, void* stream);
int xdna_conv_quant_given_amax(const void* x, int x_dtype, int x_channels_last, int64_t N, int64_t C, int64_t H,
                               int64_t W, int8_t* xp, int64_t Cp, float* sx, const uint32_t* amax, void* stream);

int xdna_conv_quant_codes(const void* q, int q_unsigned, int64_t N, int64_t C, int64_t H, int64_t W,
                          const float* scale, const float* sx_in, const float* bias, int relu_after, int pool,
                          int8_t* xp, int64_t Cp, float* sx_out, uint32_t* amax_scratch, void* stream);

/* xdna_conv_quant_codes with the per-image maxima already known (amax [N], the bit patterns the producing
 * conv wrote with XDNA_CONV_NEXT_AMAX, XDNA_CONV_NEXT_POOL iff pool): one pass over the codes instead of two. */
/* xdna_conv_quant_codes into the image-pair layout XDNA_CONV_PAIRS reads: xp [N/2, H'+2, W'+2, 128], image n's
 * channels at bytes 64 * (n % 2) .. of each pair row. C = 64, N even. amax: N words; with amax_given the
 * per-image maxima the producing conv wrote (XDNA_CONV_NEXT_AMAX), else scratch this call fills. */
int xdna_conv_quant_codes_pairs(const void* q, int q_unsigned, int64_t N, int64_t C, int64_t H, int64_t W,
                                const float* scale, const float* sx_in, const float* bias, int relu_after, int pool,
                                int8_t* xp, float* sx_out, uint32_t* amax, int amax_given, void* stream);

/* The int32 bias of XDNA_CONV_BIAS_INT32: out[n][co] = rint(bias[co] / (sw[co] * sx[n])) in f32 (the product
 * and the quotient correctly rounded, rint to nearest even), clamped to [-2^29, 2^29], NaN -> 0. bias: Co
 * values of bias_dtype (f32 / bf16 / f16); sw: the layer's weight scales [Co]; sx: the images' scales [N]. */
int xdna_conv_bias_int32(const void* bias, int bias_dtype, const float* sw, const float* sx, int64_t N, int64_t Co,
                         int32_t* out, void* stream);

int xdna_conv_quant_codes_given_amax(const void* q, int q_unsigned, int64_t N, int64_t C, int64_t H, int64_t W,
                                     const float* scale, const float* sx_in, const float* bias, int relu_after,
                                     int pool, int8_t* xp, int64_t Cp, float* sx_out, const uint32_t* amax,
                                     void* stream);

/* xdna_conv_quant_nhwc without caller-provided scratch: the same inputs, outputs and results, but the
 * per-image max lives in a 16 KB array inside the library, so the call allocates nothing and takes no
 * scratch pointer. It has no counterpart in the reference (whose quantise runs on the CPU).
 * It is for callers that must not allocate device memory: plugins whose host framework hands them all
 * of their memory up front and forbids allocation while serving, and latency-bound serving loops that
 * cannot afford cudaMalloc's device-wide synchronisation.
 * Limits and behaviour:
 *   - at most 4096 images per call; more returns XDNA_ERR_INVALID with a message;
 *   - the first call on each device looks up the array's device address (cudaGetSymbolAddress, with
 *     that device current) and caches it; make that first call before any stream capture;
 *   - every call on a device shares the one array and clears the words it uses first; calls that
 *     overlap on the GPU (other streams, or other threads) race on it and must be serialised;
 *   - the array stays allocated on every GPU that loaded the library until the process exits. */
int xdna_conv_quant_nhwc_static(const void* x, int x_dtype, int64_t N, int64_t C, int64_t H, int64_t W, int8_t* xp,
                                int64_t Cp, float* sx, void* stream);

/* NCHW int8 xq [N, C, H, W] (the xdna::conv3x3 op's input) -> bordered NHWC xp as above. */
int xdna_conv_pack_input(const int8_t* xq, int64_t N, int64_t C, int64_t H, int64_t W, int8_t* xp, int64_t Cp,
                         void* stream);

/* int8 weights wq [Co, Ci, 3, 3] (contiguous) -> wp [Co, 9, Cp]. */
int xdna_conv_pack_weight(const int8_t* wq, int64_t Co, int64_t Ci, int8_t* wp, int64_t Cp, void* stream);

/* 3x3 / stride 1 / padding 1 conv of xp by wp on the int8 tensor cores, int32 sums, and one of the
 * epilogues XDNA_CONV_Q / XDNA_CONV_DEQUANT / XDNA_CONV_CALIBRATE (see above). Rounding of the
 * requantise is round half up via an arithmetic shift, then saturation: [-128,127] int8, or
 * [0,255] uint8 when relu != 0. Output `out`: NCHW [N, Co, H, W] XDNA_I8 / XDNA_U8 for XDNA_CONV_Q;
 * channels-last [N, H, W, Co] XDNA_F32 / XDNA_BF16 / XDNA_F16 for XDNA_CONV_DEQUANT. For XDNA_CONV_CALIBRATE
 * only image 0 is computed and acc_max (one int32, cleared by this call) receives the maximum.
 * XDNA_CONV_Q_NHWC writes the same q as XDNA_CONV_Q, channels-last [N, H, W, Co] (XDNA_I8 / XDNA_U8).
 * Replaces tl.extra.npu.conv3x3.Conv3x3(...)(xq) as used by ConvLayer.npu
 * R:torch_xdna/conv.py:78-84,94-103, the CPU integers ConvLayer.cpu R:torch_xdna/conv.py:86-92,
 * the calibration sums of ConvLayer.calibrate R:torch_xdna/conv.py:71-76, and (DEQUANT) the
 * dequantise ops of conv3x3_int8 R:torch_xdna/conv.py:47-50. */
int xdna_conv3x3_i8(const int8_t* xp, const int8_t* wp, int64_t N, int64_t Ci, int64_t Cp, int64_t Co, int64_t H,
                    int64_t W, int mode, int shift, int relu, const float* scale, const float* sx, const void* bias,
                    int bias_dtype, void* out, int out_dtype, int32_t* acc_max, void* stream);

/* ------------------------------------------------------------------ the Qwen3 stack (bf16)
 * Replaces tl.extra.npu.qwen3_stack.Qwen3Stack(...)(x0, x1), the one-launch NPU program called by
 * stack.run R:torch_xdna/stack.py:360-389, for Qwen3-0.6B's shapes (hidden 1024, 16 query / 8 kv heads
 * of 128, MLP 3072), any depth, and extends it to causal and general masks and any length. */

/* epilogues of xdna_gemm_bf16 */
#define XDNA_GEMM_F32ACC 0 /* out = acc (+ bias[n]) in out_dtype */
#define XDNA_GEMM_RESID 1  /* resid[m, n] += acc (f32, in place) */
#define XDNA_GEMM_SWIGLU 2 /* B rows interleave 32 gate / 32 up rows: out[m, j] = bf16(silu(gate) * up), N/2 columns */
#define XDNA_GEMM_QKV 3    /* N = 4096 = q 2048 | k 1024 | v 1024 columns: out [M, 3072] bf16 gets q and k after the
                              per-head RMSNorm (q_norm / k_norm) and RoPE at position m % seq_len; vt [1024, ldvt]
                              bf16 gets v transposed */

/* attention masks */
#define XDNA_MASK_CAUSAL 0 /* key <= query */
#define XDNA_MASK_PREFIX 1 /* lens[b]: the first n positions see each other, later ones only themselves */
#define XDNA_MASK_BOOL 2   /* mask [B, 1|16, L, L] bytes, nonzero = may attend */
#define XDNA_MASK_NONE 3

/* One decoder layer's weights, bf16 matrices (row-major [out, in]) and f32 norm weights. */
typedef struct {
  const void* w_qkv;        /* [4096, 1024]: q_proj (2048 rows), k_proj (1024), v_proj (1024) */
  const void* w_o;          /* [1024, 2048] */
  const void* w_gu;         /* [6144, 1024]: gate_proj / up_proj interleaved in blocks of 32 rows */
  const void* w_down;       /* [1024, 3072] */
  const float* input_norm;  /* [1024] */
  const float* post_norm;   /* [1024] */
  const float* q_norm;      /* [128] */
  const float* k_norm;      /* [128] */
} xdna_qwen3_layer;

/* y [rows, D] bf16 = x * rsqrt(mean(x^2) + eps) * w, x f32 (D = 128, 512 or 1024). */
int xdna_rmsnorm_bf16(const float* x, int64_t rows, int64_t D, const float* w, float eps, void* y, void* stream);

/* x [tokens, D] f32 = table[ids] (bf16 or f32 table [vocab, D]); ids outside [0, vocab) give zeros and
 * record XDNA_ERR_INVALID in the device error word. Replaces the embed_tokens lookup of the model. */
int xdna_embed(const int64_t* ids, int64_t tokens, const void* table, int table_dtype, int64_t vocab, int64_t D,
               float* x, void* stream);

/* C [M, N] = A [M, K] . B [N, K]^T, bf16 operands (row pitches lda / ldb in elements, multiples of 8),
 * f32 accumulation on the tcgen05 tensor cores, with one of the XDNA_GEMM_* epilogues. XDNA_GEMM_QKV's
 * rope_cos / rope_sin: f32 tables of the model's inverse frequencies at positions 0..seq_len-1 in the layout
 * [16, seq_len, 4]: frequency d of position p at index (d / 4) * seq_len * 4 + p * 4 + d % 4. */
int xdna_gemm_bf16(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N, int64_t K, int mode,
                   void* out, int out_dtype, int64_t ldo, const void* bias, int bias_dtype, float* resid, int64_t ldr,
                   void* vt, int64_t ldvt, const float* rope_cos, const float* rope_sin, const float* q_norm,
                   const float* k_norm, int64_t seq_len, float eps, void* stream);

/* The head GEMM of a column-parallel stack, fused with the all-gather of its input: out [n_parts *
 * rows_per_part, N] = A . b^T (+ bias) with the XDNA_GEMM_F32ACC epilogue, where rows [i * rows_per_part,
 * (i + 1) * rows_per_part) of A are a_parts[i] ([rows_per_part, K] bf16, pitch lda) — device pointers
 * that may belong to other GPUs of the box (peer memory opened with xdna_ipc_open), read by the GEMM's
 * TMA producer over NVLink while the tensor cores run, instead of a separate all-gather. rows_per_part
 * must be a multiple of 256. maps: device memory for n_parts tensor maps (128 bytes each, 64-byte
 * aligned), written by this call (stream-ordered). The caller orders the parts' writes before this call
 * on every GPU (e.g. a barrier collective). Replaces the all-gather followed by the head GEMM of the
 * column-parallel head on several GPUs, which the reference (one device) does not have. */
int xdna_gemm_bf16_gather(const void* const* a_parts, int n_parts, int64_t rows_per_part, int64_t lda, const void* b,
                          int64_t ldb, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo, const void* bias,
                          int bias_dtype, void* maps, void* stream);

/* CUDA IPC for xdna_gemm_bf16_gather's peer parts (no reference counterpart; the only entry points
 * that allocate): a dedicated device allocation that can be shared, its release; the 64-byte handle of
 * such an allocation; the device pointer of another process's allocation on this box (NVLink peer
 * access enabled) and its release. */
int xdna_ipc_alloc(size_t bytes, void** dev_ptr);
int xdna_ipc_free(void* dev_ptr);
int xdna_ipc_handle(const void* dev_ptr, void* handle64);
int xdna_ipc_open(const void* handle64, void** dev_ptr);
int xdna_ipc_close(void* dev_ptr);

/* out [B*L, 2048] bf16 = softmax(q k^T / sqrt(128) + mask) v for 16 query heads over 8 kv heads (GQA),
 * q and k read from qk [B*L, 3072] (the XDNA_GEMM_QKV output), v from vt [1024, ldvt]. */
int xdna_attention(const void* qk, const void* vt, int64_t ldvt, void* out, int64_t B, int64_t L, int mask_kind,
                   const int32_t* lens, const uint8_t* mask, int mask_heads, void* stream);

/* Bytes of workspace xdna_qwen3_stack needs for B sequences of L tokens. */
size_t xdna_qwen3_stack_workspace(int64_t B, int64_t L);

/* The whole stack: x [B*L, 1024] f32 (the hidden states, updated in place as the residual stream)
 * through n_layers decoder layers, the final RMSNorm and the head: out [B*L, head_n] (row pitch ldo)
 * = h Whead^T (+ bias) in out_dtype. rope_cos / rope_sin: f32 tables of the model's inverse frequencies
 * at positions 0..L-1, laid out [16, L, 4] as for xdna_gemm_bf16. With out == NULL the head is skipped and the final-normed hidden
 * states [B*L, 1024] bf16 are left at the start of the workspace. */
int xdna_qwen3_stack(const xdna_qwen3_layer* layers, int n_layers, const float* final_norm, const void* head_w,
                     int64_t head_n, const void* head_bias, int head_bias_dtype, const float* rope_cos,
                     const float* rope_sin, float eps, float* x, int64_t B, int64_t L, int mask_kind,
                     const int32_t* lens, const uint8_t* mask, int mask_heads, void* out, int out_dtype, int64_t ldo,
                     void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------ generation
 * From prompts to the next token (no reference counterpart: the reference answers with the logits of whole
 * sequences). Head dimensions 64 and 128, bf16 or f16, any number of query heads per key head up to 128;
 * strides are in elements, positive multiples of 8, bases 16-byte aligned. Scores, weights and sums are f32, weights
 * enter the sums over V rounded to the operands' type. */

/* Causal attention over packed sequences: out [tokens, hq, d] (contiguous) of q [tokens, hq, d], k and v
 * [tokens, hkv, d] with the strides *_st of a token and *_sh of a head. Sequence i is the tokens
 * cu_seqlens[i] .. cu_seqlens[i + 1] - 1 (n_seqs + 1 ascending device words); a token attends to the tokens of its
 * sequence up to itself. Words outside [0, tokens] or out of order are clamped; tokens of no sequence give zeros,
 * and so do rows of which every score is -inf.
 * 0 < scale <= 2.3e38. workspace: xdna_packed_attention_workspace bytes, 256-byte aligned. */
size_t xdna_packed_attention_workspace(int64_t n_seqs, int64_t tokens, int64_t hq, int64_t hkv);
int xdna_packed_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                          const void* v, int64_t v_st, int64_t v_sh, const int32_t* cu_seqlens, int64_t n_seqs,
                          int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int dtype, float scale, void* out,
                          void* workspace, size_t workspace_bytes, void* stream);

/* One decode step's attention of B sequences that share a prefix: out [B, hq, d] (contiguous), row b's softmax over
 * the P prefix keys pk / pv [P, hkv, d] and the first lens[b] (clamped to 0..S) of its own ck / cv [B, S, hkv, d].
 * A row without any key, or with scores of -inf alone, gives zeros. Sums over V are of weights up to 2^8 before the
 * division by their sum: bf16 values for which they pass 3.4e38 overflow. How the work is split over the GPU goes by S,
 * the lengths being on the device: a cache with much more room than it holds makes a call with a prefix slower, and is
 * better passed cut to about its longest sequence. workspace: xdna_prefix_attention_workspace bytes, 256-byte aligned. */
size_t xdna_prefix_attention_workspace(int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d);
int xdna_prefix_attention(const void* q, int64_t q_sb, int64_t q_sh, const void* pk, int64_t pk_st, int64_t pk_sh,
                          const void* pv, int64_t pv_st, int64_t pv_sh, const void* ck, int64_t ck_sb, int64_t ck_st,
                          int64_t ck_sh, const void* cv, int64_t cv_sb, int64_t cv_st, int64_t cv_sh,
                          const int32_t* lens, int64_t B, int64_t P, int64_t S, int64_t hq, int64_t hkv, int64_t d,
                          int dtype, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream);

/* 4-bit weights. A weight [N, K] is codes [N, K' / 2] bytes (K' = K rounded up to 128, padded with code 8) and
 * scales [N, ceil(K / group)] (bf16 or f16; group 32, 64 or 128): w = (code - 8) * scale. A block of 128 columns is
 * 16 little-endian 32-bit words; the word at place 4 t + w holds columns 32 w + 8 t .. + 7, in the order
 * 0, 2, 4, 6, 1, 3, 5, 7 from the lowest four bits. xdna_w4_pack quantises w (f32 / bf16 / f16, row pitch ldw):
 * scale = max |w| of the group / 7, code = clamp(rint(w / scale), -8, 7) + 8. A group with a NaN or an infinity has the
 * scale NaN, so it shows in the results; f16 scales hold groups of max |w| from 2e-7 (below: zeros) to 4.5e5 (above: an
 * infinite scale, whose results are NaN). */
int xdna_w4_pack(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ldw, int group, uint8_t* codes,
                 void* scales, int scale_dtype, void* stream);

/* y [M, N] = x [M, K] . w^T (+ bias) for such a weight, f32 sums, rounded once to x's type (f32 / bf16 / f16). */
int xdna_linear_w4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* codes,
                   const void* scales, int scale_dtype, int group, int64_t N, const void* bias, int bias_dtype,
                   void* y, int64_t ldy, void* stream);

/* The logits [B, V] of the next token after penalties, bias and mask, in f32 rounded once to their type. For
 * row b and token v, with `seen` = v is among the row's first lens[b] of tokens [B, T] (32 or 64-bit; ids outside
 * [0, V) count for nothing) and c = how often it is among those from prompt_lens[b] on:
 *   l = seen ? (l > 0 ? l / repetition[b] : l * repetition[b]) : l;  l -= frequency[b] * c + (c > 0) * presence[b];
 *   l += bias[b * ld_bias + v] (ld_bias 0: one for all rows);  l = bit v of mask[b * ld_mask + v / 32] ? l : -inf.
 * At most 65535 rows; repetition at least 2^-126 (the quotient is a product with its reciprocal, one unit of f32 off).
 * Each of tokens, lens (then T), prompt_lens (then 0), repetition, presence, frequency, bias and mask may be NULL.
 * out must not overlap logits. */
int xdna_process_logits(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld_in, const void* tokens,
                        int token_bytes, int64_t T, int64_t ld_tokens, const int32_t* lens,
                        const int32_t* prompt_lens, const float* repetition, const float* presence,
                        const float* frequency, const float* bias, int64_t ld_bias, const uint32_t* mask,
                        int64_t ld_mask, void* out, int64_t ld_out, void* stream);

/* ------------------------------------------------------------------ a decoder layer around its products
 * No reference counterpart. Strides are in elements unless said otherwise; norms' weights are f32, bf16 or f16. */

/* out [T, H, D] (contiguous, x's type f32 / bf16 / f16) = x [T, H, D] with the first R = 2 * n_freq entries of each head
 * turned: pairs (p, p + R / 2), or (2 p, 2 p + 1) with interleaved, by the angle positions[t] * inv_freq[p] (in 64 bits),
 * times factor; the others stay. norm != NULL: each head is first divided by the root of its mean square (plus eps) and
 * multiplied with the weights norm[h * norm_sh ..] (norm_sh 0: one for all heads). D a multiple of 8, up to 256; x_st,
 * x_sh (of a token, of a head) and norm_sh multiples of 8; x, out and norm 16-byte aligned; positions 32 or 64 bits.
 * Sums and products are f32, rounded once. */
int xdna_rotary(const void* x, int dtype, int64_t T, int64_t H, int64_t D, int64_t x_st, int64_t x_sh,
                const void* positions, int position_bytes, const float* inv_freq, int64_t n_freq, float factor,
                int interleaved, const void* norm, int norm_dtype, int64_t norm_sh, float eps, void* out, void* stream);

/* The norms around a block, its gate and its residual: for each of `rows` rows of D (up to 16384) entries, in f32,
 *   z = post ? y / sqrt(mean y^2 + eps) * post : y;  x' = x + scale * gate * z;  h = x' / sqrt(mean x'^2 + eps) * weight
 * x_out = x' in x's type, h in y's type (h is of x' before its rounding), both contiguous [rows, D] and apart from the
 * inputs. post and gate may be NULL; ld_gate 0: one gate for all rows. Any row pitches and alignments; pieces of 16 bytes
 * where all are multiples of 8 elements and 16-byte aligned. */
int xdna_add_norm(const void* x, int x_dtype, int64_t ldx, const void* y, int y_dtype, int64_t ldy, int64_t rows,
                  int64_t D, const void* weight, int weight_dtype, const void* post, int post_dtype, const void* gate,
                  int gate_dtype, int64_t ld_gate, float scale, float eps, void* x_out, void* h, void* stream);

/* A cache of keys and values in pages and 8 bits: codes [pages][hkv][page][d] bytes (format XDNA_I8 or XDNA_E4M3; the
 * last three dimensions contiguous, kc_sp / vc_sp bytes from page to page, multiples of 16; page 16, 32, 64 or 128; d 64
 * or 128) and scales [pages][hkv] f32 (ks_sp / vs_sp elements from page to page): x = code * scale, one scale, zero or
 * more, for a head's part of a page (a block). table [n_seqs][max_pages] (int32, row pitch ld_table): the page of a
 * sequence's tokens i * page .. ; an entry outside [0, pages) is no page.
 *
 * xdna_cache_append puts new tokens k, v [tokens, hkv, d] (bf16 / f16) behind the starts[i] that sequence i has in the
 * cache: token i is sequence i's next one (cu_seqlens NULL, n_seqs == tokens), or tokens cu_seqlens[i] ..
 * cu_seqlens[i + 1] - 1 are sequence i's next ones (ascending; words outside [0, tokens] are clamped). The keys, after
 * k_norm where given, are turned to their place in the sequence as by xdna_rotary. A block's scale is the least 2^e >=
 * 2^-126 with max |x| <= 127 * 2^e (int8) or 448 * 2^e (e4m3) over its tokens; where older tokens in it had a larger one
 * that stays (one that is no power of two: the next above it, to which their codes are rounded), where they had a smaller
 * one their codes are rounded to the new one. A page whose first slot is written starts anew. A block that is given an
 * infinity or a NaN, or whose older scale is one, above 2^126 or below zero, has the scale NaN until then, and code 0 for
 * the new tokens.
 * Slots behind a sequence's last token, and all other pages, are left as they were. Tokens without a page, and sequences
 * with starts[i] < 0, are not stored. No two sequences of a call may write to one page. q [tokens, hq, d] may be NULL;
 * else q_out [tokens, hq, d] = q, after q_norm, turned to its tokens' places (zero where starts[i] < 0 and for tokens of
 * no sequence). Rows of k, v and q as for xdna_rotary. */
int xdna_cache_append(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, int dtype,
                      int64_t tokens, int64_t hkv, int64_t d, void* k_codes, int64_t kc_sp, void* v_codes, int64_t vc_sp,
                      int format, float* k_scales, int64_t ks_sp, float* v_scales, int64_t vs_sp, int64_t pages,
                      int64_t page, const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* starts,
                      const int32_t* cu_seqlens, int64_t n_seqs, const float* inv_freq, int64_t n_freq, float factor,
                      int interleaved, const void* k_norm, int k_norm_dtype, int64_t k_norm_sh, float eps, const void* q,
                      int64_t q_st, int64_t q_sh, int64_t hq, const void* q_norm, int q_norm_dtype, int64_t q_norm_sh,
                      void* q_out, void* stream);

/* Attention over such a cache: out [B, T, hq, d] (contiguous) of q [B, T, hq, d] (bf16 / f16; strides q_sb, q_st, q_sh),
 * the last T tokens of each sequence: token t attends to the first lens[b] - T + t + 1 tokens in the cache (lens clamped
 * to 0 .. max_pages * page, which is below 2^30), without those that have no page. A row without any, or with scores of
 * -inf alone, is zero. Scores and sums are f32; the weights that meet V are f16 with an exponent of their own per block
 * (terms below 2^-26 of a row's largest lose bits, those below 2^-37 are lost). The work is shared out by the lengths, on
 * the device, in one of three manners by B, the heads and max_pages * page. T is meant to be small: every 16 / (hq / hkv)
 * tokens the cache is read once more. Codes of e4m3 are numbers. workspace: xdna_paged_attention_workspace bytes for
 * most_keys = max_pages * page, 256-byte aligned (0 bytes: NULL). */
size_t xdna_paged_attention_workspace(int64_t B, int64_t T, int64_t hq, int64_t hkv, int64_t d, int64_t most_keys);
int xdna_paged_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, int64_t B, int64_t T,
                         int64_t hq, int64_t hkv, int64_t d, const void* k_codes, int64_t kc_sp, const void* v_codes,
                         int64_t vc_sp, int format, const float* k_scales, int64_t ks_sp, const float* v_scales,
                         int64_t vs_sp, int64_t pages, int64_t page, const int32_t* table, int64_t ld_table,
                         int64_t max_pages, const int32_t* lens, float scale, void* out, void* workspace,
                         size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* XDNA_B200_H */
