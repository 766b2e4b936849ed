/*
 * llmopt_float8.h -- C ABI of the decoder's steps in 8-bit floating point in libllmopt_qlinear.so (gfx950): quantizing rows
 * and weights, RMSNorm with a quantized output, the projections and the gated MLP product. Same conventions as
 * llmopt_qlinear.h: device pointers owned by the caller, `stream` a hipStream_t as void*, LLMOPT_OK or a negative
 * LLMOPT_ERR_* code, dtype codes LLMOPT_DTYPE_*; the message of a failed call of this header is in
 * llmopt_f8_last_error() (per host thread). No counterpart in the reference, whose linears hold integer codes.
 *
 * Codes are e4m3 (OCP: largest number 448, no infinities), one byte each, rows of `ld*` bytes; scales are e8m0, one byte
 * each: byte b is 2^(b - 127), 255 NaN. A code stands for code x scale:
 *   rows (activations)  codes [rows, cols], scales [rows, ceil(cols / 128)]: one per row and 128 columns
 *   weights             codes [N, K], scales [ceil(N / 128), ceil(K / 128)]: one per block of 128 x 128
 * Quantizing a group whose largest magnitude is amax gives the scale 2^e for the smallest e >= -127 with amax <= 448 2^e,
 * and a number x the code x / 2^e rounded to nearest, ties to even. A group that holds an infinity or NaN gets the scale
 * NaN and codes 0: it reads as NaN.
 */
#ifndef LLMOPT_FLOAT8_H_
#define LLMOPT_FLOAT8_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

const char* llmopt_f8_last_error(void);

/*
 * Quantizes x [rows, cols] (F32, F16 or BF16, row stride ldx elements) into codes (row stride ldc bytes) and scales (row
 * stride lds elements). block_rows 1: a scale per row and 128 columns; 128: one per block of 128 x 128.
 */
int llmopt_f8_quantize(const void* x, int64_t ldx, int dtype, int64_t rows, int64_t cols, int64_t block_rows,
                       void* codes, int64_t ldc, void* scales, int64_t lds, void* stream);

/*
 * The residual add and RMSNorm of llmopt_rmsnorm (llmopt_model.h) with a quantized output: h = residual + x rounded to
 * dtype and written to h_out (residual null: h = x, h_out not used), y = h rsqrt(mean(h^2) + eps) weight in fp32,
 * quantized by rows without another rounding. x, residual, h_out [rows, hidden] and weight [hidden] of dtype F16 or BF16
 * (F32: LLMOPT_ERR_UNSUPPORTED). h_out may be residual or x, otherwise it shares no memory with them.
 */
int llmopt_f8_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* h_out, int64_t ldh,
                      const void* weight, void* codes, int64_t ldc, void* scales, int64_t lds, int64_t rows,
                      int64_t hidden, float eps, int dtype, void* stream);

/* Bytes of workspace that llmopt_f8_linear uses to split K (0: no split), for 16-byte aligned rows. */
size_t llmopt_f8_linear_workspace(int64_t M, int64_t N, int64_t K);

/*
 * y [M, N] (F16 or BF16, row stride ldy elements; F32: LLMOPT_ERR_UNSUPPORTED) = x w^T + bias of x [M, K] quantized by rows
 * and a weight [N, K]; bias [N] of y's dtype, may be null. Products are exact, and added by the matrix cores in fp32 but for
 * this: of the products of eight neighbouring columns, what is below 2^-13 of the largest is dropped, so sums are off by 1.5e-5 to
 * 2.7e-5 of their typical size, up to 1e-4 where a few channels are 100 times as strong as the rest and more (hence no
 * F32 output). Rounded once. Rows that are no multiples of 16 bytes, or not
 * aligned to them, run on a slower kernel. With less workspace than llmopt_f8_linear_workspace asks for, K is not split
 * (correct, slower for few tokens).
 */
int llmopt_f8_linear(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* w, int64_t ldw, const void* w_scales, int64_t ldws, const void* bias, void* y,
                     int64_t ldy, int64_t N, int out_dtype, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace with which llmopt_f8_swiglu is fastest (0: it uses none). */
size_t llmopt_f8_swiglu_workspace(int64_t M, int64_t N, int64_t K);

/*
 * silu(x gate^T) * (x up^T), with silu(g) = g / (1 + exp(-g)) in fp32 on the fp32 sums, quantized by rows into codes [M, N]
 * and scales. A group's largest magnitude is summed again in fp32 where a border of the scales is within 2^-10 of it, more
 * than sums were found to be off by, so that its scale is that of exact sums; where more than 16 different numbers that one wave
 * holds are next to a border (equal features), it may be that of the matrix cores' sums. x as in llmopt_f8_linear, gate and up
 * weights [N, K]. With less workspace than llmopt_f8_swiglu_workspace
 * asks for, another kernel runs (correct, slower).
 */
int llmopt_f8_swiglu(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* gate, int64_t ldg, const void* gate_scales, int64_t ldgs, const void* up, int64_t ldu,
                     const void* up_scales, int64_t ldus, int64_t N, void* codes, int64_t ldc, void* scales,
                     int64_t lds, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LLMOPT_FLOAT8_H_ */
