/*
 * rocket_fp8.h — matrix products in 8-bit floating point on MI355X, with one fp32 scale for each block of
 * 128, and the quantisation that makes their operands (additions; the reference library has no
 * counterpart: its 8-bit path is the integer one of rocket_matmul.h).
 *
 *   rocket_quantize_rows_fp8*          activations to codes and scales
 *   rocket_quantize_glu_fp8*           the same of gated rows, act(gate) * up
 *   rocket_matmul_fp8_block*           C = A * B^T of such codes
 *   rocket_matmul_fp8_block_grouped*   the same for experts, whose rows the GPU counted
 *
 * Codes are e4m3 (sign, 4 bits of exponent of bias 7, 3 of mantissa; largest 448, no infinity, 0x7f and
 * 0xff NaN), one a byte. A row of K codes of activations has ceil(K / 128) scales; weights [N][K] have one
 * scale for each 128 rows by 128 values, [ceil(N / 128)][ceil(K / 128)] (the last of each may be a part of a
 * block). A code c stands for c * scale.
 *
 * As everywhere in this library: operands may be host or device pointers; device memory is used in place where it
 * is 16-byte aligned (src_row, expert_off and n_rows: 4-byte) and staged where it is not, which a captured call
 * does not allow; fd < 0 runs the host path (every operand host memory then), whose products are fp64; handles run
 * asynchronously where rocket_hip_set_mode says so, and a call returns 0 or a negative rocket_status: -1 for a bad
 * argument, before anything is launched. Results must not lie over a call's other operands or each other (-1).
 * Strides count elements. A product of few rows and a long K may be summed in slices of K that lie in scratch of the handle:
 * a captured one on a handle that has none yet takes none (its sums are in another order then), and graphs that hold it are replayed in the order of the
 * handle's stream.
 */
#ifndef ROCKET_FP8_H
#define ROCKET_FP8_H

#include <stddef.h>
#include <stdint.h>

#include "rocket_matmul.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- quantisation ----
 * For each row and each 128 of its values (the last group may be shorter), in fp32, divisions IEEE-rounded:
 *     a        = max(max |x|, 2^-100)
 *     scale    = a / 448
 *     code     = e4m3(clamp(x * (448 / a), -448, 448))        rounded to nearest even
 * A NaN gives a NaN code (0x7f or 0xff) and does not count in the maximum; an infinity makes its group's scale infinite,
 * so that products with the group are NaN.
 * Row m of A begins at A + m * a_rs. Results are dense: Aq[M][K], a_scale[M][ceil(K / 128)].
 * K and the strides are multiples of 8, 8 <= K <= 65536, K <= stride, M * stride <= 2^40. */
int rocket_quantize_rows_fp8(int fd, int M, int K, const float *A, int64_t a_rs, uint8_t *Aq, float *a_scale);
int rocket_quantize_rows_fp8_fp16(int fd, int M, int K, const _Float16 *A, int64_t a_rs, uint8_t *Aq, float *a_scale);

/* Gated rows: x = act(gate) * up in fp32 (act: ROCKET_ACTIVATION_SILU or _GELU, as the FFN block entries compute
 * them), of rows gate + m * rs and up + m * rs (one product may have written both side by side). n_rows: NULL, or one
 * int32: rows from *n_rows on are not read, and their results left as they were (an expert layer's rows behind the
 * last expert's: &expert_off[n_expert] of rocket_moe_route). Other rules as above. */
int rocket_quantize_glu_fp8(int fd, int M, int K, const float *gate, const float *up, int64_t rs, int act, const int32_t *n_rows,
                            uint8_t *Aq, float *a_scale);
int rocket_quantize_glu_fp8_fp16(int fd, int M, int K, const _Float16 *gate, const _Float16 *up, int64_t rs, int act,
                                 const int32_t *n_rows, uint8_t *Aq, float *a_scale);

/* ---- products ----
 * C[m][n] = sum over blocks b of a_scale[m][b] * b_scale[n / 128][b] * (sum over k in b of A[m][k] * B[n][k]).
 * A [M][K] and B [N][K] codes, dense; M, N >= 1, K a multiple of 16, 16 <= K <= 65536.
 * A block's two scales are multiplied first, in fp32 (fd < 0: in fp64), and have to keep their product from 2^-126 up to 2^128: a smaller one
 * loses bits of its block's sum (none where that is 0, as of a group of zeros), a larger one is an infinity, which makes a sum of 0 a NaN.
 * The entries with fp32 results widen the codes, so that products and sums are fp32's. Those with fp16 results
 * (rounded once; an fp32 sum past fp16 is an infinity) may use the matrix unit's 8-bit products, twice as fast: of each
 * eight neighbouring k (8 i .. 8 i + 7) it cuts every product at 2^-13 of the largest one's power of two and sums the rest in
 * fp32, which for random rows is some 1.5e-5 of a result, a fourteenth of its rounding. */
int rocket_matmul_fp8_block(int fd, int M, int K, int N, const uint8_t *A, const float *a_scale, const uint8_t *B, const float *b_scale,
                            float *C);
int rocket_matmul_fp8_block_f16out(int fd, int M, int K, int N, const uint8_t *A, const float *a_scale, const uint8_t *B,
                                   const float *b_scale, _Float16 *C);

/* The products of n_expert experts with weights B[n_expert][N][K], b_scale[n_expert][ceil(N / 128)][ceil(K / 128)].
 * expert_off[n_expert + 1], ascending from 0: rows [expert_off[e], expert_off[e + 1]) of C[rows][N] are expert e's;
 * rows from expert_off[n_expert] on are left as they were. `rows` sizes the launch: offsets count as if cut to [0, rows],
 * and a call whose offsets descend gives no defined result (it stays inside its operands). Row r of C is made of
 * row src_row[r] of A[a_rows] (a row outside [0, a_rows) gives zeros, whatever the weights hold), or, src_row NULL, of row r (a_rows >= rows then).
 * expert_off and src_row may be device memory that an earlier call of the stream writes, so that nothing waits
 * for the host and a captured call is replayed with other counts. 1 <= n_expert <= 1024; a_rows * K < 2^31.
 * n_expert * N * K may be past 2^32. */
int rocket_matmul_fp8_block_grouped(int fd, int n_expert, int rows, int a_rows, int K, int N, const uint8_t *A, const float *a_scale,
                                    const int32_t *src_row, const int32_t *expert_off, const uint8_t *B, const float *b_scale, float *C);
int rocket_matmul_fp8_block_grouped_f16out(int fd, int n_expert, int rows, int a_rows, int K, int N, const uint8_t *A,
                                           const float *a_scale, const int32_t *src_row, const int32_t *expert_off, const uint8_t *B,
                                           const float *b_scale, _Float16 *C);

#ifdef __cplusplus
}
#endif
#endif /* ROCKET_FP8_H */
