/*
 * rocket_layer.h — what stands between the products of a layer's feed-forward side on MI355X (additions; the
 * reference library has no counterpart):
 *
 *   rocket_add_norm_*      a block's result joins the residual stream: its norm, gate and scale, the sum, and
 *                          the next block's norm, whose rows may come out as the codes that rocket_fp8.h multiplies
 *   rocket_moe_add_norm_*  the same where the block is a layer of experts: their rows' weighted sum first
 *   rocket_moe_route_*     which experts a token goes to, with which weights, and the rows sorted by expert
 *
 * Operands, handles, streams, captured calls and errors as in rocket_fp8.h.
 */
#ifndef ROCKET_LAYER_H
#define ROCKET_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "rocket_matmul.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms before and after a block ----
 * With N(v; w, eps) = v / sqrt(mean(v^2) + eps) * w over a row's H values (eps < 0: N(v) = v, and w must be NULL; w NULL:
 * ones), for each row m < M, in fp32:
 *     z  = N(y[m]; w_post, eps_post)                               the block's result, y + m * y_rs
 *     h' = h[m] + alpha * gate[m / gate_every] * z                 (gate NULL: ones; y NULL: h' = h[m])
 *     x  = N(h'; w_pre, eps_pre)                                   of h' before it is rounded
 * Results, each of which may be NULL, but not all: h_out[M][H] (h' in h's type; it may be h itself, if y is not), x[M][H] in fp16, and xq[M][H] with
 * x_scale[M][ceil(H / 128)] (both or neither), x's codes and scales as rocket_quantize_rows_fp8 makes them of the
 * unrounded x. h[M][H], gate[ceil(M / gate_every)][H]: gate_every 1 is a gate for each row, the tokens of a
 * sequence one for each sequence, M or more one for all. y_rs >= H, a multiple of 8, M * y_rs <= 2^40.
 * H a multiple of 8, 8 <= H <= 16384; eps not NaN, alpha finite. An fp16 h' past fp16's range is an infinity.
 * A norm holds for rows of any finite size, also where their squares pass fp32's range; 0 / 0 (a row of zeros under eps 0) is NaN. A row with an
 * infinity is NaN there and 0 elsewhere, a row with a NaN is NaN. */
int rocket_add_norm_fp16(int fd, int M, int H, const _Float16 *h, const _Float16 *y, int64_t y_rs, const _Float16 *w_post, float eps_post,
                         const _Float16 *gate, int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, _Float16 *h_out,
                         _Float16 *x, uint8_t *xq, float *x_scale);
int rocket_add_norm_f32(int fd, int M, int H, const float *h, const float *y, int64_t y_rs, const _Float16 *w_post, float eps_post,
                        const _Float16 *gate, int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, float *h_out,
                        _Float16 *x, uint8_t *xq, float *x_scale);

/* The same with
 *     y[m] = sum over j < top_k of weight[m][j] * Y[slot[m][j]]  (+ shared[m] where shared is not NULL),
 * Y[rows][H], slot and weight [M][top_k]. A slot outside [0, rows) adds nothing, whatever its weight. 1 <= top_k <= 32. */
int rocket_moe_add_norm_fp16(int fd, int M, int H, const _Float16 *h, int rows, int top_k, const _Float16 *Y, const int32_t *slot,
                             const float *weight, const _Float16 *shared, const _Float16 *w_post, float eps_post, const _Float16 *gate,
                             int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, _Float16 *h_out, _Float16 *x,
                             uint8_t *xq, float *x_scale);
int rocket_moe_add_norm_f32(int fd, int M, int H, const float *h, int rows, int top_k, const float *Y, const int32_t *slot,
                            const float *weight, const float *shared, const _Float16 *w_post, float eps_post, const _Float16 *gate,
                            int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, float *h_out, _Float16 *x,
                            uint8_t *xq, float *x_scale);

/* ---- routing ----
 * Scores of token m's logits l[e] = logits[m * rs + e], e < E, in fp64: p = softmax(l) over all experts, or
 * p = 1 / (1 + exp(-l)); choices c = p + bias[e] (bias NULL: c = p). An expert whose logit is -inf is no candidate; +inf counts as
 * the largest finite float. With n_group > 1, the experts lie in n_group equal runs; a run's value is the sum of its
 * group_best (1 or 2) largest choices, and only candidates of the top_group runs of the largest values stay (of
 * equal ones the first). The top_k largest choices are a token's experts, in falling order, of equal ones the first
 * (without a bias they are compared as logits; numbers are compared up to 2^-42 of themselves); weight = p of the expert, divided by the sum of the token's chosen p
 * where renorm is not 0 (0 where that sum is 0), times scale, rounded to fp32 once. Where fewer candidates are
 * left, and for a token with active[m] == 0 (active NULL: all are active), the places left get id -1 and weight 0.
 * A NaN logit (or one that makes p NaN) ranks behind every number and its weights are NaN; ids stay in range.
 *     ids[M][top_k], weight[M][top_k]
 * and, all three or none, the rows of the chosen experts, sorted by expert, then by token:
 *     expert_off[E + 1]     expert e's rows are [expert_off[e], expert_off[e + 1])
 *     src_row[M * top_k]    the token of each row (places from expert_off[E] on are left as they were)
 *     slot[M][top_k]        the row of each choice, -1 where there is none
 * 1 <= E <= 1024, E % n_group == 0, 1 <= n_group <= 64, group_best 1 or 2, 1 <= top_group <= n_group,
 * 1 <= top_k <= min(32, E), M * top_k < 2^24, rs >= E, M * rs <= 2^40. Results in device memory may be 4-byte aligned. More than 32
 * tokens with a plan take scratch of the handle (a captured call needs an eager one of the same size first; graphs that
 * hold scratch of one handle are replayed in the order of its stream). */
#define ROCKET_ROUTE_SOFTMAX 0
#define ROCKET_ROUTE_SIGMOID 1
int rocket_moe_route_f32(int fd, int M, int E, const float *logits, int64_t rs, int score, const float *bias, int n_group, int group_best,
                         int top_group, int top_k, int renorm, float scale, const uint8_t *active, int32_t *ids, float *weight,
                         int32_t *expert_off, int32_t *src_row, int32_t *slot);
int rocket_moe_route_fp16(int fd, int M, int E, const _Float16 *logits, int64_t rs, int score, const float *bias, int n_group, int group_best,
                          int top_group, int top_k, int renorm, float scale, const uint8_t *active, int32_t *ids, float *weight,
                          int32_t *expert_off, int32_t *src_row, int32_t *slot);

#ifdef __cplusplus
}
#endif
#endif /* ROCKET_LAYER_H */
