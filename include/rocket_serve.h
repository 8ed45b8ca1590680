/*
 * rocket_serve.h — attention for serving on MI355X: what stands between a layer's Q / K / V products
 * and its output product besides rocket_flash_attn_fp16 (additions; the reference library has no
 * counterpart).
 *
 *   rocket_qk_norm_rope_*          norms of the query and key heads and their position rotation
 *   rocket_kv4_*                   a key / value cache held in 4 bits for a batch of sequences
 *   rocket_kv4_attn_fp16           attention over that cache: decode steps, drafts, prompt chunks
 *   rocket_flash_attn_window_fp16  causal attention over fp16 keys and values, with a sliding window
 *                                  and a few first keys that stay visible (sinks)
 *
 * As everywhere in this library: operands may be host or device pointers (the 4-bit cache alone must
 * be device memory); device memory is used in place where it is 16-byte aligned (seq_len and pos:
 * 4-byte, so that a part of a batch's array is) and staged where it is not, which a captured call does
 * not allow; fd < 0 runs the fp64 host path (every operand host memory then), handles run asynchronously
 * where rocket_hip_set_mode says so, and a call returns 0 or a negative rocket_status: -1 for a bad
 * argument, before anything is launched. Results must not lie over a call's other operands (-1).
 * Strides count elements.
 *
 * Visibility. Token t of a call's n_tokens stands at position p = len - n_tokens + t of a sequence of
 * len keys. It sees key j when
 *     0 <= j <= p  and  (window == 0  or  j > p - window  or  j < sinks).
 * With S = scale * (q . k), S = softcap * tanh(S / softcap) where softcap != 0, a token's result is
 * the softmax-weighted sum of the values of the keys it sees. A token that sees none (p < 0) gets
 * zeros. What keys that no token of a call sees hold (stale or not yet written memory, infinities,
 * NaN) does not reach any result. scale and softcap are finite, |scale| at most 2^127. The GPU holds
 * scores in fp32; they have to stay below 2^26 in size (where fp32 steps by 4).
 */
#ifndef ROCKET_SERVE_H
#define ROCKET_SERVE_H

#include <stddef.h>
#include <stdint.h>

#include "rocket_matmul.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms and rotation of the query and key heads ----
 * Rows m = s * n_tokens + t (s < n_seq) hold every head end to end: query head h of row m at
 * q + m * q_rs + h * head_dim, key head h at k + m * k_rs + h * head_dim (q and k may be columns of
 * one fused product's rows). Results are head-major, as the attention entries take them:
 *     q_out[n_seq][n_head][n_tokens][head_dim],  k_out[n_seq][n_kv_heads][n_tokens][head_dim].
 * With x a head's row, in fp32:
 *     y[i] = x[i] / sqrt(mean(x^2) + eps) * w[i]       (w = wq or wk, head_dim values; NULL: ones)
 *     eps < 0: y = x (no norm; wq and wk must be NULL)
 * then the first rot_dim values are rotated in pairs j < rot_dim / 2 by pos[m] * inv_freq[j] radians,
 *     a' = a cos - b sin,  b' = b cos + a sin,
 * (a, b) = (y[j], y[j + rot_dim / 2]) for ROCKET_ROPE_HALVES, (y[2j], y[2j + 1]) for
 * ROCKET_ROPE_PAIRS; the others pass. One rounding to fp16. The angle is reduced in fp64, so
 * positions may be any int32 (padding rows of a negative position included).
 * head_dim % 32 == 0, <= 256; rot_dim % 8 == 0, 0 <= rot_dim <= head_dim (0: inv_freq and pos are not
 * read); row strides at least the heads' values, and multiples of 8. _f32in: fp32 rows (what the
 * group-wise products write). */
#define ROCKET_ROPE_HALVES 0
#define ROCKET_ROPE_PAIRS  1
int rocket_qk_norm_rope_fp16(int fd, int n_seq, int n_tokens, int n_head, int n_kv_heads, int head_dim, int rot_dim,
                             int style, float eps, const _Float16 *q, int64_t q_rs, const _Float16 *k, int64_t k_rs,
                             const _Float16 *wq, const _Float16 *wk, const float *inv_freq, const int32_t *pos,
                             _Float16 *q_out, _Float16 *k_out);
int rocket_qk_norm_rope_f32in(int fd, int n_seq, int n_tokens, int n_head, int n_kv_heads, int head_dim, int rot_dim,
                              int style, float eps, const float *q, int64_t q_rs, const float *k, int64_t k_rs,
                              const _Float16 *wq, const _Float16 *wk, const float *inv_freq, const int32_t *pos,
                              _Float16 *q_out, _Float16 *k_out);

/* ---- the 4-bit cache ----
 * One buffer of rocket_kv4_bytes(shape) bytes of device memory, 16-byte aligned, that the caller
 * owns (host memory for fd < 0). It needs no initialisation. A group of 32 values of one key or
 * value row is stored as 4-bit codes c and an fp16 (scale, minimum):
 *     minimum = min(x),  scale = fp16((max(x) - min(x)) / 15)  (the next lower fp16 where 15 * scale + minimum
 *     would not be a finite fp16),
 *     c = clamp(rint((x - minimum) / scale), 0, 15)  (0 where scale is 0),  in fp32,
 *     value = c * scale + minimum  (rocket_kv4_read_fp16 rounds it to fp16, once; attention on the GPU multiplies the
 *     values of V so rounded and those of K as they are, the host path both as they are).
 * Inputs should be finite; an infinity is taken as the largest finite fp16 of its sign, a NaN as 0.
 * Parts, each starting at a multiple of 256 bytes, cap = capacity rounded up to 32:
 *     key codes    [n_seq][n_kv_heads][cap][head_dim / 2] bytes, value 2b in byte b's low nibble
 *     key scales   [n_seq][n_kv_heads][cap][head_dim / 32] (scale, minimum) fp16
 *     value codes  [n_seq][n_kv_heads][cap / 8][dv / 8][8 keys][4] bytes, nibbles as above
 *     value scales [n_seq][n_kv_heads][cap / 8][dv / 32][8 keys] (scale, minimum) fp16
 * n_seq, n_kv_heads >= 1, head_dim and dv multiples of 32 up to 256, 1 <= capacity <= 2^23,
 * n_seq * n_kv_heads <= 65535. rocket_kv4_bytes returns 0 for any other shape (or NULL). */
typedef struct rocket_kv4_shape {
    int32_t n_seq, n_kv_heads, head_dim, dv, capacity;
} rocket_kv4_shape;
size_t rocket_kv4_bytes(const rocket_kv4_shape *shape);

/* Quantises n_tokens new keys and values of each of the sequences seq0 .. seq0 + n_seq - 1.
 * seq_len[n_seq]: the sequences' lengths with these tokens; token t of sequence s goes to position
 * seq_len[s] - n_tokens + t. Tokens at a negative position are skipped (padding in front of a ragged
 * batch; seq_len 0: the sequence takes no token), and those past the capacity (a host array with a
 * length above the capacity is refused). Nothing else of the cache is written.
 * Key of token t, head h of sequence s (of the call) at K + s * k_ss + h * k_hs + t * k_rs, the value
 * likewise; strides are multiples of 8, not negative and at most 2^40. */
int rocket_kv4_append_fp16(int fd, const rocket_kv4_shape *shape, void *cache, int seq0, int n_seq, int n_tokens,
                           const _Float16 *K, int64_t k_ss, int64_t k_hs, int64_t k_rs,
                           const _Float16 *V, int64_t v_ss, int64_t v_hs, int64_t v_rs, const int32_t *seq_len);

/* The values that the cache stands for: the last n_tokens positions of each sequence, in fp16, K[n_seq][n_kv_heads][n_tokens][head_dim], V[n_seq][n_kv_heads][n_tokens][dv].
 * Either may be NULL. Positions outside [0, capacity) read zeros. */
int rocket_kv4_read_fp16(int fd, const rocket_kv4_shape *shape, const void *cache, int seq0, int n_seq, int n_tokens,
                         const int32_t *seq_len, _Float16 *K, _Float16 *V);

/* Attention of n_tokens tokens of each of the sequences seq0 .. seq0 + n_seq - 1 over their cached
 * keys, the tokens' own among them (append first). Q[n_seq][n_head][n_tokens][head_dim], results
 * out[n_seq][n_head][n_tokens][dv]; head h reads KV head h / (n_head / n_kv_heads). seq_len[n_seq] as
 * above; every length from 1 to max_kv (<= capacity) is served, and a sequence of any other length gets
 * zeros (idle places of a batch; a host array with a length above max_kv is refused). max_kv bounds the
 * work that is laid out, so a captured call may be replayed with other lengths up to it. window 0: none;
 * sinks without a window must be 0. n_head % n_kv_heads == 0. */
int rocket_kv4_attn_fp16(int fd, const rocket_kv4_shape *shape, const void *cache, int seq0, int n_seq, int n_tokens,
                         int max_kv, int n_head, float scale, float softcap, int window, int sinks,
                         const _Float16 *Q, const int32_t *seq_len, _Float16 *out);

/* ---- windowed attention over fp16 keys and values ----
 * rocket_flash_attn_fp16 with the visibility above in place of a mask (and no clamp of the scores):
 * one sequence of n_kv keys, whose last n_tokens positions are the tokens'. Q[n_head][n_tokens][head_dim],
 * K[n_kv_heads][kv_stride][head_dim], V[n_kv_heads][dv][kv_stride] (kv_stride >= n_kv: room for more
 * keys behind the last one, which is not read into any result), out[n_head][n_tokens][dv].
 * n_head % n_kv_heads == 0, head_dim % 32 == 0, dv % 16 == 0, both <= 256 on the GPU. Tiles that no
 * token of a block sees are skipped, so a long cache under a window costs what the window costs. */
int rocket_flash_attn_window_fp16(int fd, int n_tokens, int n_kv, int kv_stride, int head_dim, int dv, int n_head,
                                  int n_kv_heads, float scale, float softcap, int window, int sinks,
                                  const _Float16 *Q, const _Float16 *K, const _Float16 *V, _Float16 *out);

#ifdef __cplusplus
}
#endif
#endif /* ROCKET_SERVE_H */
