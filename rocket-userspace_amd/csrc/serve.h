// serve.h — launches behind rocket_serve.h: head norms with rotation (rope.hip), the 4-bit key / value
// cache (kv4.hip) and attention over it or under a window (serve_attn.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "rocket_serve.h"

namespace rk {

constexpr int kServeMaxDim = 256;    // head_dim and dv
constexpr int kServeMaxCap = 1 << 23;

// The cache's parts (rocket_serve.h states the layout): byte offsets of key codes, key scales, value
// codes and value scales from the buffer's start, and its size; cap = capacity rounded up to 32.
struct Kv4Layout {
    size_t kc, ks, vc, vs, bytes;
    int cap;
};
// false for a shape that the cache does not come in.
bool kv4_layout(const rocket_kv4_shape *s, Kv4Layout *l);

// A group's scale, minimum and codes, the same steps on the host and on the GPU (fp32, IEEE division).
__host__ __device__ inline float kv4_finite(float x)
{
    return x != x ? 0.f : x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;
}
// (A scale that rounded up may carry code 15 past the largest fp16: then the next lower one, so that every value that a
// cache stands for is finite.)
__host__ __device__ inline _Float16 kv4_scale(float lo, float hi)
{
    const _Float16 s = (_Float16)((hi - lo) / 15.f);
    if (fmaf(15.f, (float)s, lo) < 65520.f) return s;
    return __builtin_bit_cast(_Float16, (uint16_t)(__builtin_bit_cast(uint16_t, s) - 1));
}
__host__ __device__ inline int kv4_code(float x, float lo, float scale)
{
    if (!(scale > 0.f)) return 0;
    const float c = rintf((x - lo) / scale);
    return c < 0.f ? 0 : c > 15.f ? 15 : (int)c;
}

struct RopeLaunch {
    const void *q = nullptr, *k = nullptr;   // fp16, or fp32 (f32)
    bool f32 = false, pairs = false, norm = false;
    long q_rs = 0, k_rs = 0;
    const _Float16 *wq = nullptr, *wk = nullptr;
    const float *inv_freq = nullptr;
    const int32_t *pos = nullptr;
    _Float16 *q_out = nullptr, *k_out = nullptr;
    int n_seq = 0, n_tokens = 0, n_head = 0, n_kv = 0, dim = 0, rot = 0;
    float eps = 0.f;
};
hipError_t qk_norm_rope(const RopeLaunch &L, hipStream_t s, uint64_t *blocks);

// The call's part of a cache: places seq0 .. seq0 + n_seq - 1.
struct Kv4View {
    char *kc, *ks, *vc, *vs;   // the first place's parts
    int heads, dk, dv, cap, capacity, n_seq;
};
Kv4View kv4_view(const rocket_kv4_shape &s, const Kv4Layout &l, void *cache, int seq0, int n_seq);

struct Kv4Rows {
    const _Float16 *K = nullptr, *V = nullptr;   // append: new rows; strides of sequence, head, token
    long k_ss = 0, k_hs = 0, k_rs = 0, v_ss = 0, v_hs = 0, v_rs = 0;
    _Float16 *Ko = nullptr, *Vo = nullptr;       // read: dense results (either null)
    const int32_t *seq_len = nullptr;
    int n_tokens = 0;
};
hipError_t kv4_append(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks);
hipError_t kv4_read(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks);

// Attention of n_tokens tokens a sequence. Over the cache, or (Kf) over fp16 keys [kv head][stride][dk]
// and values [kv head][dv][stride] of one sequence of max_kv keys.
struct ServeAttn {
    Kv4View c{};
    const _Float16 *Kf = nullptr, *Vf = nullptr;
    long stride = 0, k_hs = 0;               // keys a V^T row holds; elements a head's keys take
    const _Float16 *Q = nullptr;
    _Float16 *out = nullptr;
    const int32_t *seq_len = nullptr;   // null: max_kv
    int n_seq = 1, n_tokens = 0, n_head = 0, gqa = 1, dk = 0, dv = 0, max_kv = 0, window = 0, sinks = 0;
    float scale = 1.f, softcap = 0.f;
    // workspace for splits of the key axis (serve_attn_ws); without it a workgroup walks every key
    float *ws = nullptr;
    size_t ws_bytes = 0;
};
bool serve_few_rows(const ServeAttn &a);
size_t serve_attn_ws(const ServeAttn &a);
hipError_t serve_attn(const ServeAttn &a, hipStream_t s, uint64_t *blocks);

// Few query rows a KV head over the cache (kv4_rows.hip).
bool kv4_few_rows(const ServeAttn &a);
size_t kv4_rows_ws(const ServeAttn &a);
hipError_t kv4_rows(const ServeAttn &a, hipStream_t s, uint64_t *blocks);

// More rows, over either (serve_tiles.hip); few over fp16 keys are fa_rows' (attn_decode.hip).
size_t serve_tiles_ws(const ServeAttn &a);
hipError_t serve_tiles(const ServeAttn &a, hipStream_t s, uint64_t *blocks);

// The fp64 host paths (fd < 0); false where host memory runs out.
bool qk_norm_rope_ref(const RopeLaunch &L);
void kv4_append_ref(const Kv4View &c, const Kv4Rows &r);
void kv4_read_ref(const Kv4View &c, const Kv4Rows &r);
bool serve_attn_ref(const ServeAttn &a);

}  // namespace rk
