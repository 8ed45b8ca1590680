// serve_entry.cpp — rocket_serve.h: argument checks, staging and launches of the head norms with
// rotation (rope.hip), the 4-bit cache (kv4.hip) and attention over it or under a window.
#include "attn.h"
#include "internal.h"
#include "ops.h"
#include "serve.h"

#include <math.h>

#include <algorithm>
#include <new>

using namespace rk;

namespace {

constexpr int64_t kMaxStride = (int64_t)1 << 40;
// Lengths and positions are read one by one: a part of a batch's array (seq_len + seq0) is used in place.
constexpr size_t kIntAlign = sizeof(int32_t);

size_t h16(size_t n) { return n * sizeof(_Float16); }

bool overlap(const void *a, size_t an, const void *b, size_t bn)
{
    return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

// Nothing may throw across the C ABI (the staging lists allocate).
template <class F> int guarded(const char *who, F &&f) noexcept
{
    try {
        return f();
    } catch (const std::bad_alloc &) {
        ROCKET_LOGE("%s: out of host memory\n", who);
        return ROCKET_E_NOMEM;
    }
}

int launched(Call &c, hipError_t e, uint64_t blocks)
{
    if (e != hipSuccess) {
        (void)hipGetLastError();
        ROCKET_LOGE("%s: kernel launch rejected: %s\n", c.who(), hipGetErrorString(e));
        (void)c.finish();
        return e == hipErrorInvalidValue ? ROCKET_E_SHAPE : ROCKET_E_DEVICE;
    }
    count_launch(blocks);
    return c.finish();
}

int bad(const char *who, const char *what)
{
    ROCKET_LOGE("%s: %s\n", who, what);
    return ROCKET_E_SHAPE;
}

int bad_fd(const char *who, int fd)
{
    ROCKET_LOGE("%s: fd %d is not an open rocket handle\n", who, fd);
    return ROCKET_E_DEVICE;
}

int rope(const char *who, int fd, RopeLaunch L, int style)
{
    if (L.n_seq < 1 || L.n_tokens < 1 || L.n_head < 1 || L.n_kv < 1 || L.n_seq > kDimMax || L.n_tokens > kDimMax || L.n_head > kDimMax ||
        L.n_kv > kDimMax || (long)L.n_seq * L.n_tokens >= kDimMax || (long)L.n_head + L.n_kv > 65535)
        return bad(who, "a count is below 1 or too large");
    if (L.dim < 32 || L.dim % 32 || L.dim > kServeMaxDim || L.rot < 0 || L.rot % 8 || L.rot > L.dim)
        return bad(who, "head_dim is a multiple of 32 up to 256, rot_dim one of 8 up to head_dim");
    if (style != ROCKET_ROPE_HALVES && style != ROCKET_ROPE_PAIRS) return bad(who, "unknown rotation style");
    L.pairs = style == ROCKET_ROPE_PAIRS;
    if (isnan(L.eps)) return bad(who, "eps is NaN");
    L.norm = L.eps >= 0.f;
    if (!L.norm && (L.wq || L.wk)) return bad(who, "weights without a norm");
    if (!L.q || !L.k || !L.q_out || !L.k_out || (L.rot && (!L.inv_freq || !L.pos))) return bad(who, "null operand");
    if (L.q_rs % 8 || L.k_rs % 8 || L.q_rs < (long)L.n_head * L.dim || L.k_rs < (long)L.n_kv * L.dim || L.q_rs > kMaxStride || L.k_rs > kMaxStride)
        return bad(who, "a row stride is a multiple of 8 and holds the row's heads");
    const size_t e = L.f32 ? sizeof(float) : sizeof(_Float16), rows = (size_t)L.n_seq * L.n_tokens;
    const size_t qb = ((rows - 1) * L.q_rs + (size_t)L.n_head * L.dim) * e, kb = ((rows - 1) * L.k_rs + (size_t)L.n_kv * L.dim) * e;
    const size_t wb = h16((size_t)L.dim), fb = (size_t)L.rot / 2 * sizeof(float), pb = rows * sizeof(int32_t);
    const size_t qo = h16(rows * L.n_head * L.dim), ko = h16(rows * L.n_kv * L.dim);
    if (!L.rot) L.inv_freq = nullptr, L.pos = nullptr;
    const struct { const void *p; size_t n, align; } in[] = {{L.q, qb, 16}, {L.k, kb, 16}, {L.wq, wb, 16}, {L.wk, wb, 16}, {L.inv_freq, fb, 16}, {L.pos, pb, kIntAlign}};
    for (const auto &i : in)
        if (overlap(i.p, i.n, L.q_out, qo) || overlap(i.p, i.n, L.k_out, ko)) return bad(who, "results over operands");
    if (overlap(L.q_out, qo, L.k_out, ko)) return bad(who, "results over each other");
    if (fd < 0) return qk_norm_rope_ref(L) ? ROCKET_OK : ROCKET_E_NOMEM;
    Locked lk(fd);
    if (!lk.ok()) return bad_fd(who, fd);
    Call c(lk.h, who);
    for (const auto &i : in)
        if (i.p) c.want(i.p, i.n, i.align);
    c.want(L.q_out, qo);
    c.want(L.k_out, ko);
    if (int rc = c.begin()) return rc;
    const void *d[6];
    for (int i = 0; i < 6; i++) {
        d[i] = in[i].p ? c.in(in[i].p, in[i].n, in[i].align) : nullptr;
        if (in[i].p && !d[i]) return c.finish();
    }
    L.q = d[0];
    L.k = d[1];
    L.wq = static_cast<const _Float16 *>(d[2]);
    L.wk = static_cast<const _Float16 *>(d[3]);
    L.inv_freq = static_cast<const float *>(d[4]);
    L.pos = static_cast<const int32_t *>(d[5]);
    L.q_out = static_cast<_Float16 *>(c.out(L.q_out, qo));
    L.k_out = static_cast<_Float16 *>(c.out(L.k_out, ko));
    if (!L.q_out || !L.k_out) return c.finish();
    uint64_t blocks = 0;
    return launched(c, qk_norm_rope(L, c.stream(), &blocks), blocks);
}

// The cache, its places and the lengths that a call names. On success *l is the layout.
int kv4_args(const char *who, const rocket_kv4_shape *s, const void *cache, int seq0, int n_seq, int n_tokens, const int32_t *seq_len, Kv4Layout *l)
{
    if (!kv4_layout(s, l)) return bad(who, "unsupported cache shape");
    if (!cache || !seq_len) return bad(who, "null operand");
    if ((uintptr_t)cache & 15u) return bad(who, "the cache is not 16-byte aligned");
    if (seq0 < 0 || n_seq < 1 || seq0 > s->n_seq - n_seq) return bad(who, "places outside the cache");
    if (n_tokens < 1 || n_tokens > kServeMaxCap) return bad(who, "n_tokens below 1 or too large");
    return ROCKET_OK;
}

// Lengths that the host can see stay within `most`.
bool lens_ok(const int32_t *seq_len, int n, int most)
{
    for (int i = 0; i < n; i++)
        if (seq_len[i] > most) return false;
    return true;
}
bool lens_ok(Handle *h, const int32_t *seq_len, int n, int most)
{
    hipPointerAttribute_t a;
    if (h->trust_device) return true;
    if (hipPointerGetAttributes(&a, seq_len) != hipSuccess) (void)hipGetLastError();   // plain host memory
    else if (a.type != hipMemoryTypeUnregistered && a.type != hipMemoryTypeHost) return true;
    return lens_ok(seq_len, n, most);
}
bool on_device(Handle *h, const void *p) { return h->trust_device || is_device_ptr(p, h->device); }

// Elements from the first of a strided operand to past its last.
size_t span(int n_seq, long ss, int heads, long hs, int tokens, long rs, int d)
{
    return (size_t)(n_seq - 1) * ss + (size_t)(heads - 1) * hs + (size_t)(tokens - 1) * rs + d;
}

int attn_args(const char *who, int n_tokens, int n_head, int kv_heads, float scale, float softcap, int window, int sinks)
{
    if (n_head < 1 || n_head > 65535 || kv_heads < 1 || n_head % kv_heads) return bad(who, "n_head is not a multiple of the KV heads, or too large");
    if (window < 0 || sinks < 0 || (!window && sinks)) return bad(who, "window and sinks are not negative, and sinks need a window");
    if (!(fabsf(scale) <= 0x1p127f) || !isfinite(softcap)) return bad(who, "scale or softcap is not finite, or scale above 2^127");
    if ((long)n_tokens * n_head > (long)1 << 30) return bad(who, "too many rows");
    return ROCKET_OK;
}

}  // namespace

extern "C" {

int rocket_qk_norm_rope_fp16(int fd, int n_seq, int n_tokens, int n_head, int n_kv_heads, int head_dim, int rot_dim, int style, float eps,
                             const _Float16 *q, int64_t q_rs, const _Float16 *k, int64_t k_rs, const _Float16 *wq, const _Float16 *wk,
                             const float *inv_freq, const int32_t *pos, _Float16 *q_out, _Float16 *k_out)
{
    static const char *who = "rocket_qk_norm_rope_fp16";
    RopeLaunch L;
    L.q = q; L.k = k; L.q_rs = q_rs; L.k_rs = k_rs; L.wq = wq; L.wk = wk; L.inv_freq = inv_freq; L.pos = pos; L.q_out = q_out; L.k_out = k_out;
    L.n_seq = n_seq; L.n_tokens = n_tokens; L.n_head = n_head; L.n_kv = n_kv_heads; L.dim = head_dim; L.rot = rot_dim; L.eps = eps;
    return guarded(who, [&] { return rope(who, fd, L, style); });
}

int rocket_qk_norm_rope_f32in(int fd, int n_seq, int n_tokens, int n_head, int n_kv_heads, int head_dim, int rot_dim, int style, float eps,
                              const float *q, int64_t q_rs, const float *k, int64_t k_rs, const _Float16 *wq, const _Float16 *wk,
                              const float *inv_freq, const int32_t *pos, _Float16 *q_out, _Float16 *k_out)
{
    static const char *who = "rocket_qk_norm_rope_f32in";
    RopeLaunch L;
    L.f32 = true;
    L.q = q; L.k = k; L.q_rs = q_rs; L.k_rs = k_rs; L.wq = wq; L.wk = wk; L.inv_freq = inv_freq; L.pos = pos; L.q_out = q_out; L.k_out = k_out;
    L.n_seq = n_seq; L.n_tokens = n_tokens; L.n_head = n_head; L.n_kv = n_kv_heads; L.dim = head_dim; L.rot = rot_dim; L.eps = eps;
    return guarded(who, [&] { return rope(who, fd, L, style); });
}

size_t rocket_kv4_bytes(const rocket_kv4_shape *shape)
{
    Kv4Layout l;
    return kv4_layout(shape, &l) ? l.bytes : 0;
}

int rocket_kv4_append_fp16(int fd, const rocket_kv4_shape *shape, void *cache, int seq0, int n_seq, int n_tokens, const _Float16 *K,
                           int64_t k_ss, int64_t k_hs, int64_t k_rs, const _Float16 *V, int64_t v_ss, int64_t v_hs, int64_t v_rs,
                           const int32_t *seq_len)
{
    static const char *who = "rocket_kv4_append_fp16";
    return guarded(who, [&]() -> int {
        Kv4Layout l;
        if (int rc = kv4_args(who, shape, cache, seq0, n_seq, n_tokens, seq_len, &l)) return rc;
        if (!K || !V) return bad(who, "null operand");
        for (int64_t s : {k_ss, k_hs, k_rs, v_ss, v_hs, v_rs})
            if (s < 0 || s % 8 || s > kMaxStride) return bad(who, "a stride is negative, too large or no multiple of 8");
        const size_t kb = h16(span(n_seq, k_ss, shape->n_kv_heads, k_hs, n_tokens, k_rs, shape->head_dim));
        const size_t vb = h16(span(n_seq, v_ss, shape->n_kv_heads, v_hs, n_tokens, v_rs, shape->dv)), nb = (size_t)n_seq * sizeof(int32_t);
        if (overlap(cache, l.bytes, K, kb) || overlap(cache, l.bytes, V, vb) || overlap(cache, l.bytes, seq_len, nb)) return bad(who, "the cache over operands");
        Kv4Rows r;
        r.k_ss = k_ss; r.k_hs = k_hs; r.k_rs = k_rs; r.v_ss = v_ss; r.v_hs = v_hs; r.v_rs = v_rs;
        r.n_tokens = n_tokens;
        const Kv4View view = kv4_view(*shape, l, cache, seq0, n_seq);
        if (fd < 0) {
            if (!lens_ok(seq_len, n_seq, shape->capacity)) return bad(who, "a length above the capacity");
            r.K = K; r.V = V; r.seq_len = seq_len;
            kv4_append_ref(view, r);
            return ROCKET_OK;
        }
        Locked lk(fd);
        if (!lk.ok()) return bad_fd(who, fd);
        if (!on_device(lk.h, cache)) return bad(who, "the cache is not memory of the handle's device");
        if (!lens_ok(lk.h, seq_len, n_seq, shape->capacity)) return bad(who, "a length above the capacity");
        Call c(lk.h, who);
        c.want(K, kb);
        c.want(V, vb);
        c.want(seq_len, nb, kIntAlign);
        if (int rc = c.begin()) return rc;
        r.K = static_cast<const _Float16 *>(c.in(K, kb));
        r.V = static_cast<const _Float16 *>(c.in(V, vb));
        r.seq_len = static_cast<const int32_t *>(c.in(seq_len, nb, kIntAlign));
        if (!r.K || !r.V || !r.seq_len) return c.finish();
        uint64_t blocks = 0;
        return launched(c, kv4_append(view, r, c.stream(), &blocks), blocks);
    });
}

int rocket_kv4_read_fp16(int fd, const rocket_kv4_shape *shape, const void *cache, int seq0, int n_seq, int n_tokens, const int32_t *seq_len,
                         _Float16 *K, _Float16 *V)
{
    static const char *who = "rocket_kv4_read_fp16";
    return guarded(who, [&]() -> int {
        Kv4Layout l;
        if (int rc = kv4_args(who, shape, cache, seq0, n_seq, n_tokens, seq_len, &l)) return rc;
        const size_t rows = (size_t)n_seq * shape->n_kv_heads * n_tokens, nb = (size_t)n_seq * sizeof(int32_t);
        const size_t kb = K ? h16(rows * shape->head_dim) : 0, vb = V ? h16(rows * shape->dv) : 0;
        if (overlap(cache, l.bytes, K, kb) || overlap(cache, l.bytes, V, vb) || overlap(seq_len, nb, K, kb) || overlap(seq_len, nb, V, vb) ||
            overlap(K, kb, V, vb))
            return bad(who, "results over operands or each other");
        if (!K && !V) return ROCKET_OK;
        Kv4Rows r;
        r.n_tokens = n_tokens;
        const Kv4View view = kv4_view(*shape, l, const_cast<void *>(cache), seq0, n_seq);
        if (fd < 0) {
            r.Ko = K; r.Vo = V; r.seq_len = seq_len;
            kv4_read_ref(view, r);
            return ROCKET_OK;
        }
        Locked lk(fd);
        if (!lk.ok()) return bad_fd(who, fd);
        if (!on_device(lk.h, cache)) return bad(who, "the cache is not memory of the handle's device");
        Call c(lk.h, who);
        c.want(seq_len, nb, kIntAlign);
        if (K) c.want(K, kb);
        if (V) c.want(V, vb);
        if (int rc = c.begin()) return rc;
        r.seq_len = static_cast<const int32_t *>(c.in(seq_len, nb, kIntAlign));
        r.Ko = K ? static_cast<_Float16 *>(c.out(K, kb)) : nullptr;
        r.Vo = V ? static_cast<_Float16 *>(c.out(V, vb)) : nullptr;
        if (!r.seq_len || (K && !r.Ko) || (V && !r.Vo)) return c.finish();
        uint64_t blocks = 0;
        return launched(c, kv4_read(view, r, c.stream(), &blocks), blocks);
    });
}

int rocket_kv4_attn_fp16(int fd, const rocket_kv4_shape *shape, const void *cache, int seq0, int n_seq, int n_tokens, int max_kv, int n_head,
                         float scale, float softcap, int window, int sinks, const _Float16 *Q, const int32_t *seq_len, _Float16 *out)
{
    static const char *who = "rocket_kv4_attn_fp16";
    return guarded(who, [&]() -> int {
        Kv4Layout l;
        if (int rc = kv4_args(who, shape, cache, seq0, n_seq, n_tokens, seq_len, &l)) return rc;
        if (int rc = attn_args(who, n_tokens, n_head, shape->n_kv_heads, scale, softcap, window, sinks)) return rc;
        if (!Q || !out) return bad(who, "null operand");
        if (max_kv < 1 || max_kv > shape->capacity) return bad(who, "max_kv outside [1, capacity]");
        const size_t rows = (size_t)n_seq * n_head * n_tokens, nb = (size_t)n_seq * sizeof(int32_t);
        if (rows > (size_t)1 << 30) return bad(who, "too many rows");
        const size_t qb = h16(rows * shape->head_dim), ob = h16(rows * shape->dv);
        if (overlap(out, ob, Q, qb) || overlap(out, ob, cache, l.bytes) || overlap(out, ob, seq_len, nb)) return bad(who, "results over operands");
        ServeAttn a;
        a.c = kv4_view(*shape, l, const_cast<void *>(cache), seq0, n_seq);
        a.n_seq = n_seq; a.n_tokens = n_tokens; a.n_head = n_head; a.gqa = n_head / shape->n_kv_heads; a.dk = shape->head_dim; a.dv = shape->dv;
        a.max_kv = max_kv; a.window = std::min(window, kServeMaxCap); a.sinks = std::min(sinks, kServeMaxCap); a.scale = scale; a.softcap = softcap;
        if (fd < 0) {
            if (!lens_ok(seq_len, n_seq, max_kv)) return bad(who, "a length above max_kv");
            a.Q = Q; a.out = out; a.seq_len = seq_len;
            return serve_attn_ref(a) ? ROCKET_OK : ROCKET_E_NOMEM;
        }
        Locked lk(fd);
        if (!lk.ok()) return bad_fd(who, fd);
        if (!on_device(lk.h, cache)) return bad(who, "the cache is not memory of the handle's device");
        if (!lens_ok(lk.h, seq_len, n_seq, max_kv)) return bad(who, "a length above max_kv");
        Call c(lk.h, who);
        c.want(Q, qb);
        c.want(seq_len, nb, kIntAlign);
        c.want(out, ob);
        const size_t ws = c.want_optional(serve_attn_ws(a), max_kv >= 512);
        if (int rc = c.begin()) return rc;
        a.ws = static_cast<float *>(c.optional(ws));
        a.ws_bytes = a.ws ? ws : 0;
        a.Q = static_cast<const _Float16 *>(c.in(Q, qb));
        a.seq_len = static_cast<const int32_t *>(c.in(seq_len, nb, kIntAlign));
        a.out = static_cast<_Float16 *>(c.out(out, ob));
        if (!a.Q || !a.seq_len || !a.out) return c.finish();
        uint64_t blocks = 0;
        return launched(c, serve_attn(a, c.stream(), &blocks), blocks);
    });
}

int rocket_flash_attn_window_fp16(int fd, int n_tokens, int n_kv, int kv_stride, int head_dim, int dv, int n_head, int n_kv_heads, float scale,
                                  float softcap, int window, int sinks, const _Float16 *Q, const _Float16 *K, const _Float16 *V, _Float16 *out)
{
    static const char *who = "rocket_flash_attn_window_fp16";
    return guarded(who, [&]() -> int {
        if (n_tokens < 1 || n_kv < 1 || kv_stride < n_kv || n_tokens > kServeMaxCap || kv_stride > kServeMaxCap / 2 - 64)
            return bad(who, "n_tokens or n_kv below 1, kv_stride below n_kv, or one too large");
        if (int rc = attn_args(who, n_tokens, n_head, n_kv_heads, scale, softcap, window, sinks)) return rc;
        if (head_dim < 32 || head_dim % 32 || head_dim > kServeMaxDim || dv < 16 || dv % 16 || dv > kServeMaxDim)
            return bad(who, "head_dim is a multiple of 32 and dv one of 16, up to 256");
        if (!Q || !K || !V || !out) return bad(who, "null operand");
        const size_t qb = h16((size_t)n_head * n_tokens * head_dim), ob = h16((size_t)n_head * n_tokens * dv);
        const size_t kb = h16((size_t)n_kv_heads * kv_stride * head_dim), vb = h16((size_t)n_kv_heads * kv_stride * dv);
        if (overlap(out, ob, Q, qb) || overlap(out, ob, K, kb) || overlap(out, ob, V, vb)) return bad(who, "results over operands");
        ServeAttn a;
        a.n_tokens = n_tokens; a.n_head = n_head; a.gqa = n_head / n_kv_heads; a.dk = head_dim; a.dv = dv; a.stride = kv_stride; a.k_hs = (long)kv_stride * head_dim;
        a.max_kv = n_kv; a.window = std::min(window, kServeMaxCap); a.sinks = std::min(sinks, kServeMaxCap); a.scale = scale; a.softcap = softcap;
        if (fd < 0) {
            a.Q = Q; a.Kf = K; a.Vf = V; a.out = out;
            return serve_attn_ref(a) ? ROCKET_OK : ROCKET_E_NOMEM;
        }
        Locked lk(fd);
        if (!lk.ok()) return bad_fd(who, fd);
        Call c(lk.h, who);
        c.want(Q, qb);
        c.want(K, kb);
        c.want(V, vb);
        c.want(out, ob);
        // (the tiles read chunks of eight keys: V^T rows of fewer are copied into longer ones)
        a.Kf = K;
        const int padded = kv_stride < 8 && !serve_few_rows(a) ? 64 : kv_stride;
        const size_t pb = padded != kv_stride ? h16((size_t)n_kv_heads * dv * padded) : 0;
        if (pb) c.want_scratch(pb);
        const size_t ws = c.want_optional(serve_attn_ws(a), n_kv >= 512);
        if (int rc = c.begin()) return rc;
        a.Q = static_cast<const _Float16 *>(c.in(Q, qb));
        a.Kf = static_cast<const _Float16 *>(c.in(K, kb));
        a.Vf = static_cast<const _Float16 *>(c.in(V, vb));
        a.out = static_cast<_Float16 *>(c.out(out, ob));
        if (!a.Q || !a.Kf || !a.Vf || !a.out) return c.finish();
        uint64_t blocks = 0;
        if (pb) {
            _Float16 *const vp = static_cast<_Float16 *>(c.scratch(pb));
            if (!vp) return c.finish();
            if (pad_cols_f16(a.Vf, vp, (long)n_kv_heads * dv, nullptr, nullptr, 0, kv_stride, padded, c.stream(), &blocks) != hipSuccess)
                return launched(c, hipErrorInvalidValue, 0);
            count_launch(blocks);
            a.Vf = vp;
            a.stride = padded;
        }
        a.ws = static_cast<float *>(c.optional(ws));
        a.ws_bytes = a.ws ? ws : 0;
        return launched(c, serve_attn(a, c.stream(), &blocks), blocks);
    });
}

}  // extern "C"
