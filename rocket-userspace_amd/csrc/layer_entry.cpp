// layer_entry.cpp — rocket_fp8.h and rocket_layer.h: argument checks, staging and launches of the products of e4m3 codes
// (fp8_gemm.hip, fp8_rows.hip), their quantisation (fp8_quant.hip), block norms (add_norm.hip) and routing (moe_route.hip).
#include "internal.h"
#include "layer.h"
#include "ops.h"

#include <math.h>
#include <string.h>

#include <new>

using namespace rk;

namespace {

constexpr int64_t kMaxSpan = (int64_t)1 << 40;   // elements of strided rows
constexpr size_t kIntAlign = sizeof(int32_t);

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

int bad(const char *who, const char *what)
{
    ROCKET_LOGE("%s: %s\n", who, what);
    return ROCKET_E_SHAPE;
}

// One operand of a call: where it is, its bytes, the launch's pointer to it (of any type), and the alignment that the kernels need.
// part: a result that the launch may write in part, whose rest has to stay.
struct Operand {
    const void *p;
    size_t bytes;
    void *to;
    size_t align = 16;
    bool part = false;
    void set(const void *at) const { memcpy(to, &at, sizeof at); }
};
template <class T> Operand operand(T *&p, size_t bytes, size_t align = 16)
{
    return {p, bytes, const_cast<void *>(static_cast<const volatile void *>(&p)), align};
}
template <class T> Operand in_part(T *&p, size_t bytes, bool part = true, size_t align = 16)
{
    Operand o = operand(p, bytes, align);
    o.part = part;
    return o;
}

bool overlap(const void *a, size_t an, const void *b, size_t bn)
{
    return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

// Results over operands or each other; `in_place`: the first result may be the first operand, whole.
template <size_t NI, size_t NO> bool clash(const Operand (&in)[NI], const Operand (&out)[NO], bool in_place = false)
{
    for (size_t o = 0; o < NO; o++) {
        for (size_t i = 0; i < NI; i++)
            if (overlap(in[i].p, in[i].bytes, out[o].p, out[o].bytes) && !(in_place && !o && !i && in[i].p == out[o].p)) return true;
        for (size_t u = 0; u < o; u++)
            if (overlap(out[o].p, out[o].bytes, out[u].p, out[u].bytes)) return true;
    }
    return false;
}

// Stages the operands on the handle, has `go` launch, and finishes the call. Scratch: bytes that the launch needs (needed) or
// can do without.
template <size_t NI, size_t NO, class F>
int on_gpu(const char *who, int fd, const Operand (&in)[NI], const Operand (&out)[NO], size_t needed, size_t optional, F &&go)
{
    Locked lk(fd);
    if (!lk.ok()) {
        ROCKET_LOGE("%s: fd %d is not an open rocket handle\n", who, fd);
        return ROCKET_E_DEVICE;
    }
    Call c(lk.h, who);
    for (const Operand &i : in)
        if (i.p) c.want(i.p, i.bytes, i.align);
    for (const Operand &o : out)
        if (o.p) c.want(o.p, o.bytes, o.align);
    if (needed) c.want_scratch(needed);
    const size_t opt = optional ? c.want_optional(optional, true) : 0;
    if (int rc = c.begin()) return rc;
    for (const Operand &i : in) {
        const void *at = i.p ? c.in(i.p, i.bytes, i.align) : nullptr;
        if (i.p && !at) return c.finish();
        i.set(at);
    }
    for (const Operand &o : out) {
        const void *at = o.p ? c.out(const_cast<void *>(o.p), o.bytes, o.align) : nullptr;
        if (o.p && !at) return c.finish();
        if (o.part && at != o.p && hipMemcpyAsync(const_cast<void *>(at), o.p, o.bytes, hipMemcpyDefault, c.stream()) != hipSuccess) {
            (void)hipGetLastError();
            ROCKET_LOGE("%s: host-to-device copy failed\n", who);
            (void)c.finish();
            return ROCKET_E_DEVICE;
        }
        o.set(at);
    }
    void *scratch = needed ? c.scratch(needed) : c.optional(opt);
    if (needed && !scratch) return c.finish();
    uint64_t blocks = 0;
    const hipError_t e = go(scratch, c.stream(), &blocks);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        ROCKET_LOGE("%s: kernel launch rejected: %s\n", who, hipGetErrorString(e));
        (void)c.finish();
        return e == hipErrorInvalidValue ? ROCKET_E_SHAPE : ROCKET_E_DEVICE;
    }
    count_launch(blocks);
    return c.finish();
}

// ---- quantisation ----
int quantise(const char *who, int fd, QuantF8 L, bool gated)
{
    if (L.M < 1 || L.M > kDimMax || L.K < 8 || L.K % 8 || L.K > kF8MaxK) return bad(who, "M below 1 or too large, or K no multiple of 8 up to 65536");
    if (L.rs < L.K || L.rs % 8 || L.rs > kMaxSpan / L.M) return bad(who, "a row stride is a multiple of 8 and holds the row, and all rows are up to 2^40 values");
    if (gated && L.act != kActSilu && L.act != kActGelu) return bad(who, "the activation is neither SiLU nor GELU");
    if (!L.a || (gated && !L.up) || !L.q || !L.scale) return bad(who, "null operand");
    const int nb = f8_blocks(L.K);
    if ((int64_t)L.M * nb >= (int64_t)1 << 31) return bad(who, "too many values");
    const size_t rows = (size_t)L.M, ab = ((rows - 1) * L.rs + L.K) * (L.f32 ? sizeof(float) : sizeof(_Float16));
    const Operand in[] = {operand(L.a, ab), operand(L.up, ab), operand(L.n_rows, sizeof(int32_t), kIntAlign)};
    const Operand out[] = {in_part(L.q, rows * L.K, L.n_rows), in_part(L.scale, rows * nb * sizeof(float), L.n_rows)};
    if (clash(in, out)) return bad(who, "results over operands or each other");
    if (fd < 0) {
        quant_fp8_ref(L);
        return ROCKET_OK;
    }
    return on_gpu(who, fd, in, out, 0, 0, [&](void *, hipStream_t s, uint64_t *blocks) { return quant_fp8(L, s, blocks); });
}

// ---- products ----
int product(const char *who, int fd, GemmF8 L, bool grouped)
{
    if (L.M < 1 || L.M > kDimMax || L.N < 1 || L.N > kDimMax || L.K < 16 || L.K % 16 || L.K > kF8MaxK)
        return bad(who, "M or N below 1 or too large, or K no multiple of 16 up to 65536");
    if (grouped && (L.n_expert < 1 || L.n_expert > kMaxExperts)) return bad(who, "n_expert outside [1, 1024]");
    if (grouped && (L.a_rows < 1 || (!L.src && L.a_rows < L.M) || (int64_t)L.a_rows * L.K >= (int64_t)1 << 31))
        return bad(who, "a_rows below 1, or fewer than the rows that are read in order, or a_rows * K too large");
    if (!L.A || !L.sa || !L.B || !L.sb || !L.C || (grouped && !L.off)) return bad(who, "null operand");
    if (!grouped) L.a_rows = L.M;
    const size_t nb = f8_blocks(L.K), E = (size_t)L.n_expert, bn = f8_blocks(L.N);
    const Operand in[] = {operand(L.A, (size_t)L.a_rows * L.K), operand(L.sa, (size_t)L.a_rows * nb * sizeof(float)),
                          operand(L.B, E * L.N * L.K), operand(L.sb, E * bn * nb * sizeof(float)),
                          operand(L.src, (size_t)L.M * sizeof(int32_t), kIntAlign), operand(L.off, (E + 1) * sizeof(int32_t), kIntAlign)};
    const Operand out[] = {in_part(L.C, (size_t)L.M * L.N * (L.f16 ? sizeof(_Float16) : sizeof(float)), grouped)};
    if (clash(in, out)) return bad(who, "results over operands");
    if (fd < 0) return gemm_fp8_ref(L) ? ROCKET_OK : ROCKET_E_NOMEM;
    const size_t ws_bytes = gemm_fp8_plan(L);
    return on_gpu(who, fd, in, out, 0, ws_bytes, [&](void *ws, hipStream_t s, uint64_t *blocks) {
        L.ws = static_cast<float *>(ws);
        return gemm_fp8(L, s, blocks);
    });
}

// ---- norms ----
int norms(const char *who, int fd, AddNorm L, bool experts)
{
    if (L.M < 1 || L.M > kDimMax || L.H < 8 || L.H % 8 || L.H > kNormMaxH) return bad(who, "M below 1 or too large, or H no multiple of 8 up to 16384");
    if (isnan(L.eps_post) || isnan(L.eps_pre) || !isfinite(L.alpha)) return bad(who, "eps is NaN or alpha not finite");
    if ((L.eps_post < 0.f && L.w_post) || (L.eps_pre < 0.f && L.w_pre)) return bad(who, "weights without a norm");
    if (!L.h || (!L.h_out && !L.x && !L.xq) || !L.xq != !L.x_scale) return bad(who, "null operand, or codes without scales");
    if (L.gate && L.gate_every < 1) return bad(who, "gate_every below 1");
    if (experts) {
        if (L.top_k < 1 || L.top_k > kMaxTop || L.rows < 1 || L.rows > kDimMax) return bad(who, "top_k outside [1, 32], or rows below 1 or too large");
        if (!L.y || !L.slot || !L.weight) return bad(who, "null operand");
    } else if (L.y && (L.y_rs < L.H || L.y_rs % 8 || L.y_rs > kMaxSpan / L.M)) {
        return bad(who, "a row stride is a multiple of 8 and holds the row, and all rows are up to 2^40 values");
    }
    const size_t e = L.f32 ? sizeof(float) : sizeof(_Float16), rows = (size_t)L.M, hb = rows * L.H * e, wb = (size_t)L.H * sizeof(_Float16);
    const size_t yb = !L.y ? 0 : experts ? (size_t)L.rows * L.H * e : ((rows - 1) * L.y_rs + L.H) * e;
    const size_t gb = L.gate ? ((rows - 1) / L.gate_every + 1) * wb : 0, jb = rows * L.top_k * 4, nb = f8_blocks(L.H);
    const Operand in[] = {operand(L.h, hb), operand(L.y, yb), operand(L.shared, hb), operand(L.w_post, wb), operand(L.w_pre, wb),
                          operand(L.gate, gb), operand(L.slot, jb, kIntAlign), operand(L.weight, jb, kIntAlign)};
    const Operand out[] = {operand(L.h_out, hb), operand(L.x, rows * L.H * sizeof(_Float16)), operand(L.xq, rows * L.H),
                           operand(L.x_scale, rows * nb * sizeof(float))};
    if (clash(in, out, true)) return bad(who, "results over operands or each other");
    if (fd < 0) return add_norm_ref(L) ? ROCKET_OK : ROCKET_E_NOMEM;
    return on_gpu(who, fd, in, out, 0, 0, [&](void *, hipStream_t s, uint64_t *blocks) { return add_norm(L, s, blocks); });
}

// ---- routing ----
int route(const char *who, int fd, Route L, int score)
{
    if (L.M < 1 || L.M > kDimMax || L.E < 1 || L.E > kMaxExperts) return bad(who, "M below 1 or too large, or E outside [1, 1024]");
    if (L.top_k < 1 || L.top_k > kMaxTop || L.top_k > L.E || (int64_t)L.M * L.top_k >= kDimMax) return bad(who, "top_k outside [1, min(32, E)], or too many choices");
    if (L.n_group < 1 || L.n_group > kMaxGroups || L.E % L.n_group || L.top_group < 1 || L.top_group > L.n_group || L.group_best < 1 || L.group_best > 2)
        return bad(who, "n_group outside [1, 64] or no divisor of E, top_group outside [1, n_group], or group_best neither 1 nor 2");
    if (score != ROCKET_ROUTE_SOFTMAX && score != ROCKET_ROUTE_SIGMOID) return bad(who, "unknown score");
    if (L.rs < L.E || L.rs > kMaxSpan / L.M) return bad(who, "a row stride below E or too large");
    if (!isfinite(L.scale)) return bad(who, "scale is not finite");
    if (!L.logits || !L.ids || !L.weight || !L.off != !L.src || !L.off != !L.slot) return bad(who, "null operand, or a part of the plan");
    L.sigmoid = score == ROCKET_ROUTE_SIGMOID;
    const size_t rows = (size_t)L.M, e = L.f32 ? sizeof(float) : sizeof(_Float16), kb = rows * L.top_k * 4;
    const Operand in[] = {operand(L.logits, ((rows - 1) * L.rs + L.E) * e, e), operand(L.bias, (size_t)L.E * sizeof(float), kIntAlign),
                          operand(L.active, rows, 1)};
    const Operand out[] = {operand(L.ids, kb, kIntAlign), operand(L.weight, kb, kIntAlign), operand(L.off, ((size_t)L.E + 1) * sizeof(int32_t), kIntAlign),
                           in_part(L.src, kb, true, kIntAlign), operand(L.slot, kb, kIntAlign)};
    if (clash(in, out)) return bad(who, "results over operands or each other");
    if (fd < 0) return moe_route_ref(L) ? ROCKET_OK : ROCKET_E_NOMEM;
    return on_gpu(who, fd, in, out, route_ws(L), 0, [&](void *ws, hipStream_t s, uint64_t *blocks) {
        L.counts = static_cast<int32_t *>(ws);
        return moe_route(L, s, blocks);
    });
}

}  // namespace

extern "C" {

int rocket_quantize_rows_fp8(int fd, int M, int K, const float *A, int64_t a_rs, uint8_t *Aq, float *a_scale)
{
    static const char *who = "rocket_quantize_rows_fp8";
    QuantF8 L;
    L.a = A; L.rs = a_rs; L.f32 = true; L.M = M; L.K = K; L.q = Aq; L.scale = a_scale;
    return guarded(who, [&] { return quantise(who, fd, L, false); });
}

int rocket_quantize_rows_fp8_fp16(int fd, int M, int K, const _Float16 *A, int64_t a_rs, uint8_t *Aq, float *a_scale)
{
    static const char *who = "rocket_quantize_rows_fp8_fp16";
    QuantF8 L;
    L.a = A; L.rs = a_rs; L.M = M; L.K = K; L.q = Aq; L.scale = a_scale;
    return guarded(who, [&] { return quantise(who, fd, L, false); });
}

int rocket_quantize_glu_fp8(int fd, int M, int K, const float *gate, const float *up, int64_t rs, int act, const int32_t *n_rows, uint8_t *Aq,
                            float *a_scale)
{
    static const char *who = "rocket_quantize_glu_fp8";
    QuantF8 L;
    L.a = gate; L.up = up; L.rs = rs; L.f32 = true; L.act = act; L.M = M; L.K = K; L.n_rows = n_rows; L.q = Aq; L.scale = a_scale;
    return guarded(who, [&] { return quantise(who, fd, L, true); });
}

int rocket_quantize_glu_fp8_fp16(int fd, int M, int K, const _Float16 *gate, const _Float16 *up, int64_t rs, int act, const int32_t *n_rows,
                                 uint8_t *Aq, float *a_scale)
{
    static const char *who = "rocket_quantize_glu_fp8_fp16";
    QuantF8 L;
    L.a = gate; L.up = up; L.rs = rs; L.act = act; L.M = M; L.K = K; L.n_rows = n_rows; L.q = Aq; L.scale = a_scale;
    return guarded(who, [&] { return quantise(who, fd, L, true); });
}

int rocket_matmul_fp8_block(int fd, int M, int K, int N, const uint8_t *A, const float *a_scale, const uint8_t *B, const float *b_scale, float *C)
{
    static const char *who = "rocket_matmul_fp8_block";
    GemmF8 L;
    L.A = A; L.B = B; L.sa = a_scale; L.sb = b_scale; L.C = C; L.M = M; L.K = K; L.N = N;
    return guarded(who, [&] { return product(who, fd, L, false); });
}

int rocket_matmul_fp8_block_f16out(int fd, int M, int K, int N, const uint8_t *A, const float *a_scale, const uint8_t *B, const float *b_scale,
                                   _Float16 *C)
{
    static const char *who = "rocket_matmul_fp8_block_f16out";
    GemmF8 L;
    L.A = A; L.B = B; L.sa = a_scale; L.sb = b_scale; L.C = C; L.f16 = true; L.M = M; L.K = K; L.N = N;
    return guarded(who, [&] { return product(who, fd, L, false); });
}

int rocket_matmul_fp8_block_grouped(int fd, int n_expert, int rows, int a_rows, int K, int N, const uint8_t *A, const float *a_scale,
                                    const int32_t *src_row, const int32_t *expert_off, const uint8_t *B, const float *b_scale, float *C)
{
    static const char *who = "rocket_matmul_fp8_block_grouped";
    GemmF8 L;
    L.A = A; L.B = B; L.sa = a_scale; L.sb = b_scale; L.src = src_row; L.off = expert_off; L.C = C; L.M = rows; L.K = K; L.N = N;
    L.n_expert = n_expert; L.a_rows = a_rows;
    return guarded(who, [&] { return product(who, fd, L, true); });
}

int rocket_matmul_fp8_block_grouped_f16out(int fd, int n_expert, int rows, int a_rows, int K, int N, const uint8_t *A, const float *a_scale,
                                           const int32_t *src_row, const int32_t *expert_off, const uint8_t *B, const float *b_scale, _Float16 *C)
{
    static const char *who = "rocket_matmul_fp8_block_grouped_f16out";
    GemmF8 L;
    L.A = A; L.B = B; L.sa = a_scale; L.sb = b_scale; L.src = src_row; L.off = expert_off; L.C = C; L.f16 = true; L.M = rows; L.K = K; L.N = N;
    L.n_expert = n_expert; L.a_rows = a_rows;
    return guarded(who, [&] { return product(who, fd, L, true); });
}

int rocket_add_norm_fp16(int fd, int M, int H, const _Float16 *h, const _Float16 *y, int64_t y_rs, const _Float16 *w_post, float eps_post,
                         const _Float16 *gate, int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, _Float16 *h_out, _Float16 *x,
                         uint8_t *xq, float *x_scale)
{
    static const char *who = "rocket_add_norm_fp16";
    AddNorm L;
    L.h = h; L.y = y; L.y_rs = y_rs; L.h_out = h_out; L.w_post = w_post; L.w_pre = w_pre; L.gate = gate; L.eps_post = eps_post; L.eps_pre = eps_pre;
    L.alpha = alpha; L.gate_every = gate_every; L.M = M; L.H = H; L.x = x; L.xq = xq; L.x_scale = x_scale;
    return guarded(who, [&] { return norms(who, fd, L, false); });
}

int rocket_add_norm_f32(int fd, int M, int H, const float *h, const float *y, int64_t y_rs, const _Float16 *w_post, float eps_post,
                        const _Float16 *gate, int gate_every, float alpha, const _Float16 *w_pre, float eps_pre, float *h_out, _Float16 *x,
                        uint8_t *xq, float *x_scale)
{
    static const char *who = "rocket_add_norm_f32";
    AddNorm L;
    L.f32 = true;
    L.h = h; L.y = y; L.y_rs = y_rs; L.h_out = h_out; L.w_post = w_post; L.w_pre = w_pre; L.gate = gate; L.eps_post = eps_post; L.eps_pre = eps_pre;
    L.alpha = alpha; L.gate_every = gate_every; L.M = M; L.H = H; L.x = x; L.xq = xq; L.x_scale = x_scale;
    return guarded(who, [&] { return norms(who, fd, L, false); });
}

int rocket_moe_add_norm_fp16(int fd, int M, int H, const _Float16 *h, int rows, int top_k, const _Float16 *Y, const int32_t *slot, const float *weight,
                             const _Float16 *shared, const _Float16 *w_post, float eps_post, const _Float16 *gate, int gate_every, float alpha,
                             const _Float16 *w_pre, float eps_pre, _Float16 *h_out, _Float16 *x, uint8_t *xq, float *x_scale)
{
    static const char *who = "rocket_moe_add_norm_fp16";
    AddNorm L;
    L.h = h; L.y = Y; L.shared = shared; L.slot = slot; L.weight = weight; L.rows = rows; L.top_k = top_k; L.h_out = h_out; L.w_post = w_post;
    L.w_pre = w_pre; L.gate = gate; L.eps_post = eps_post; L.eps_pre = eps_pre; L.alpha = alpha; L.gate_every = gate_every; L.M = M; L.H = H;
    L.x = x; L.xq = xq; L.x_scale = x_scale;
    return guarded(who, [&] { return norms(who, fd, L, true); });
}

int rocket_moe_add_norm_f32(int fd, int M, int H, const float *h, int rows, int top_k, const float *Y, const int32_t *slot, const float *weight,
                            const float *shared, const _Float16 *w_post, float eps_post, const _Float16 *gate, int gate_every, float alpha,
                            const _Float16 *w_pre, float eps_pre, float *h_out, _Float16 *x, uint8_t *xq, float *x_scale)
{
    static const char *who = "rocket_moe_add_norm_f32";
    AddNorm L;
    L.f32 = true;
    L.h = h; L.y = Y; L.shared = shared; L.slot = slot; L.weight = weight; L.rows = rows; L.top_k = top_k; L.h_out = h_out; L.w_post = w_post;
    L.w_pre = w_pre; L.gate = gate; L.eps_post = eps_post; L.eps_pre = eps_pre; L.alpha = alpha; L.gate_every = gate_every; L.M = M; L.H = H;
    L.x = x; L.xq = xq; L.x_scale = x_scale;
    return guarded(who, [&] { return norms(who, fd, L, true); });
}

int rocket_moe_route_f32(int fd, int M, int E, const float *logits, int64_t rs, int score, const float *bias, int n_group, int group_best, int top_group,
                         int top_k, int renorm, float scale, const uint8_t *active, int32_t *ids, float *weight, int32_t *expert_off, int32_t *src_row,
                         int32_t *slot)
{
    static const char *who = "rocket_moe_route_f32";
    Route L;
    L.f32 = true;
    L.logits = logits; L.rs = rs; L.bias = bias; L.active = active; L.M = M; L.E = E; L.n_group = n_group; L.group_best = group_best;
    L.top_group = top_group; L.top_k = top_k; L.renorm = renorm != 0; L.scale = scale; L.ids = ids; L.weight = weight; L.off = expert_off;
    L.src = src_row; L.slot = slot;
    return guarded(who, [&] { return route(who, fd, L, score); });
}

int rocket_moe_route_fp16(int fd, int M, int E, const _Float16 *logits, int64_t rs, int score, const float *bias, int n_group, int group_best,
                          int top_group, int top_k, int renorm, float scale, const uint8_t *active, int32_t *ids, float *weight, int32_t *expert_off,
                          int32_t *src_row, int32_t *slot)
{
    static const char *who = "rocket_moe_route_fp16";
    Route L;
    L.logits = logits; L.rs = rs; L.bias = bias; L.active = active; L.M = M; L.E = E; L.n_group = n_group; L.group_best = group_best;
    L.top_group = top_group; L.top_k = top_k; L.renorm = renorm != 0; L.scale = scale; L.ids = ids; L.weight = weight; L.off = expert_off;
    L.src = src_row; L.slot = slot;
    return guarded(who, [&] { return route(who, fd, L, score); });
}

}  // extern "C"
