// serve_ref.cpp — the host paths of rocket_serve.h (fd < 0): the cache's layout and quantiser, and
// fp64 forms of the rotation and of attention, every result rounded to fp16 once.
#include "serve.h"

#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

namespace rk {

bool kv4_layout(const rocket_kv4_shape *s, Kv4Layout *l)
{
    if (!s || s->n_seq < 1 || s->n_kv_heads < 1 || s->capacity < 1 || s->capacity > kServeMaxCap) return false;
    if ((long)s->n_seq * s->n_kv_heads > 65535) return false;
    for (int d : {s->head_dim, s->dv})
        if (d < 32 || d % 32 || d > kServeMaxDim) return false;
    l->cap = (s->capacity + 31) / 32 * 32;
    const size_t rows = (size_t)s->n_seq * s->n_kv_heads * l->cap;
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    l->kc = 0;
    l->ks = up(rows * (s->head_dim / 2));
    l->vc = l->ks + up(rows * (s->head_dim / 32 * 4));
    l->vs = l->vc + up(rows * (s->dv / 2));
    l->bytes = l->vs + up(rows * (s->dv / 32 * 4));
    return true;
}

Kv4View kv4_view(const rocket_kv4_shape &s, const Kv4Layout &l, void *cache, int seq0, int n_seq)
{
    const size_t row0 = (size_t)seq0 * s.n_kv_heads * l.cap;
    char *b = static_cast<char *>(cache);
    Kv4View v;
    v.kc = b + l.kc + row0 * (s.head_dim / 2);
    v.ks = b + l.ks + row0 * (s.head_dim / 32 * 4);
    v.vc = b + l.vc + row0 * (s.dv / 2);
    v.vs = b + l.vs + row0 * (s.dv / 32 * 4);
    v.heads = s.n_kv_heads; v.dk = s.head_dim; v.dv = s.dv; v.cap = l.cap; v.capacity = s.capacity; v.n_seq = n_seq;
    return v;
}

namespace {

struct ScaleMin { _Float16 s, m; };

// Where group g (32 values) of position j of head row `hr` (place * heads + head) lies.
struct Group {
    uint8_t *code[4];   // eight values each
    ScaleMin *sm;
};
Group key_group(const Kv4View &c, size_t hr, long j, int g)
{
    const size_t row = hr * c.cap + j;
    Group x;
    for (int i = 0; i < 4; i++) x.code[i] = reinterpret_cast<uint8_t *>(c.kc) + row * (c.dk / 2) + 16 * g + 4 * i;
    x.sm = reinterpret_cast<ScaleMin *>(c.ks) + row * (c.dk / 32) + g;
    return x;
}
Group value_group(const Kv4View &c, size_t hr, long j, int g)
{
    const size_t block = hr * (c.cap / 8) + j / 8;
    Group x;
    for (int i = 0; i < 4; i++)
        x.code[i] = reinterpret_cast<uint8_t *>(c.vc) + ((block * (c.dv / 8) + 4 * g + i) * 8 + j % 8) * 4;
    x.sm = reinterpret_cast<ScaleMin *>(c.vs) + (block * (c.dv / 32) + g) * 8 + j % 8;
    return x;
}

void store(const Group &x, const _Float16 *src)
{
    float v[32], lo = INFINITY, hi = -INFINITY;
    for (int i = 0; i < 32; i++) {
        v[i] = kv4_finite((float)src[i]);
        lo = std::min(lo, v[i]);
        hi = std::max(hi, v[i]);
    }
    lo += 0.f;   // (-0 becomes 0)
    const _Float16 s = kv4_scale(lo, hi);
    for (int i = 0; i < 4; i++)
        for (int b = 0; b < 4; b++)
            x.code[i][b] = (uint8_t)(kv4_code(v[8 * i + 2 * b], lo, (float)s) | kv4_code(v[8 * i + 2 * b + 1], lo, (float)s) << 4);
    *x.sm = ScaleMin{s, (_Float16)lo};
}

// (a double holds code * scale + minimum exactly)
double value(const Group &x, int i)
{
    const int byte = x.code[i / 8][i % 8 / 2];
    return (double)(i & 1 ? byte >> 4 : byte & 15) * (double)x.sm->s + (double)x.sm->m;
}

}  // namespace

void kv4_append_ref(const Kv4View &c, const Kv4Rows &r)
{
    for (int s = 0; s < c.n_seq; s++)
        for (int t = 0; t < r.n_tokens; t++) {
            const long j = (long)r.seq_len[s] - r.n_tokens + t;
            if (j < 0 || j >= c.capacity) continue;
            for (int h = 0; h < c.heads; h++) {
                const size_t hr = (size_t)s * c.heads + h;
                for (int g = 0; g < c.dk / 32; g++) store(key_group(c, hr, j, g), r.K + s * r.k_ss + h * r.k_hs + t * r.k_rs + 32 * g);
                for (int g = 0; g < c.dv / 32; g++) store(value_group(c, hr, j, g), r.V + s * r.v_ss + h * r.v_hs + t * r.v_rs + 32 * g);
            }
        }
}

void kv4_read_ref(const Kv4View &c, const Kv4Rows &r)
{
    for (int s = 0; s < c.n_seq; s++)
        for (int h = 0; h < c.heads; h++)
            for (int t = 0; t < r.n_tokens; t++) {
                const long j = (long)r.seq_len[s] - r.n_tokens + t;
                const bool in = j >= 0 && j < c.capacity;
                const size_t hr = (size_t)s * c.heads + h, row = hr * r.n_tokens + t;
                for (int i = 0; r.Ko && i < c.dk; i++) r.Ko[row * c.dk + i] = in ? (_Float16)value(key_group(c, hr, j, i / 32), i % 32) : (_Float16)0.f;
                for (int i = 0; r.Vo && i < c.dv; i++) r.Vo[row * c.dv + i] = in ? (_Float16)value(value_group(c, hr, j, i / 32), i % 32) : (_Float16)0.f;
            }
}

bool qk_norm_rope_ref(const RopeLaunch &L)
try {
    std::vector<double> y((size_t)L.dim);
    const int half = L.rot / 2;
    for (int s = 0; s < L.n_seq; s++)
        for (int t = 0; t < L.n_tokens; t++)
            for (int h = 0; h < L.n_head + L.n_kv; h++) {
                const bool key = h >= L.n_head;
                const int hh = key ? h - L.n_head : h, heads = key ? L.n_kv : L.n_head;
                const size_t m = (size_t)s * L.n_tokens + t;
                const size_t at = m * (key ? L.k_rs : L.q_rs) + (size_t)hh * L.dim;
                const void *x = key ? L.k : L.q;
                const _Float16 *w = key ? L.wk : L.wq;
                double sq = 0;
                for (int i = 0; i < L.dim; i++) {
                    y[i] = L.f32 ? (double)static_cast<const float *>(x)[at + i] : (double)static_cast<const _Float16 *>(x)[at + i];
                    sq += y[i] * y[i];
                }
                if (L.norm)
                    for (int i = 0; i < L.dim; i++) y[i] = y[i] / sqrt(sq / L.dim + (double)L.eps) * (w ? (double)w[i] : 1.0);
                for (int j = 0; j < half; j++) {
                    const double a = (double)L.pos[m] * (double)L.inv_freq[j], c = cos(a), n = sin(a);
                    double &u = y[L.pairs ? 2 * j : j], &v = y[L.pairs ? 2 * j + 1 : j + half];
                    const double u0 = u;
                    u = u0 * c - v * n;
                    v = v * c + u0 * n;
                }
                _Float16 *o = (key ? L.k_out : L.q_out) + (((size_t)s * heads + hh) * L.n_tokens + t) * L.dim;
                for (int i = 0; i < L.dim; i++) o[i] = (_Float16)y[i];
            }
    return true;
} catch (const std::bad_alloc &) {
    return false;
}

bool serve_attn_ref(const ServeAttn &a)
try {
    std::vector<double> p((size_t)a.max_kv), o((size_t)a.dv), key((size_t)a.dk);
    const int kvh = a.n_head / a.gqa;
    for (int s = 0; s < a.n_seq; s++) {
        const int n = a.seq_len ? a.seq_len[s] : a.max_kv;
        const bool served = n >= 1 && n <= a.max_kv;
        for (int h = 0; h < a.n_head; h++)
            for (int t = 0; t < a.n_tokens; t++) {
                const size_t row = ((size_t)s * a.n_head + h) * a.n_tokens + t, hr = (size_t)s * kvh + h / a.gqa;
                const _Float16 *q = a.Q + row * a.dk;
                const long pos = (long)n - a.n_tokens + t;
                auto sees = [&](long j) { return j <= pos && (!a.window || j > pos - a.window || j < a.sinks); };
                double mx = -INFINITY, sum = 0;
                for (long j = 0; served && j <= pos; j++) {
                    if (!sees(j)) continue;
                    double x = 0;
                    for (int i = 0; i < a.dk; i++)
                        x += (double)q[i] * (a.Kf ? (double)a.Kf[(size_t)(h / a.gqa) * a.k_hs + (size_t)j * a.dk + i] : value(key_group(a.c, hr, j, i / 32), i % 32));
                    x *= (double)a.scale;
                    if (a.softcap != 0.f) x = (double)a.softcap * tanh(x / (double)a.softcap);
                    p[j] = x;
                    mx = std::max(mx, x);
                }
                std::fill(o.begin(), o.end(), 0.0);
                for (long j = 0; served && j <= pos; j++) {
                    if (!sees(j)) continue;
                    const double w = exp(p[j] - mx);
                    sum += w;
                    for (int i = 0; i < a.dv; i++)
                        o[i] += w * (a.Kf ? (double)a.Vf[((size_t)(h / a.gqa) * a.dv + i) * a.stride + j] : value(value_group(a.c, hr, j, i / 32), i % 32));
                }
                for (int i = 0; i < a.dv; i++) a.out[row * a.dv + i] = (_Float16)(sum == 0 ? 0.0 : o[i] / sum);
            }
    }
    return true;
} catch (const std::bad_alloc &) {
    return false;
}

}  // namespace rk
