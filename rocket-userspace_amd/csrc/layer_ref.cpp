// layer_ref.cpp — the host paths (fd < 0) of rocket_fp8.h and rocket_layer.h: codes by the formula in fp32, products, norms and
// scores in fp64, each result rounded once.
#include "gemm.h"
#include "host_ref.h"
#include "layer.h"

#include <algorithm>
#include <new>
#include <vector>

namespace rk {

namespace {

double f8_value(uint8_t c)
{
    const int e = c >> 3 & 15, f = c & 7;
    const double v = e == 15 && f == 7 ? (double)NAN : e ? ldexp(8 + f, e - 10) : ldexp(f, -9);
    return c & 0x80 ? -v : v;
}

// The nearest e4m3 code of |v| <= 448, ties to the even one.
uint8_t f8_code(float v)
{
    if (v != v) return 0x7f;
    const uint8_t sign = std::signbit(v) ? 0x80 : 0;
    const double x = fabs((double)v);
    int e = x > 0 ? std::max(ilogb(x), -6) : -6;
    int f = (int)nearbyint(ldexp(x, 3 - e));   // 0 .. 16, in steps of 2^(e - 3)
    if (f == 16) f = 8, e++;
    return (uint8_t)(sign | (f < 8 ? f : (e + 7) << 3 | (f - 8)));
}

void quantise(const float *v, int n, uint8_t *q, float *scale)
{
    float a = 0.f;
    for (int i = 0; i < n; i++) a = fmaxf(a, fabsf(v[i]));
    a = f8_amax(a);
    const float s = 448.f / a;
    for (int i = 0; i < n; i++) q[i] = f8_code(f8_clamp(v[i] * s));
    *scale = a / 448.f;
}

float at(const void *p, bool f32, size_t i) { return f32 ? static_cast<const float *>(p)[i] : (float)static_cast<const _Float16 *>(p)[i]; }

}  // namespace

void quant_fp8_ref(const QuantF8 &L)
{
    const int nb = f8_blocks(L.K);
    float v[kF8Block];
    for (int m = 0; m < L.M && (!L.n_rows || m < *L.n_rows); m++)
        for (int b = 0; b < nb; b++) {
            const int k0 = b * kF8Block, n = std::min(kF8Block, L.K - k0);
            for (int i = 0; i < n; i++) {
                const size_t j = (size_t)m * L.rs + k0 + i;
                v[i] = at(L.a, L.f32, j);
                if (L.act) v[i] = (float)(hostref::activation(L.act, v[i]) * (double)at(L.up, L.f32, j));
            }
            quantise(v, n, L.q + (size_t)m * L.K + k0, L.scale + (size_t)m * nb + b);
        }
}

bool gemm_fp8_ref(const GemmF8 &L)
{
    const int nb = f8_blocks(L.K), nbn = f8_blocks(L.N);
    std::vector<double> row;
    try {
        row.resize(L.K);
    } catch (const std::bad_alloc &) {
        return false;
    }
    double value[256];
    for (int i = 0; i < 256; i++) value[i] = f8_value((uint8_t)i);
    for (int e = 0; e < L.n_expert; e++) {
        const int lo = L.off ? std::min(std::max(L.off[e], 0), L.M) : 0, hi = L.off ? std::min(std::max(L.off[e + 1], lo), L.M) : L.M;
        for (int m = lo; m < hi; m++) {
            const int r = L.src ? L.src[m] : m;
            const bool in = !L.src || (r >= 0 && r < L.a_rows);
            for (int k = 0; k < L.K; k++) row[k] = in ? value[L.A[(size_t)r * L.K + k]] : 0.0;
            for (int n = 0; n < L.N; n++) {
                const uint8_t *b = L.B + ((size_t)e * L.N + n) * L.K;
                const float *sb = L.sb + ((size_t)e * nbn + n / kF8Block) * nb;
                double sum = 0.0;
                for (int g = 0; in && g < nb; g++) {
                    double p = 0.0;
                    for (int k = g * kF8Block; k < std::min(L.K, (g + 1) * kF8Block); k++) p += row[k] * value[b[k]];
                    sum += p * ((double)L.sa[(size_t)r * nb + g] * (double)sb[g]);
                }
                const size_t o = (size_t)m * L.N + n;
                if (L.f16) static_cast<_Float16 *>(L.C)[o] = (_Float16)sum;
                else static_cast<float *>(L.C)[o] = (float)sum;
            }
        }
    }
    return true;
}

bool add_norm_ref(const AddNorm &L)
{
    std::vector<double> z, h;
    std::vector<float> x;
    try {
        z.resize(L.H);
        h.resize(L.H);
        x.resize(L.H);
    } catch (const std::bad_alloc &) {
        return false;
    }
    const auto norm = [&](std::vector<double> &v, const _Float16 *w, float eps) {
        if (!(eps >= 0.f)) return;
        double q = 0.0;
        for (double t : v) q += t * t;
        const double r = 1.0 / sqrt(q / L.H + (double)eps);
        for (int i = 0; i < L.H; i++) v[i] *= r * (w ? (double)w[i] : 1.0);
    };
    const int nb = f8_blocks(L.H);
    for (int m = 0; m < L.M; m++) {
        const size_t row = (size_t)m * L.H;
        for (int i = 0; i < L.H; i++) h[i] = at(L.h, L.f32, row + i);
        if (L.y) {
            for (int i = 0; i < L.H; i++) z[i] = L.top_k ? (L.shared ? at(L.shared, L.f32, row + i) : 0.0) : (double)at(L.y, L.f32, (size_t)m * L.y_rs + i);
            for (int j = 0; j < L.top_k; j++) {
                const int r = L.slot[(size_t)m * L.top_k + j];
                if (r < 0 || r >= L.rows) continue;
                const double w = L.weight[(size_t)m * L.top_k + j];
                for (int i = 0; i < L.H; i++) z[i] += w * (double)at(L.y, L.f32, (size_t)r * L.H + i);
            }
            norm(z, L.w_post, L.eps_post);
            for (int i = 0; i < L.H; i++) h[i] += (double)L.alpha * (L.gate ? (double)L.gate[(size_t)(m / L.gate_every) * L.H + i] : 1.0) * z[i];
        }
        for (int i = 0; L.h_out && i < L.H; i++) {
            if (L.f32) static_cast<float *>(L.h_out)[row + i] = (float)h[i];
            else static_cast<_Float16 *>(L.h_out)[row + i] = (_Float16)h[i];
        }
        norm(h, L.w_pre, L.eps_pre);
        for (int i = 0; i < L.H; i++) {
            x[i] = (float)h[i];
            if (L.x) L.x[row + i] = (_Float16)h[i];
        }
        for (int b = 0; L.xq && b < nb; b++)
            quantise(x.data() + b * kF8Block, std::min(kF8Block, L.H - b * kF8Block), L.xq + row + b * kF8Block, L.x_scale + (size_t)m * nb + b);
    }
    return true;
}

bool moe_route_ref(const Route &L)
{
    struct Key { double key, group, p; };
    std::vector<Key> s;
    std::vector<double> value;
    std::vector<int> next;
    try {
        s.resize(L.E);
        value.resize(L.n_group);
        next.resize((size_t)L.E + 1);
    } catch (const std::bad_alloc &) {
        return false;
    }
    const auto rank = [](double v) { return v == v ? std::min(std::max(v, -1e300), 1e300) : -4e300; };   // (two -1e300 are a run's)
    const int run = L.E / L.n_group;
    for (int m = 0; m < L.M; m++) {
        int32_t *ids = L.ids + (size_t)m * L.top_k;
        float *weight = L.weight + (size_t)m * L.top_k;
        std::fill(ids, ids + L.top_k, -1);
        std::fill(weight, weight + L.top_k, 0.f);
        if (L.active && !L.active[m]) continue;
        double most = -INFINITY, sum = 0.0;
        for (int e = 0; e < L.E; e++) {
            const float v = at(L.logits, L.f32, (size_t)m * L.rs + e);
            s[e].key = (double)(v > 3.402823466e38f ? 3.402823466e38f : v);
            most = fmax(most, s[e].key);
        }
        if (most == -INFINITY) most = 0.0;
        for (Key &k : s) {
            k.p = L.sigmoid ? 1.0 / (1.0 + exp(-k.key)) : exp(k.key - most);
            sum += k.p;
        }
        for (int e = 0; e < L.E; e++) {
            Key &k = s[e];
            if (!L.sigmoid) k.p /= sum;
            const double c = L.bias ? k.p + (double)L.bias[e] : k.p;
            const bool can = k.key != -INFINITY;
            k.key = can ? rank(L.bias ? c : k.key) : -INFINITY;
            k.group = can ? rank(c) : -INFINITY;
        }
        if (L.n_group > 1) {
            for (int g = 0; g < L.n_group; g++) {
                double first = -INFINITY, second = -INFINITY;
                for (int e = g * run; e < (g + 1) * run; e++) {
                    const double k = s[e].group;
                    if (k > first) second = first, first = k;
                    else if (k > second) second = k;
                }
                value[g] = L.group_best == 2 && second > -INFINITY ? first + second : first;
            }
            uint64_t in = 0;
            for (int i = 0; i < L.top_group; i++) {
                const int g = (int)(std::max_element(value.begin(), value.end()) - value.begin());
                if (value[g] == -INFINITY) break;
                in |= (uint64_t)1 << g;
                value[g] = -INFINITY;
            }
            for (int e = 0; e < L.E; e++)
                if (!((in >> (e / run)) & 1)) s[e].key = -INFINITY;
        }
        double chosen = 0.0, p[kMaxTop];
        int n = 0;
        for (; n < L.top_k; n++) {
            const auto best = std::max_element(s.begin(), s.end(), [](const Key &a, const Key &b) { return a.key < b.key; });
            if (best->key == -INFINITY) break;
            ids[n] = (int32_t)(best - s.begin());
            p[n] = best->p;
            chosen += best->p;
            best->key = -INFINITY;
        }
        for (int j = 0; j < n; j++) weight[j] = (float)((L.renorm ? (chosen == 0.0 ? 0.0 : p[j] / chosen) : p[j]) * (double)L.scale);
    }
    if (!L.off) return true;
    const size_t total = (size_t)L.M * L.top_k;
    for (size_t i = 0; i < total; i++)
        if (L.ids[i] >= 0) next[L.ids[i] + 1]++;
    for (int e = 0; e < L.E; e++) next[e + 1] += next[e];
    std::copy(next.begin(), next.end(), L.off);
    for (size_t i = 0; i < total; i++) {
        const int id = L.ids[i];
        L.slot[i] = id < 0 ? -1 : next[id]++;
        if (id >= 0) L.src[L.slot[i]] = (int32_t)(i / L.top_k);
    }
    return true;
}

}  // namespace rk
