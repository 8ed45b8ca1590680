// rope.hip — norms of the query and key heads and their rotation, one pass over the rows.
//
// A head is G lanes (a power of two, eight values a lane), a wave 64 / G heads. A lane holds whole
// pairs: values [4 l, 4 l + 4) of both halves of the rotated part (HALVES) or eight neighbours
// (PAIRS), and behind the rotated part eight neighbours that pass. So a head is read once, its square sum
// is a shuffle over G lanes, and the rotation stays in registers. The angle is reduced in fp64 to a
// quarter turn around a multiple of one (a position of 10^6 times a frequency of 1 keeps 33 bits of
// the fraction), where the series of sine and cosine are within 2^-22.
//
// Memory bounds it: 4096 fp32 rows of 40 heads of 128 (126 MB read and written) 21.9 us by trace, 5.7 TB/s, as a
// large copy moves; one token of 16 sequences, 24 heads of 256, is a launch: 3.3 us.
#include "serve.h"

#include <algorithm>

namespace rk {
namespace {

typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

struct RopeArgs {
    const void *q, *k;
    long q_rs, k_rs;
    const _Float16 *wq, *wk;
    const float *inv_freq;
    const int32_t *pos;
    _Float16 *q_out, *k_out;
    int rows, n_tokens, n_head, n_kv, dim, rot;
    float eps, rdim;
    int norm, step;   // step: heads of a row that the grid takes at once
};

__device__ __forceinline__ f32x4 load4(const _Float16 *p)
{
    const f16x4 v = *reinterpret_cast<const f16x4 *>(p);
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
__device__ __forceinline__ f32x4 load4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
__device__ __forceinline__ void store4(_Float16 *p, f32x4 v)
{
    *reinterpret_cast<f16x4 *>(p) = f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

// Sine and cosine of `t` turns: the nearest quarter turn taken off in fp64, then Taylor's series on
// [-pi/4, pi/4] (the first terms left out: 2e-9 and 2e-9), and the quadrant's swap and signs.
__device__ __forceinline__ void sincos_turns(double t, float &s, float &c)
{
    const double k = rint(4.0 * t);
    const float r = (float)((t - 0.25 * k) * 6.283185307179586477), r2 = r * r;
    const int q = (int)(k - 4.0 * floor(0.25 * k));   // 0 .. 3
    const float sn = r + r * r2 * (-1.f / 6 + r2 * (1.f / 120 + r2 * (-1.f / 5040 + r2 * (1.f / 362880))));
    const float cn = 1.f + r2 * (-0.5f + r2 * (1.f / 24 + r2 * (-1.f / 720 + r2 * (1.f / 40320 + r2 * (-1.f / 3628800)))));
    s = q & 1 ? cn : sn;
    c = q & 1 ? sn : cn;
    if (q & 2) s = -s;
    if (q == 1 || q == 2) c = -c;
}

template <typename T, int G, bool PAIRS> __global__ __launch_bounds__(256) void k_qk_norm_rope(const RopeArgs a)
{
    const int row = blockIdx.x, tid = threadIdx.x, l = tid % G;
    const int heads = a.n_head + a.n_kv, half = a.rot / 2;
    // the lane's two runs of four values
    const bool turns = 8 * l < a.rot, in = 8 * l < a.dim;
    const int d0 = !in ? 0 : !PAIRS && turns ? 4 * l : 8 * l, d1 = !in ? 0 : !PAIRS && turns ? half + 4 * l : 8 * l + 4;
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; i++) cs[i] = 1.f, sn[i] = 0.f;
    if (turns) {
        const double p = (double)a.pos[row] * 0.15915494309189533577;   // 1 / (2 pi)
        const f32x4 f = *reinterpret_cast<const f32x4 *>(a.inv_freq + 4 * l);
#pragma unroll
        for (int i = 0; i < 4; i++) sincos_turns(p * (double)f[i], sn[i], cs[i]);
    }
    const int s = row / a.n_tokens, t = row - s * a.n_tokens;
    for (int h = blockIdx.y * (256 / G) + tid / G; h < heads; h += a.step) {
        const bool key = h >= a.n_head;
        const int hh = key ? h - a.n_head : h;
        const T *x = key ? static_cast<const T *>(a.k) + (size_t)row * a.k_rs : static_cast<const T *>(a.q) + (size_t)row * a.q_rs;
        x += (size_t)hh * a.dim;
        f32x4 u = {0.f, 0.f, 0.f, 0.f}, v = u;
        if (in) {
            u = load4(x + d0);
            v = load4(x + d1);
        }
        if (a.norm) {
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) sq += u[i] * u[i] + v[i] * v[i];
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
            const float r = 1.f / sqrtf(sq * a.rdim + a.eps);
            const _Float16 *w = key ? a.wk : a.wq;
            f32x4 wu = {1.f, 1.f, 1.f, 1.f}, wv = wu;
            if (w) {
                wu = load4(w + d0);
                wv = load4(w + d1);
            }
            u *= r * wu;
            v *= r * wv;
        }
        if constexpr (PAIRS) {
            const f32x4 x0 = u, x1 = v;
            u = f32x4{x0[0] * cs[0] - x0[1] * sn[0], x0[1] * cs[0] + x0[0] * sn[0], x0[2] * cs[1] - x0[3] * sn[1], x0[3] * cs[1] + x0[2] * sn[1]};
            v = f32x4{x1[0] * cs[2] - x1[1] * sn[2], x1[1] * cs[2] + x1[0] * sn[2], x1[2] * cs[3] - x1[3] * sn[3], x1[3] * cs[3] + x1[2] * sn[3]};
        } else {
            const f32x4 x0 = u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u[i] = x0[i] * cs[i] - v[i] * sn[i];
                v[i] = v[i] * cs[i] + x0[i] * sn[i];
            }
        }
        if (in) {
            _Float16 *o = key ? a.k_out : a.q_out;
            o += (((size_t)s * (key ? a.n_kv : a.n_head) + hh) * a.n_tokens + t) * a.dim;
            store4(o + d0, u);
            store4(o + d1, v);
        }
    }
}

template <typename T, int G> hipError_t launch(const RopeArgs &a, bool pairs, dim3 grid, hipStream_t s)
{
    if (pairs) hipLaunchKernelGGL((k_qk_norm_rope<T, G, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_qk_norm_rope<T, G, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}
template <typename T> hipError_t launch(const RopeArgs &a, bool pairs, int g, dim3 grid, hipStream_t s)
{
    switch (g) {
    case 4: return launch<T, 4>(a, pairs, grid, s);
    case 8: return launch<T, 8>(a, pairs, grid, s);
    case 16: return launch<T, 16>(a, pairs, grid, s);
    default: return launch<T, 32>(a, pairs, grid, s);
    }
}

}  // namespace

hipError_t qk_norm_rope(const RopeLaunch &L, hipStream_t s, uint64_t *blocks)
{
    int g = 4;
    while (8 * g < L.dim) g *= 2;
    RopeArgs a;
    a.q = L.q; a.k = L.k; a.q_rs = L.q_rs; a.k_rs = L.k_rs; a.wq = L.wq; a.wk = L.wk; a.inv_freq = L.inv_freq; a.pos = L.pos;
    a.q_out = L.q_out; a.k_out = L.k_out; a.rows = L.n_seq * L.n_tokens; a.n_tokens = L.n_tokens; a.n_head = L.n_head; a.n_kv = L.n_kv;
    a.dim = L.dim; a.rot = L.rot; a.eps = L.eps; a.rdim = 1.f / (float)L.dim; a.norm = L.norm;
    // Workgroups of a row: as many as its heads fill, but no more than make about four a CU (1024): with more rows a
    // lane takes several heads with one sine and cosine (4096 rows of 40 heads of 128: 27.0 us for three workgroups a
    // row, 22.8 for one; 512 such rows 5.5 for three, 5.1 for two, 5.6 for one; 16 rows of 24 heads of 256 3.7 for three,
    // 4.7 for one).
    const int per = 256 / g, most = (L.n_head + L.n_kv + per - 1) / per, y = std::max(1, std::min(most, (1024 + a.rows - 1) / a.rows));
    a.step = y * per;
    const dim3 grid((unsigned)a.rows, (unsigned)y);
    *blocks = (uint64_t)a.rows * y;
    return L.f32 ? launch<float>(a, L.pairs, g, grid, s) : launch<_Float16>(a, L.pairs, g, grid, s);
}

}  // namespace rk
