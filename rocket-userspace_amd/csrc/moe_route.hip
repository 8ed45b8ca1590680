// moe_route.hip — which experts a token goes to, and the rows sorted by expert.
//
// Scores are fp64, so that rounding changes no choice but one between choices within 2^-42 of each other: a key is an unsigned
// 64-bit number of the choice's order whose last ten bits are the expert's, the first one's the largest. What bounds it is the
// number of instructions a token: up to 256 experts a token is a row of 16 lanes, each with up to 16 neighbouring experts, four
// tokens a wave, whose reductions stay in registers (DPP rotations within a row); more experts are a wave a token, where a lane
// sorts its keys once and moves on where it has won. The sort by expert needs no order of atomics: a workgroup's tokens set their
// bit in one mask an expert, and a choice's place among them is the count of bits below its own. Few tokens are one workgroup and
// one launch; more write their counts, which a second launch turns into starts and a third into rows. 16 tokens of 64 experts take
// 5.4 us, 8192 tokens of 256 with groups and a bias 24.3: 14 the scores and choices, 4.6 and 4.0 the sort.
#include "layer.h"

#include <algorithm>
#include <atomic>

#include "lds_optin.h"

namespace rk {
namespace {

struct RArgs {
    const void *logits;
    long rs;
    const float *bias;
    const uint8_t *active;
    int M, E, n_group, run, lanes, run_magic, vec, group_best, top_group, top_k, renorm, sigmoid, f32, plan;
    float scale;
    int32_t *ids, *off, *src, *slot, *counts;
    float *weight;
};

constexpr int kTokens = 32;   // of a workgroup, where there are several
constexpr int kOne = 32;      // up to so many tokens are one workgroup

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The largest of the lanes' v, in every lane: rows of 16 by rotation, then the rows' last lanes onwards.
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#if defined(__HIP_DEVICE_COMPILE__)
#define RK_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, ctrl, rows, 0xf, false))
    RK_DPP_MAX(0x121, 0xf);   // row_ror:1
    RK_DPP_MAX(0x122, 0xf);   // row_ror:2
    RK_DPP_MAX(0x124, 0xf);   // row_ror:4
    RK_DPP_MAX(0x128, 0xf);   // row_ror:8
    RK_DPP_MAX(0x142, 0xa);   // row_bcast:15
    RK_DPP_MAX(0x143, 0xc);   // row_bcast:31
#undef RK_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
#else
    return v;
#endif
}

// A key of the order of finite numbers, above 0; 0 stands for what is no candidate.
__device__ __forceinline__ uint64_t ordered(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);   // (-0 and 0 are one)
    return b >> 63 ? ~b : b | (uint64_t)1 << 63;
}
__device__ __forceinline__ double ranked(double v) { return v == v ? fmin(fmax(v, -1e300), 1e300) : -4e300; }   // (two -1e300 are a run's)

// The largest of keys that differ where they are not 0 (0: all are), in every lane.
__device__ __forceinline__ uint64_t wave_best(uint64_t key)
{
    const uint32_t hi = (uint32_t)(key >> 32), top = wave_max(hi);
    const uint64_t m = __ballot(hi == top);
    const uint32_t low = m & (m - 1) ? wave_max(hi == top ? (uint32_t)key : 0u) : (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, __builtin_ctzll(m));
    return (uint64_t)top << 32 | low;
}

// e^x by Taylor's series of 2^-k e^x around 0 (|r| <= 0.35: 0.35^14 / 14! = 5e-18 left out), within two steps of fp64; r by Cody and
// Waite's reduction, ln 2 in two parts of which the first has 32 bits, so that k times it is exact.
__device__ __forceinline__ double exp64(double x)
{
#if defined(__HIP_DEVICE_COMPILE__)
    x = x == x ? fmin(fmax(x, -2000.0), 2000.0) : x;
    const double k = rint(x * 1.4426950408889634074);
    double r = fma(k, -6.93147180369123816490e-01, x);
    r = fma(k, -1.90821492927058770002e-10, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)k);
#else
    return x;
#endif
}
// 1 / d of 1 <= d <= 2^11, by two steps of Newton's method.
__device__ __forceinline__ double inverse(double d)
{
#if defined(__HIP_DEVICE_COMPILE__)
    double r = __builtin_amdgcn_rcp(d);
    r = fma(fma(-d, r, 1.0), r, r);
    return fma(fma(-d, r, 1.0), r, r);
#else
    return d;
#endif
}
__device__ __forceinline__ double sigmoid(double x)
{
    const double e = exp64(-fabs(x)), r = inverse(1.0 + e);
    return x < 0.0 ? e * r : r;   // (a NaN: r, which is one)
}

__device__ __forceinline__ float logit(const RArgs &a, int m, int e)
{
    const size_t i = (size_t)m * a.rs + e;
    const float v = a.f32 ? static_cast<const float *>(a.logits)[i] : (float)static_cast<const _Float16 *>(a.logits)[i];
    return v > 3.402823466e38f ? 3.402823466e38f : v;
}

// Falling order, by exchanges of neighbours at a distance (odd-even merges).
template <int N> __device__ __forceinline__ void sort(uint64_t (&k)[N])
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int d = p; d >= 1; d /= 2)
#pragma unroll
            for (int j = d % p; j + d < N; j += 2 * d)
#pragma unroll
                for (int i = 0; i < d; i++)
                    if (i + j + d < N && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
                        const uint64_t x = k[i + j], y = k[i + j + d];
                        k[i + j] = x > y ? x : y;
                        k[i + j + d] = x > y ? y : x;
                    }
}

// Token m's experts: lane j < top_k gets the j-th one's id (-1: none) and weight. `keys`: E doubles of LDS (groups).
template <int NE> __device__ void route_token(const RArgs &a, int m, double *keys, int &id, float &weight)
{
    const int lane = threadIdx.x & 63;
    id = -1;
    weight = 0.f;
    if (a.active && !a.active[m]) return;
    float f[NE];
    uint64_t key[NE];
#pragma unroll
    for (int i = 0; i < NE; i++) f[i] = lane + 64 * i < a.E ? logit(a, m, lane + 64 * i) : -INFINITY;
    const bool scores = a.bias || a.n_group > 1;   // (without either the logits' order is the scores', who are summed alone)
    double p[NE], most = 0.0, scale = 1.0;
    if (!a.sigmoid) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NE; i++) top = fmaxf(top, f[i]);   // (passes over a NaN)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        most = top == -INFINITY ? 0.0 : (double)top;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NE; i++) {
            p[i] = exp64((double)f[i] - most);
            sum += p[i];
        }
        sum = wave_sum(sum);
        scale = sum > 0.0 || sum != sum ? inverse(sum) : 0.0;
    } else if (scores) {
#pragma unroll
        for (int i = 0; i < NE; i++) p[i] = sigmoid((double)f[i]);
    }
    // the keys: choices, or logits where no bias changes the order; behind every number a NaN, and behind that what is no candidate
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int e = lane + 64 * i;
        const bool can = f[i] != -INFINITY;   // (not one past the last)
        double c = (double)f[i];
        if (scores) {
            const double s = a.sigmoid ? p[i] : p[i] * scale, choice = a.bias && e < a.E ? s + (double)a.bias[e] : s;
            if (a.n_group > 1 && e < a.E) keys[e] = can ? ranked(choice) : -INFINITY;
            if (a.bias) c = choice;
        }
        key[i] = can ? (ordered(ranked(c)) & ~(uint64_t)1023) | (uint64_t)(1023 - e) : 0;
    }
    if (a.n_group > 1) {
        // A run is `lanes` lanes, whose two largest are merged. (One wave's own part of LDS: its writes are seen by its later reads.)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int g = lane / a.lanes;
        double first = -INFINITY, second = -INFINITY;
        if (g < a.n_group)
            for (int j = lane % a.lanes; j < a.run; j += a.lanes) {
                const double k = keys[g * a.run + j];
                second = fmax(second, fmin(first, k));
                first = fmax(first, k);
            }
        for (int o = 1; o < a.lanes; o *= 2) {
            const double x = __shfl_xor(first, o, 64), y = __shfl_xor(second, o, 64);
            second = fmax(fmax(second, y), fmin(first, x));
            first = fmax(first, x);
        }
        const double value = a.group_best == 2 && second > -INFINITY ? first + second : first;
        uint64_t k = g < a.n_group && lane % a.lanes == 0 && value > -INFINITY ? (ordered(value) & ~(uint64_t)1023) | (uint64_t)(1023 - g) : 0, in = 0;
        for (int i = 0; i < a.top_group; i++) {
            const uint64_t best = wave_best(k);
            if (!best) break;
            in |= (uint64_t)1 << (1023 - (int)(best & 1023));
            if (k == best) k = 0;
        }
#pragma unroll
        for (int i = 0; i < NE; i++)
            if (!((in >> (((uint32_t)(lane + 64 * i) * (uint32_t)a.run_magic >> 22) & 63)) & 1)) key[i] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    sort(key);
    for (int j = 0; j < a.top_k; j++) {
        const uint64_t best = wave_best(key[0]);
        if (!best) break;
        if (lane == j) id = 1023 - (int)(best & 1023);
        const bool won = key[0] == best;
#pragma unroll
        for (int i = 0; i < NE; i++) key[i] = won ? (i + 1 < NE ? key[i + 1] : 0) : key[i];
    }
    double w = 0.0;
    if (id >= 0) {
        const double x = (double)logit(a, m, id);
        w = a.sigmoid ? sigmoid(x) : exp64(x - most) * scale;
    }
    if (a.renorm) {
        const double sum = wave_sum(w);
        w = sum == 0.0 ? 0.0 : w / sum;
    }
    weight = id < 0 ? 0.f : (float)(w * (double)a.scale);
}

// Rotations within a row of 16 lanes.
template <int N> __device__ __forceinline__ uint32_t row_ror(uint32_t v)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true);
#else
    return v;
#endif
}
template <int N> __device__ __forceinline__ double row_ror(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)row_ror<N>((uint32_t)(b >> 32)) << 32 | row_ror<N>((uint32_t)b)));
}
__device__ __forceinline__ double row_sum(double v)   // (a rotation by 8, 4, 2, 1: every lane adds the same pairs)
{
    v += row_ror<8>(v);
    v += row_ror<4>(v);
    v += row_ror<2>(v);
    return v + row_ror<1>(v);
}
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    v = max(v, row_ror<8>(v));
    v = max(v, row_ror<4>(v));
    v = max(v, row_ror<2>(v));
    return max(v, row_ror<1>(v));
}
__device__ __forceinline__ uint64_t row_best(uint64_t key)
{
    const uint32_t hi = (uint32_t)(key >> 32), top = row_max(hi);
    return (uint64_t)top << 32 | row_max(hi == top ? (uint32_t)key : 0u);
}

// Token m's experts by a row of 16 lanes: lane l gets the choices l and 16 + l. `keys`: E doubles of LDS (groups).
template <int NE> __device__ void route_row(const RArgs &a, int m, double *keys, int (&id)[2], float (&weight)[2])
{
    const int l = threadIdx.x & 15, e0 = NE * l;
    id[0] = id[1] = -1;
    weight[0] = weight[1] = 0.f;
    if (a.active && !a.active[m]) return;   // (whole rows: the reductions stay within them)
    float f[NE];
    bool loaded = false;
    if constexpr (NE % 4 == 0) {
        if (a.vec) {   // (E and the rows' starts are multiples of four)
            loaded = true;
#pragma unroll
            for (int i = 0; i < NE; i += 4) {
                float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (e0 + i < a.E) {
                    const size_t at = (size_t)m * a.rs + e0 + i;
                    if (a.f32) {
                        const float4 x = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.logits) + at);
                        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
                    } else {
                        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                        const h4 x = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.logits) + at);
#pragma unroll
                        for (int c = 0; c < 4; c++) v[c] = (float)x[c];
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) f[i + c] = v[c] > 3.402823466e38f ? 3.402823466e38f : v[c];
            }
        }
    }
    if (!loaded) {
#pragma unroll
        for (int i = 0; i < NE; i++) f[i] = e0 + i < a.E ? logit(a, m, e0 + i) : -INFINITY;
    }
    const bool scores = a.bias || a.n_group > 1;   // (without either the logits' order is the scores', who are summed alone)
    double p[NE], most = 0.0, scale = 1.0;
    if (!a.sigmoid) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NE; i++) top = fmaxf(top, f[i]);   // (passes over a NaN)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        most = top == -INFINITY ? 0.0 : (double)top;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NE; i++) {
            p[i] = exp64((double)f[i] - most);
            sum += p[i];
        }
        sum = row_sum(sum);
        scale = sum > 0.0 || sum != sum ? inverse(sum) : 0.0;
    } else if (scores) {
#pragma unroll
        for (int i = 0; i < NE; i++) p[i] = sigmoid((double)f[i]);
    }
    uint64_t key[NE];
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int e = e0 + i;
        const bool can = f[i] != -INFINITY;   // (not one past the last)
        double c = (double)f[i];
        if (scores) {
            const double s = a.sigmoid ? p[i] : p[i] * scale, choice = a.bias && e < a.E ? s + (double)a.bias[e] : s;
            if (a.n_group > 1 && e < a.E) keys[e] = can ? ranked(choice) : -INFINITY;
            if (a.bias) c = choice;
        }
        key[i] = can ? (ordered(ranked(c)) & ~(uint64_t)1023) | (uint64_t)(1023 - e) : 0;
    }
    if (a.n_group > 1) {
        // A run is `lanes` lanes, whose two largest are merged, or a lane has several. (A row's own part of LDS: its wave's writes
        // are seen by its later reads.)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint64_t value[4] = {0, 0, 0, 0}, in = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int g = l / a.lanes + 16 / a.lanes * u;
            if (u && 16 * u >= a.n_group) continue;   // (several only where `lanes` is 1)
            double first = -INFINITY, second = -INFINITY;
            if (g < a.n_group)
                for (int j = l % a.lanes; j < a.run; j += a.lanes) {
                    const double k = keys[g * a.run + j];
                    second = fmax(second, fmin(first, k));
                    first = fmax(first, k);
                }
            for (int o = 1; o < a.lanes; o *= 2) {
                const double x = __shfl_xor(first, o, 64), y = __shfl_xor(second, o, 64);
                second = fmax(fmax(second, y), fmin(first, x));
                first = fmax(first, x);
            }
            const double v = a.group_best == 2 && second > -INFINITY ? first + second : first;
            if (g < a.n_group && v > -INFINITY) value[u] = (ordered(v) & ~(uint64_t)1023) | (uint64_t)(1023 - g);
        }
        for (int i = 0; i < a.top_group; i++) {
            uint64_t k = value[0];
#pragma unroll
            for (int u = 1; u < 4; u++) k = value[u] > k ? value[u] : k;
            const uint64_t best = row_best(k);
            if (best) in |= (uint64_t)1 << (1023 - (int)(best & 1023));
#pragma unroll
            for (int u = 0; u < 4; u++) value[u] = value[u] == best ? 0 : value[u];
        }
#pragma unroll
        for (int i = 0; i < NE; i++)
            if (!((in >> (((uint32_t)(e0 + i) * (uint32_t)a.run_magic >> 22) & 63)) & 1)) key[i] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    for (int j = 0; j < a.top_k; j++) {
        uint64_t k = key[0];
#pragma unroll
        for (int i = 1; i < NE; i++) k = key[i] > k ? key[i] : k;
        const uint64_t best = row_best(k);
        if (best && l == (j & 15)) id[j >> 4] = 1023 - (int)(best & 1023);
#pragma unroll
        for (int i = 0; i < NE; i++) key[i] = key[i] == best ? 0 : key[i];
    }
    double w[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        w[u] = 0.0;
        if (id[u] >= 0) {
            const double x = (double)logit(a, m, id[u]);
            w[u] = a.sigmoid ? sigmoid(x) : exp64(x - most) * scale;
        }
    }
    if (a.renorm) {
        const double sum = row_sum(w[0] + w[1]);
#pragma unroll
        for (int u = 0; u < 2; u++) w[u] = sum == 0.0 ? 0.0 : w[u] / sum;
    }
#pragma unroll
    for (int u = 0; u < 2; u++) weight[u] = id[u] < 0 ? 0.f : (float)(w[u] * (double)a.scale);
}

// Exclusive sums of v over the workgroup's threads, and the sum of all. `part`: a word a wave.
__device__ __forceinline__ int group_scan(int v, int *part, int &all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (blockDim.x + 63) / 64;
    int upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(upto, o, 64);
        if (lane >= o) upto += u;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < waves; w++) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    __syncthreads();
    return before + upto - v;
}

// Lanes of a token, experts of a lane. Waves of a workgroup: eight where the registers of sixteen do not hold a lane's keys.
template <int L_, int NE_> struct Form {
    static constexpr int L = L_, NE = NE_, WAVES = L == 16 || NE == 16 ? 8 : 16, E = L * NE;
};

// A workgroup's tokens. ONE: all tokens (up to kOne), with the plan; otherwise kTokens of them, and their counts.
template <class F, bool ONE> __global__ __launch_bounds__(64 * F::WAVES) void k_route(const RArgs a)
{
    constexpr int T = ONE ? kOne : kTokens;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int part[16], start[ONE ? F::E : 1], chosen[ONE ? T * kMaxTop : 1];
    __shared__ unsigned mask[F::E];
    const int l = threadIdx.x % F::L, row = threadIdx.x / F::L, rows = blockDim.x / F::L, t0 = blockIdx.x * T;
    double *const keys = reinterpret_cast<double *>(smem) + (size_t)row * a.E;
    if (a.plan) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) mask[e] = 0;
        __syncthreads();
    }
    for (int t = row; t < T && t0 + t < a.M; t += rows) {
        const int m = t0 + t;
        int id[2];
        float w[2];
        if constexpr (F::L == 16) route_row<F::NE>(a, m, keys, id, w);
        else route_token<F::NE>(a, m, keys, id[0], w[0]);
#pragma unroll
        for (int u = 0; u < (F::L == 16 ? 2 : 1); u++) {
            const int j = l + 16 * u;
            if (j < a.top_k) {
                a.ids[(size_t)m * a.top_k + j] = id[u];
                a.weight[(size_t)m * a.top_k + j] = w[u];
                if (ONE) chosen[t * a.top_k + j] = id[u];
                if (a.plan && id[u] >= 0) atomicOr(&mask[id[u]], 1u << t);
            }
        }
    }
    if (!a.plan) return;
    __syncthreads();
    if constexpr (!ONE) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) a.counts[(size_t)blockIdx.x * a.E + e] = __popc(mask[e]);
    } else {
        const int per = (a.E + blockDim.x - 1) / blockDim.x, e0 = threadIdx.x * per, e1 = min(a.E, e0 + per);   // experts a thread, neighbours
        int n = 0;
        for (int e = e0; e < e1; e++) n += __popc(mask[e]);
        int all;
        int at = group_scan(n, part, all);
        for (int e = e0; e < e1; e++) {
            start[e] = at;
            a.off[e] = at;
            at += __popc(mask[e]);
        }
        if (threadIdx.x == 0) a.off[a.E] = all;
        __syncthreads();
        for (int i = threadIdx.x; i < a.M * a.top_k; i += blockDim.x) {
            const int t = i / a.top_k, id = chosen[i];
            int r = -1;
            if (id >= 0) {
                r = start[id] + __popc(mask[id] & ((1u << t) - 1u));
                a.src[r] = t;
            }
            a.slot[i] = r;
        }
    }
}

// The workgroups' counts of an expert to its rows' starts from its first, in place, and their sum behind all counts. A workgroup
// has 16 experts, 64 threads an expert's column.
__global__ __launch_bounds__(1024) void k_starts(const RArgs a, int nblk)
{
    __shared__ int sums[64][17];
    const int c = threadIdx.x % 16, e = blockIdx.x * 16 + c, s = threadIdx.x / 16, per = (nblk + 63) / 64;
    const int b0 = min(nblk, s * per), b1 = min(nblk, b0 + per);
    const bool in = e < a.E;
    int n = 0;
    if (in) {
#pragma unroll 4
        for (int b = b0; b < b1; b++) n += a.counts[(size_t)b * a.E + e];
    }
    sums[s][c] = n;
    __syncthreads();
    // the parts before: thread (lane, column) of the first 16 waves scans column `wave` over its 64 lanes
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int upto = sums[lane][w];
    const int own = upto;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(upto, o, 64);
        if (lane >= o) upto += u;
    }
    __syncthreads();
    sums[lane][w] = upto - own;
    if (lane == 63 && (int)blockIdx.x * 16 + w < a.E) a.counts[(size_t)nblk * a.E + blockIdx.x * 16 + w] = upto;
    __syncthreads();
    if (in) {
        int f = sums[s][c];
#pragma unroll 4
        for (int b = b0; b < b1; b++) {
            const size_t i = (size_t)b * a.E + e;
            const int x = a.counts[i];
            a.counts[i] = f;
            f += x;
        }
    }
}

// Rows of a workgroup's tokens; the first writes the experts' offsets. `per`: experts a thread, neighbours.
__global__ __launch_bounds__(256) void k_rows(const RArgs a, int nblk)
{
    __shared__ int part[16], start[kMaxExperts];
    __shared__ unsigned mask[kMaxExperts];
    const int per = (a.E + 255) / 256, e0 = threadIdx.x * per, e1 = min(a.E, e0 + per);
    const int *const totals = a.counts + (size_t)nblk * a.E;
    int sum = 0;
    for (int e = e0; e < e1; e++) {
        mask[e] = 0;
        sum += totals[e];
    }
    int all;
    int at = group_scan(sum, part, all);   // (a barrier behind the masks)
    const int *const mine = a.counts + (size_t)blockIdx.x * a.E;
    for (int e = e0; e < e1; e++) {
        if (blockIdx.x == 0) a.off[e] = at;
        start[e] = at + mine[e];
        at += totals[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.off[a.E] = all;
    const int t0 = blockIdx.x * kTokens, n = min(kTokens, a.M - t0) * a.top_k;
    const size_t i0 = (size_t)t0 * a.top_k;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int id = a.ids[i0 + i];
        if (id >= 0) atomicOr(&mask[id], 1u << (i / a.top_k));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int id = a.ids[i0 + i], t = i / a.top_k;
        int r = -1;
        if (id >= 0) {
            r = start[id] + __popc(mask[id] & ((1u << t) - 1u));
            a.src[r] = t0 + t;
        }
        a.slot[i0 + i] = r;
    }
}

template <class F> hipError_t launch(const RArgs &a, hipStream_t s, uint64_t *blocks)
{
    static std::atomic<uint64_t> opt1{0}, opt2{0};
    // One workgroup of as many waves as the tokens fill, or several.
    const bool one = a.M <= kOne;
    const int nblk = one ? 1 : (a.M + kTokens - 1) / kTokens, all = (one ? a.M : kTokens) * F::L, waves = std::min(F::WAVES, (all + 63) / 64);
    const int row = a.n_group > 1 ? a.E * (int)sizeof(double) : 0, lds = waves * (64 / F::L) * row, most = F::WAVES * (64 / F::L) * F::E * (int)sizeof(double);
    if (one) {
        if (hipError_t e = lds_opt_in(reinterpret_cast<const void *>(&k_route<F, true>), std::min(most, 140 << 10), opt1)) return e;
        hipLaunchKernelGGL((k_route<F, true>), dim3(1), dim3(64 * waves), lds, s, a);
    } else {
        if (hipError_t e = lds_opt_in(reinterpret_cast<const void *>(&k_route<F, false>), std::min(most, 140 << 10), opt2)) return e;
        hipLaunchKernelGGL((k_route<F, false>), dim3((unsigned)nblk), dim3(64 * waves), lds, s, a);
    }
    *blocks = (uint64_t)nblk;
    if (one || !a.plan) return hipGetLastError();
    if (hipError_t e = hipGetLastError()) return e;
    const int columns = (a.E + 15) / 16;
    hipLaunchKernelGGL(k_starts, dim3((unsigned)columns), dim3(1024), 0, s, a, nblk);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(k_rows, dim3((unsigned)nblk), dim3(256), 0, s, a, nblk);
    *blocks += (uint64_t)nblk + columns;
    return hipGetLastError();
}

}  // namespace

size_t route_ws(const Route &L) { return L.off && L.M > kOne ? (size_t)((L.M + kTokens - 1) / kTokens + 1) * L.E * sizeof(int32_t) : 0; }

hipError_t moe_route(const Route &L, hipStream_t s, uint64_t *blocks)
{
    RArgs a;
    a.logits = L.logits; a.rs = L.rs; a.bias = L.bias; a.active = L.active; a.M = L.M; a.E = L.E; a.n_group = L.n_group; a.run = L.E / L.n_group;
    // A row of 16 lanes a token where that is few experts a lane, or many tokens, whose instructions count: 8192 tokens of 256
    // experts 24.3 us, by a wave a token 28.4; of few tokens a wave's lanes have less to do in a row: 16 tokens 12.8 us, by rows 14.4.
    const bool wide = L.E > 256 || (L.E > 64 && L.M <= 16);
    const int lanes = wide ? 64 : 16;
    a.lanes = 1;
    while (2 * a.lanes * L.n_group <= lanes) a.lanes *= 2;
    a.run_magic = ((1 << 22) + a.run - 1) / a.run;   // e / run = e * run_magic >> 22: exact for e < 1024
    a.vec = L.E % 4 == 0 && L.rs % 4 == 0 && ((uintptr_t)L.logits & (L.f32 ? 15 : 7)) == 0;
    a.group_best = L.group_best; a.top_group = L.top_group; a.top_k = L.top_k; a.renorm = L.renorm; a.sigmoid = L.sigmoid; a.f32 = L.f32;
    a.plan = L.off != nullptr; a.scale = L.scale; a.ids = L.ids; a.off = L.off; a.src = L.src; a.slot = L.slot; a.counts = L.counts; a.weight = L.weight;
    if (wide) {
        if (L.E <= 256) return launch<Form<64, 4>>(a, s, blocks);
        return L.E <= 512 ? launch<Form<64, 8>>(a, s, blocks) : launch<Form<64, 16>>(a, s, blocks);
    }
    if (L.E <= 16) return launch<Form<16, 1>>(a, s, blocks);
    if (L.E <= 64) return launch<Form<16, 4>>(a, s, blocks);
    return L.E <= 128 ? launch<Form<16, 8>>(a, s, blocks) : launch<Form<16, 16>>(a, s, blocks);
}

}  // namespace rk
