// moe_route.hip — which experts a token goes to, and the rows sorted by expert.
//
// A wave is a token, a lane every 64th expert; scores are fp64, so that rounding changes no choice. top_k rounds take
// the wave's largest key. The sort needs no order of atomics: a workgroup's tokens set their bit in one mask an expert, and a
// choice's place among them is the count of bits below its own. Up to 64 tokens are one workgroup and one launch; more write
// their counts, which a second launch turns into starts and a third into rows.
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
    int M, E, n_group, run, group_best, top_group, top_k, renorm, sigmoid, f32, plan;
    float scale;
    int32_t *ids, *off, *src, *slot, *counts;
    float *weight;
};

constexpr int kTokens = 32;   // of a workgroup, where there are several

__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// The largest key and its lowest index; every lane gets them.
__device__ __forceinline__ void wave_best(double &key, int &idx)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const double k = __shfl_xor(key, o, 64);
        const int i = __shfl_xor(idx, o, 64);
        if (k > key || (k == key && i < idx)) key = k, idx = i;
    }
}

// Token m's experts: lane j < top_k gets the j-th one's id (-1: none) and weight. `keys`: E doubles of LDS (groups).
template <int NE> __device__ void route_token(const RArgs &a, int m, double *keys, int &id, float &weight)
{
    const int lane = threadIdx.x & 63;
    id = -1;
    weight = 0.f;
    if (a.active && !a.active[m]) return;
    double x[NE], p[NE], key[NE];
    double most = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int e = lane + 64 * i;
        float v = -INFINITY;
        if (e < a.E) v = a.f32 ? static_cast<const float *>(a.logits)[(size_t)m * a.rs + e] : (float)static_cast<const _Float16 *>(a.logits)[(size_t)m * a.rs + e];
        x[i] = v > 3.402823466e38f ? 3.402823466e38 : (double)v;
        most = fmax(most, x[i]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < NE; i++) p[i] = 1.0 / (1.0 + exp(-x[i]));
    } else {
        most = wave_max(most);
        if (most == -INFINITY) most = 0.0;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NE; i++) {
            p[i] = exp(x[i] - most);
            sum += p[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < NE; i++) p[i] = p[i] / sum;
    }
    // the keys: choices, or logits where no bias changes the order; behind every number a NaN, and behind that what is no candidate
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int e = lane + 64 * i;
        const bool can = e < a.E && x[i] != -INFINITY;
        const double c = a.bias && e < a.E ? p[i] + (double)a.bias[e] : p[i];
        const double k = a.bias ? c : x[i];
        key[i] = !can ? -INFINITY : k == k ? fmin(fmax(k, -1e300), 1e300) : -1e300;
        if (a.n_group > 1 && e < a.E) keys[e] = !can ? -INFINITY : c == c ? fmin(fmax(c, -1e300), 1e300) : -1e300;
    }
    if (a.n_group > 1) {
        // (one wave's own part of LDS: its writes are seen by its later reads)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        double value = -INFINITY;
        if (lane < a.n_group) {
            double first = -INFINITY, second = -INFINITY;
            for (int j = 0; j < a.run; j++) {
                const double k = keys[lane * a.run + j];
                if (k > first) second = first, first = k;
                else if (k > second) second = k;
            }
            value = a.group_best == 2 && second > -INFINITY ? first + second : first;
        }
        uint64_t in = 0;
        for (int g = 0; g < a.top_group; g++) {
            double k = value;
            int i = lane;
            wave_best(k, i);
            if (k == -INFINITY) break;
            in |= (uint64_t)1 << i;
            if (lane == i) value = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < NE; i++) {
            const int e = lane + 64 * i;
            if (e < a.E && !((in >> (e / a.run)) & 1)) key[i] = -INFINITY;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    double sum = 0.0, mine = 0.0;
    for (int j = 0; j < a.top_k; j++) {
        double k = key[0];
        int at = lane;
#pragma unroll
        for (int i = 1; i < NE; i++)
            if (key[i] > k) k = key[i], at = lane + 64 * i;
        wave_best(k, at);
        if (k == -INFINITY) break;
        double w = 0.0;
#pragma unroll
        for (int i = 0; i < NE; i++)
            if (lane + 64 * i == at) {
                w = p[i];
                key[i] = -INFINITY;
            }
        w = __shfl(w, at & 63, 64);
        sum += w;
        if (lane == j) id = at, mine = w;
    }
    if (a.renorm) mine = sum == 0.0 ? 0.0 : mine / sum;
    weight = id < 0 ? 0.f : (float)(mine * (double)a.scale);
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

// A workgroup's tokens. ONE: all tokens (up to 64), with the plan; otherwise kTokens of them, and their counts.
template <int NE, bool ONE> __global__ __launch_bounds__(1024) void k_route(const RArgs a)
{
    using Mask = std::conditional_t<ONE, unsigned long long, unsigned>;
    constexpr int T = ONE ? 64 : kTokens;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int part[16], start[kMaxExperts + 1];
    __shared__ Mask mask[kMaxExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / 64, t0 = blockIdx.x * T;
    double *const keys = reinterpret_cast<double *>(smem) + (size_t)wave * a.E;
    if (a.plan) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) mask[e] = 0;
        __syncthreads();
    }
    for (int t = wave; t < T && t0 + t < a.M; t += waves) {
        const int m = t0 + t;
        int id;
        float w;
        route_token<NE>(a, m, keys, id, w);
        if (lane < a.top_k) {
            a.ids[(size_t)m * a.top_k + lane] = id;
            a.weight[(size_t)m * a.top_k + lane] = w;
            if (a.plan && id >= 0) atomicOr(&mask[id], (Mask)1 << t);
        }
    }
    if (!a.plan) return;
    __syncthreads();
    if constexpr (!ONE) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) a.counts[(size_t)blockIdx.x * a.E + e] = __popc(mask[e]);
    } else {
        // (1024 threads, at most as many experts)
        const int n = (int)threadIdx.x < a.E ? __popcll(mask[threadIdx.x]) : 0;
        int all;
        const int at = group_scan(n, part, all);
        if ((int)threadIdx.x < a.E) {
            start[threadIdx.x] = at;
            a.off[threadIdx.x] = at;
        }
        if (threadIdx.x == 0) a.off[a.E] = all;
        __syncthreads();
        for (int i = threadIdx.x; i < a.M * a.top_k; i += blockDim.x) {
            const int t = i / a.top_k, id = a.ids[i];
            int r = -1;
            if (id >= 0) {
                r = start[id] + __popcll(mask[id] & (((Mask)1 << t) - 1));
                a.src[r] = t;
            }
            a.slot[i] = r;
        }
    }
}

// Counts of the workgroups of tokens to starts, in place: one workgroup of 1024 threads. Threads split the blocks of an
// expert where there are fewer experts than threads.
__global__ __launch_bounds__(1024) void k_starts(const RArgs a, int nblk)
{
    __shared__ int part[16], sums[1024];
    int P = 1;                                     // parts of an expert's column
    while (2 * P * a.E <= 1024) P *= 2;
    const int e = threadIdx.x % a.E, s = threadIdx.x / a.E, per = (nblk + P - 1) / P;
    const bool in = s < P && (int)threadIdx.x < P * a.E;
    const int b0 = min(nblk, s * per), b1 = min(nblk, b0 + per);
    int n = 0;
    if (in)
        for (int b = b0; b < b1; b++) n += a.counts[(size_t)b * a.E + e];
    sums[threadIdx.x] = in ? n : 0;
    __syncthreads();
    int total = 0;
    if ((int)threadIdx.x < a.E)
        for (int i = 0; i < P; i++) total += sums[i * a.E + threadIdx.x];
    int all;
    const int at = group_scan(total, part, all);
    if ((int)threadIdx.x < a.E) a.off[threadIdx.x] = at;
    if (threadIdx.x == 0) a.off[a.E] = all;
    // (starts of the parts: the expert's, and the parts before)
    __shared__ int first[1024];
    if ((int)threadIdx.x < a.E) {
        int f = at;
        for (int i = 0; i < P; i++) {
            first[i * a.E + threadIdx.x] = f;
            f += sums[i * a.E + threadIdx.x];
        }
    }
    __syncthreads();
    if (in) {
        int f = first[threadIdx.x];
        for (int b = b0; b < b1; b++) {
            const size_t i = (size_t)b * a.E + e;
            const int c = a.counts[i];
            a.counts[i] = f;
            f += c;
        }
    }
}

// Rows of a workgroup's tokens.
__global__ __launch_bounds__(256) void k_rows(const RArgs a)
{
    __shared__ unsigned mask[kMaxExperts];
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) mask[e] = 0;
    __syncthreads();
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
            r = a.counts[(size_t)blockIdx.x * a.E + id] + __popc(mask[id] & ((1u << t) - 1u));
            a.src[r] = t0 + t;
        }
        a.slot[i0 + i] = r;
    }
}

template <int NE> hipError_t launch(const RArgs &a, hipStream_t s, uint64_t *blocks)
{
    static std::atomic<uint64_t> opt1{0}, opt2{0};
    const bool one = a.M <= 64;
    const int waves = std::min(one ? 16 : 8, a.M), threads = one ? 1024 : 512, nblk = one ? 1 : (a.M + kTokens - 1) / kTokens;
    (void)waves;
    const int lds = a.n_group > 1 ? threads / 64 * a.E * (int)sizeof(double) : 0, most = threads / 64 * 64 * NE * (int)sizeof(double);
    if (one) {
        if (most > 48 << 10)
            if (hipError_t e = lds_opt_in(reinterpret_cast<const void *>(&k_route<NE, true>), most, opt1)) return e;
        hipLaunchKernelGGL((k_route<NE, true>), dim3(1), dim3(threads), lds, s, a);
    } else {
        if (most > 48 << 10)
            if (hipError_t e = lds_opt_in(reinterpret_cast<const void *>(&k_route<NE, false>), most, opt2)) return e;
        hipLaunchKernelGGL((k_route<NE, false>), dim3((unsigned)nblk), dim3(threads), lds, s, a);
    }
    *blocks = (uint64_t)nblk;
    if (one || !a.plan) return hipGetLastError();
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(k_starts, dim3(1), dim3(1024), 0, s, a, nblk);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(k_rows, dim3((unsigned)nblk), dim3(256), 0, s, a);
    *blocks += (uint64_t)nblk + 1;
    return hipGetLastError();
}

}  // namespace

size_t route_ws(const Route &L) { return L.off && L.M > 64 ? (size_t)((L.M + kTokens - 1) / kTokens) * L.E * sizeof(int32_t) : 0; }

hipError_t moe_route(const Route &L, hipStream_t s, uint64_t *blocks)
{
    RArgs a;
    a.logits = L.logits; a.rs = L.rs; a.bias = L.bias; a.active = L.active; a.M = L.M; a.E = L.E; a.n_group = L.n_group; a.run = L.E / L.n_group;
    a.group_best = L.group_best; a.top_group = L.top_group; a.top_k = L.top_k; a.renorm = L.renorm; a.sigmoid = L.sigmoid; a.f32 = L.f32;
    a.plan = L.off != nullptr; a.scale = L.scale; a.ids = L.ids; a.off = L.off; a.src = L.src; a.slot = L.slot; a.counts = L.counts; a.weight = L.weight;
    if (L.E <= 64) return launch<1>(a, s, blocks);
    if (L.E <= 128) return launch<2>(a, s, blocks);
    if (L.E <= 256) return launch<4>(a, s, blocks);
    if (L.E <= 512) return launch<8>(a, s, blocks);
    return launch<16>(a, s, blocks);
}

}  // namespace rk
