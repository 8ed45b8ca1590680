// add_norm.hip — a block's result joins the residual stream: (the experts' weighted sum,) its norm, gate and scale, the
// sum, the next block's norm, and its rows as fp16 and / or e4m3 codes, one pass.
//
// A workgroup is a row, a lane eight neighbours of it (two such runs above 8192 values), so a row is read once and kept in
// registers through both norms; each square sum is a shuffle over the wave and one exchange through LDS. Sixteen lanes
// hold a group of 128, whose maximum is a shuffle. Memory bounds long calls: 4096 fp32 rows of 3840 with codes 44.0 us, 4.7 TB/s.
// Two exchanges and the loads' latency bound short ones: 16 rows of 2048, six experts' rows each, 5.4 us, of which a launch is some
// 4. (Four experts' rows in flight instead of one: 5.7 us, and 38.9 instead of 37.6 for 4096 tokens.)
#include "f8codes.h"
#include "gemm_impl.h"

namespace rk {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct NArgs {
    const void *h, *y, *shared;
    void *h_out;
    long y_rs;
    const _Float16 *w_post, *w_pre, *gate;
    float eps_post, eps_pre, alpha, rH;
    int gate_every, H, nb, top_k, rows;
    const int32_t *slot;
    const float *weight;
    _Float16 *x;
    uint8_t *xq;
    float *x_scale;
};

__device__ __forceinline__ void store8(_Float16 *p, const float (&v)[8])
{
    f16x8 o;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = (_Float16)v[e];
    *reinterpret_cast<f16x8 *>(p) = o;
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8])
{
    *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}

// The sum of squares of the row whose values the workgroup holds, the same in every thread. `part`: a word a wave.
template <int V> __device__ __forceinline__ float row_squares(const float (&v)[V][8], float *part)
{
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) q = fmaf(v[i][e], v[i][e], q);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) q += __shfl_xor(q, o, 64);
    const int waves = blockDim.x / 64;
    if (waves > 1) {
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = q;
        __syncthreads();
        q = 0.f;
        for (int w = 0; w < waves; w++) q += part[w];
    }
    return q;
}

// 1 / sqrt(mean of squares + eps) of the row, for its values as the call leaves them: where the squares pass fp32's range, or lie so low in
// it that they lose bits, the values are scaled by a power of two, which the norm does not see. Scaled down (2^48 is the largest then, and
// the row's mean square at least 2^-46), a value loses bits only where its norm is below 2^-103; scaled up, none does.
template <int V> __device__ __forceinline__ float row_rsqrt(float (&v)[V][8], float rH, float eps, float *part)
{
    float d = fmaf(row_squares<V>(v, part), rH, eps);
    if (!(d >= 0x1p-96f && d <= 3.402823466e38f)) {   // (a NaN too; the same in every thread)
        const float s = d < 1.f ? 0x1p100f : 0x1p-80f;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= s;
        __syncthreads();   // (all have read `part`)
        d = fmaf(row_squares<V>(v, part), rH, eps * s * s);
    }
    return 1.f / sqrtf(d);
}

template <bool F16, bool MOE, int V> __global__ __launch_bounds__(1024) void k_add_norm(const NArgs a)
{
    using T = std::conditional_t<F16, _Float16, float>;
    __shared__ float part[2][16];
    const int m = blockIdx.x;
    const size_t row = (size_t)m * a.H;
    int k[V];
    bool in[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        k[i] = (i * blockDim.x + threadIdx.x) * 8;
        in[i] = k[i] < a.H;
    }
    float hv[V][8], z[V][8];
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) hv[i][e] = z[i][e] = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
        if (in[i]) gk::load8f<F16>(a.h, row + k[i], hv[i]);
    if (MOE || a.y) {
        if constexpr (MOE) {
            const int32_t *slot = a.slot + (size_t)m * a.top_k;
            const float *weight = a.weight + (size_t)m * a.top_k;
            for (int j = 0; j < a.top_k; j++) {
                const int r = slot[j];
                if (r < 0 || r >= a.rows) continue;
                const float w = weight[j];
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (in[i]) {
                        float u[8];
                        gk::load8f<F16>(a.y, (size_t)r * a.H + k[i], u);
#pragma unroll
                        for (int e = 0; e < 8; e++) z[i][e] = fmaf(w, u[e], z[i][e]);
                    }
            }
            if (a.shared) {
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (in[i]) {
                        float u[8];
                        gk::load8f<F16>(a.shared, row + k[i], u);
#pragma unroll
                        for (int e = 0; e < 8; e++) z[i][e] += u[e];
                    }
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (in[i]) gk::load8f<F16>(a.y, (long)m * a.y_rs + k[i], z[i]);
        }
        const float r = a.eps_post >= 0.f ? row_rsqrt<V>(z, a.rH, a.eps_post, part[0]) : 1.f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            float w[8], g[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = g[e] = 1.f;
            if (in[i] && a.w_post) gk::load8f<true>(a.w_post, k[i], w);
            if (in[i] && a.gate) gk::load8f<true>(a.gate, (size_t)(m / a.gate_every) * a.H + k[i], g);
#pragma unroll
            for (int e = 0; e < 8; e++) hv[i][e] = fmaf(a.alpha * g[e], z[i][e] * r * w[e], hv[i][e]);
        }
    }
    if (a.h_out) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (in[i]) store8(static_cast<T *>(a.h_out) + row + k[i], hv[i]);
    }
    if (!a.x && !a.xq) return;
    const float r = a.eps_pre >= 0.f ? row_rsqrt<V>(hv, a.rH, a.eps_pre, part[1]) : 1.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = 1.f;
        if (in[i] && a.w_pre) gk::load8f<true>(a.w_pre, k[i], w);
#pragma unroll
        for (int e = 0; e < 8; e++) hv[i][e] *= r * w[e];
        if (in[i] && a.x) store8(a.x + row + k[i], hv[i]);
        if (a.xq) {
            const float x = f8_group_amax(hv[i]);
            if (in[i]) {
                *reinterpret_cast<uint2 *>(a.xq + row + k[i]) = f8_codes(hv[i], 448.f / x);
                if (threadIdx.x % 16 == 0) a.x_scale[(size_t)m * a.nb + k[i] / kF8Block] = x / 448.f;
            }
        }
    }
}

template <bool F16, bool MOE> void launch(const NArgs &a, int M, int threads, hipStream_t s)
{
    if (a.H <= 8192) hipLaunchKernelGGL((k_add_norm<F16, MOE, 1>), dim3((unsigned)M), dim3((unsigned)threads), 0, s, a);
    else hipLaunchKernelGGL((k_add_norm<F16, MOE, 2>), dim3((unsigned)M), dim3((unsigned)threads), 0, s, a);
}

}  // namespace

hipError_t add_norm(const AddNorm &L, hipStream_t s, uint64_t *blocks)
{
    NArgs a;
    a.h = L.h; a.y = L.y; a.shared = L.shared; a.h_out = L.h_out; a.y_rs = L.y_rs; a.w_post = L.w_post; a.w_pre = L.w_pre; a.gate = L.gate;
    a.eps_post = L.eps_post; a.eps_pre = L.eps_pre; a.alpha = L.alpha; a.rH = 1.f / (float)L.H; a.gate_every = L.gate_every; a.H = L.H;
    a.nb = f8_blocks(L.H); a.top_k = L.top_k; a.rows = L.rows; a.slot = L.slot; a.weight = L.weight; a.x = L.x; a.xq = L.xq; a.x_scale = L.x_scale;
    const int per = L.H <= 8192 ? 8 : 16, threads = (L.H + per * 64 - 1) / (per * 64) * 64;
    *blocks = (uint64_t)L.M;
    if (L.f32) L.top_k ? launch<false, true>(a, L.M, threads, s) : launch<false, false>(a, L.M, threads, s);
    else L.top_k ? launch<true, true>(a, L.M, threads, s) : launch<true, false>(a, L.M, threads, s);
    return hipGetLastError();
}

}  // namespace rk
