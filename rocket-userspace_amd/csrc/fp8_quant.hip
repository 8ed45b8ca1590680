// fp8_quant.hip — rows, or gated rows, to e4m3 codes with one fp32 scale for each 128 values, one pass.
//
// A group of 128 is 16 lanes of eight values: two wide loads a lane, the maximum a shuffle over 16 lanes, eight
// codes one 8-byte store. Groups are counted through all rows, so that no size of row leaves lanes idle but in a last
// part of a group. Memory bounds it: 512 fp32 rows of 15360 take 7.6 us (5.2 TB/s, as a large copy), 24576 gated fp16 rows of 1408
// 34 us (5.1 TB/s).
#include "f8codes.h"
#include "gemm_impl.h"

namespace rk {
namespace {

struct QArgs {
    const void *a, *up;
    long rs;
    uint8_t *q;
    float *scale;
    const int32_t *n_rows;
    uint32_t groups;      // of all rows
    int K, nb;
    float rnb;            // 1 / nb
};

template <bool F16, int ACT> __global__ __launch_bounds__(256) void k_quant_fp8(const QArgs a)
{
    const int l = threadIdx.x % 16;
    const uint32_t g0 = blockIdx.x * 16u;
    const uint32_t m0 = g0 / (uint32_t)a.nb;
    const int rest = (int)(g0 - m0 * (uint32_t)a.nb) + threadIdx.x / 16;   // < nb + 16
    const int dm = (int)((rest + 0.5f) * a.rnb);                           // exact: nb <= 512
    const uint32_t m = m0 + (uint32_t)dm;
    const int b = rest - dm * a.nb, k = b * kF8Block + 8 * l;
    const bool row = g0 + threadIdx.x / 16 < a.groups && (!a.n_rows || (int)m < *a.n_rows);
    const bool in = row && k < a.K;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.f;
    if (in) {
        gk::load8f<F16>(a.a, (long)m * a.rs + k, v);
        if constexpr (ACT != kActIdentity) {
            float u[8];
            gk::load8f<F16>(a.up, (long)m * a.rs + k, u);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = gk::act_k<ACT>(v[e]) * u[e];
        }
    }
    const float x = f8_group_amax(v);
    if (in) *reinterpret_cast<uint2 *>(a.q + (size_t)m * a.K + k) = f8_codes(v, 448.f / x);
    if (row && l == 0) a.scale[(size_t)m * a.nb + b] = x / 448.f;
}

}  // namespace

hipError_t quant_fp8(const QuantF8 &L, hipStream_t s, uint64_t *blocks)
{
    QArgs a;
    a.a = L.a; a.up = L.up; a.rs = L.rs; a.q = L.q; a.scale = L.scale; a.n_rows = L.n_rows; a.K = L.K; a.nb = f8_blocks(L.K);
    const uint64_t groups = (uint64_t)L.M * a.nb;
    if (groups >= (uint64_t)1 << 31) return hipErrorInvalidValue;
    a.groups = (uint32_t)groups;
    a.rnb = 1.f / (float)a.nb;
    *blocks = (groups + 15) / 16;
    const dim3 grid((unsigned)*blocks);
    if (L.act == kActSilu) {
        if (L.f32) hipLaunchKernelGGL((k_quant_fp8<false, kActSilu>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_quant_fp8<true, kActSilu>), grid, dim3(256), 0, s, a);
    } else if (L.act == kActGelu) {
        if (L.f32) hipLaunchKernelGGL((k_quant_fp8<false, kActGelu>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_quant_fp8<true, kActGelu>), grid, dim3(256), 0, s, a);
    } else {
        if (L.f32) hipLaunchKernelGGL((k_quant_fp8<false, kActIdentity>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_quant_fp8<true, kActIdentity>), grid, dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace rk
