// fp8_rows.hip — products of e4m3 codes with block scales for few rows of activations: a pass over the weights.
//
// A workgroup has NB blocks of 16 rows of the weights and up to 16 rows of activations (of one expert); its waves take the
// blocks of 128 codes of K in turn, each straight from memory to registers, and join their sums through LDS. Codes are
// widened to fp16, whose products the matrix unit sums in fp32: beside the weights' way from memory that is free.
#include "f8tile.h"

#include <algorithm>

namespace rk {
namespace f8 {
namespace {

// NB: blocks of 16 weight rows a workgroup.
template <int NB, bool F16> __global__ __launch_bounds__(512) void k_rows_fp8(const Args a)
{
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int bn = blockIdx.x % a.nbn, tile = blockIdx.x / a.nbn;
    int e, m0, m1;
    tile_rows<16>(a, tile, e, m0, m1);
    if (m0 >= m1) return;
    const int n0 = bn * 16 * NB, q = lane >> 4, c = lane & 15;

    const uint8_t *const Bt = a.B + ((size_t)e * a.N + n0) * a.K;
    const Rsrc rB = gk::rsrc_u(Bt, (uint32_t)min(16 * NB, a.N - n0) * (uint32_t)a.K);
    const uint8_t *const At = a.src ? a.A : a.A + (size_t)m0 * a.K;
    const float *const sat = a.src ? a.sa : a.sa + (size_t)m0 * a.nb;
    const uint32_t arows = a.src ? (uint32_t)a.a_rows : (uint32_t)(m1 - m0);
    const Rsrc rA = gk::rsrc_u(At, arows * (uint32_t)a.K), rS = gk::rsrc_u(sat, arows * (uint32_t)a.nb * 4u);
    const int r = m0 + c < m1 ? (a.src ? source(a, m0 + c) : c) : -1;
    const uint32_t va = r < 0 ? kOOB : (uint32_t)r * (uint32_t)a.K + 16u * q, vs = r < 0 ? kOOB : (uint32_t)r * (uint32_t)a.nb * 4u;
    uint32_t vb[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) vb[j] = (uint32_t)(16 * j + c) * (uint32_t)a.K + 16u * q;
    const float *const sb = a.sb + ((size_t)e * ((a.N + 127) / 128) + n0 / 128) * a.nb;

    f32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // A wave's next block is on its way while this one is multiplied. (Codes past K read zeros.)
    struct Block {
        i32x4 wb[NB][2], wa[2];
        float sa, sb;
    } x[2];
    auto load = [&](Block &x, int b) __attribute__((always_inline)) {
        const uint32_t k = (uint32_t)b * 128u;
        const uint32_t z0 = k + 16u * q < (uint32_t)a.K ? 0u : kOOB, z1 = k + 64u + 16u * q < (uint32_t)a.K ? 0u : kOOB;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            x.wb[j][0] = gk::ld16(rB, (vb[j] + k) | z0);
            x.wb[j][1] = gk::ld16(rB, (vb[j] + k + 64u) | z1);
        }
        x.wa[0] = gk::ld16(rA, (va + k) | z0);
        x.wa[1] = gk::ld16(rA, (va + k + 64u) | z1);
        x.sa = gk::ld4f(rS, vs + (uint32_t)b * 4u);
        x.sb = sb[b];
    };
    auto step = [&](Block &x, Block &y, int b) __attribute__((always_inline)) {
        if (b + waves < a.nb) load(y, b + waves);
        __builtin_amdgcn_sched_barrier(0);
        Frag<true> fa;
        fa.set(x.wa[0], x.wa[1]);
        const float f = x.sa * x.sb;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            Frag<true> fb;
            fb.set(x.wb[j][0], x.wb[j][1]);
            const f32x4 d = product(fb, fa);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[j][i] = fmaf(d[i], f, acc[j][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (wave < a.nb) load(x[0], wave);
    for (int b = wave; b < a.nb; b += 2 * waves) {
        step(x[0], x[1], b);
        if (b + waves < a.nb) step(x[1], x[0], b + waves);
    }

    // the waves' sums, in order of the waves: thread t has what lane t % 64 of every wave had of block t / 64
    f32x4 *const part = reinterpret_cast<f32x4 *>(smem);
#pragma unroll
    for (int j = 0; j < NB; j++) part[(wave * NB + j) * 64 + lane] = acc[j];
    __syncthreads();
    for (int t = threadIdx.x; t < NB * 64; t += blockDim.x) {
        f32x4 v = part[t];
        for (int w = 1; w < waves; w++) v += part[w * NB * 64 + t];
        if (r < 0) v = f32x4{0.f, 0.f, 0.f, 0.f};   // (row t & 15 is the lane's own c; without a source its sums are zeros times the weights)
        const int m = m0 + (t & 15), n = n0 + 16 * (t >> 6) + 4 * (t >> 4 & 3);
        using T = std::conditional_t<F16, _Float16, float>;
        if (m < m1) store4(static_cast<T *>(a.C) + (size_t)m * a.N, n, a.N, a.N % 4 == 0, v);
    }
#endif
}

template <int NB> hipError_t launch(Args a, const GemmF8 &L, int waves, hipStream_t s, uint64_t *blocks)
{
    a.nbn = (L.N + 16 * NB - 1) / (16 * NB);
    const long grid = row_tiles(L, 16) * a.nbn;
    if (grid >= (long)1 << 31) return hipErrorInvalidValue;
    *blocks = (uint64_t)grid;
    const int lds = waves * NB * 64 * 16;
    if (L.f16) hipLaunchKernelGGL((k_rows_fp8<NB, true>), dim3((unsigned)grid), dim3(64 * waves), lds, s, a);
    else hipLaunchKernelGGL((k_rows_fp8<NB, false>), dim3((unsigned)grid), dim3(64 * waves), lds, s, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace f8

namespace {

// Weight rows a workgroup, in blocks of 16: a CU takes some 28 KB a us through registers, the activations' rows (from L2) among them, so
// that which has to pass through the fullest CU decides. 3840 -> 15360, 16 rows, one, two and four blocks: 17.1, 13.1, 11.8 us;
// 15360 -> 3840, one row: 11.8, 18.4, 31.6 us.
struct Rows {
    int nb;
    float us;
};
Rows rows_plan(const GemmF8 &L)
{
    const float used = L.off ? (float)std::min(L.n_expert, L.M) : 1.f, mean = (float)L.M / used;
    if (mean > 16.f) return {1, INFINITY};
    const float tiles = L.off ? used * std::max(1.f, mean / 16.f + 0.5f) : 1.f, mem = used * (float)L.N * (float)L.K / 5.9e6f;
    Rows r = {1, INFINITY};
    for (int nb : {1, 2, 4}) {
        const float w = tiles * (float)((L.N + 16 * nb - 1) / (16 * nb));
        const float cu = ceilf(w / 256.f) * (16 * nb + std::min(16.f, mean)) * (float)L.K / 28e3f;
        const float us = 2.f + std::max(cu, mem) + 0.02f * cu;   // (of equal ones the one that takes fewer bytes)
        if (us < r.us) r = {nb, us};
    }
    return r;
}

}  // namespace

float gemm_fp8_rows_us(const GemmF8 &L) { return rows_plan(L).us; }

hipError_t gemm_fp8_rows(const GemmF8 &L, hipStream_t s, uint64_t *blocks)
{
    using namespace f8;
    const Args a = args(L);
    const int nb = rows_plan(L).nb;
    // Six waves where a CU has one workgroup (3840 -> 15360, one row: 11.3 us, with four 12.6, with eight 12.2; 15360 -> 3840: 12.2,
    // 14.5, 12.0), four where it has several (64 experts' 2048 -> 2816, a row or two each: 40.6 us, with six 50.0).
    const int waves = row_tiles(L, 16) * ((L.N + 16 * nb - 1) / (16 * nb)) <= 256 ? 6 : 4;
    if (nb == 1) return launch<1>(a, L, waves, s, blocks);
    if (nb == 2) return launch<2>(a, L, waves, s, blocks);
    return launch<4>(a, L, waves, s, blocks);
}

}  // namespace rk
