// f8tile.h — what the kernels of e4m3 products share: which rows of which expert a workgroup has, the rows' addresses,
// the matrix unit's products of codes, and the stores.
//
// A result block is 16 x 16: the weights' rows are the MFMA's first operand, the activations' its second, so that a lane
// holds one row m = l % 16 of C and four columns 4 (l / 16) + r. One scale a lane and block of 128, columns that are
// neighbours in memory. A lane supplies 32 of a row's 128 codes; which ones does not matter to the sum, if both operands
// hold the same: chunks l / 16 and 4 + l / 16 of 16 codes.
#pragma once

#include "gemm_impl.h"
#include "layer.h"

namespace rk {
namespace f8 {

using gk::f32x4;
using gk::i32x4;
using gk::Rsrc;
typedef int      i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kOOB = gk::kOOB;

struct Args {
    const uint8_t *A, *B;
    const float *sa, *sb;
    const int32_t *src, *off;
    void *C;
    float *ws;            // slices of K: [slice][M][N rounded up to 4]
    int M, K, N, nb, E, a_rows;
    int nbn, bm_tiles;    // column tiles; row tiles (experts: the most that there can be)
    int slices, per;      // slices of K and the blocks of one
    int band;             // row tiles that neighbours in the launch share columns over
};

// The rows [m0, m1) of C that tile t has, and their expert; m0 == m1: none. Experts' tiles of BM rows are counted in order
// of the experts, by one wave's scan of 64 experts at a time; every lane gets the result.
template <int BM> __device__ __forceinline__ void tile_rows(const Args &a, int t, int &e, int &m0, int &m1)
{
    if (!a.off) {
        e = 0;
        m0 = t * BM;
        m1 = min(a.M, m0 + BM);
        return;
    }
    const int lane = threadIdx.x & 63;
    e = 0;
    m0 = m1 = 0;
    for (int e0 = 0, first = 0; e0 < a.E; e0 += 64) {
        const int i = min(e0 + lane, a.E - 1);
        const int lo = min(max(a.off[i], 0), a.M), hi = min(max(a.off[i + 1], lo), a.M);
        int n = e0 + lane < a.E ? (hi - lo + BM - 1) / BM : 0, upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            if (lane >= o) upto += v;
        }
        const int all = __shfl(upto, 63, 64);
        if (t < first + all) {   // (the same in every lane)
            const uint64_t past = __ballot(first + upto > t);
            const int w = __builtin_ctzll(past);
            const int at = t - first - (__shfl(upto, w, 64) - __shfl(n, w, 64));
            e = __builtin_amdgcn_readfirstlane(e0 + w);
            const int l = __shfl(lo, w, 64), h = __shfl(hi, w, 64);
            m0 = __builtin_amdgcn_readfirstlane(l + at * BM);
            m1 = __builtin_amdgcn_readfirstlane(min(h, l + (at + 1) * BM));
            return;
        }
        first += all;
    }
}

// Row of A that row m of C is made of; -1: none (zeros).
__device__ __forceinline__ int source(const Args &a, int m)
{
    if (!a.src) return m;
    const int r = a.src[m];
    return (unsigned)r < (unsigned)a.a_rows ? r : -1;
}

// 32 codes as fp16, in the order that they lie in (e4m3 is exact in fp16).
__device__ __forceinline__ void widen(const i32x4 &c, f16x8 (&w)[2])
{
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true);
        w[i / 2][4 * (i & 1)] = lo[0];
        w[i / 2][4 * (i & 1) + 1] = lo[1];
        w[i / 2][4 * (i & 1) + 2] = hi[0];
        w[i / 2][4 * (i & 1) + 3] = hi[1];
    }
#endif
}

// A lane's 32 codes of a row's block, as the products take them. WIDE: fp16, whose products the matrix unit sums in
// fp32; otherwise the codes, of whose products it cuts each eight at 2^-13 of the largest.
template <bool WIDE> struct Frag;
template <> struct Frag<false> {
    i32x8 v;
    __device__ __forceinline__ void set(const i32x4 &lo, const i32x4 &hi)
    {
        v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
template <> struct Frag<true> {
    f16x8 v[4];
    __device__ __forceinline__ void set(const i32x4 &lo, const i32x4 &hi)
    {
        f16x8 w[2];
        widen(lo, w);
        v[0] = w[0];
        v[1] = w[1];
        widen(hi, w);
        v[2] = w[0];
        v[3] = w[1];
    }
};
// The same as it was loaded, which is kept where a widened one would take too many registers.
struct Codes {
    i32x4 lo, hi;
};
__device__ __forceinline__ f32x4 product(const Frag<false> &b, const Frag<false> &a)
{
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, z, 0, 0, 0, 0, 0, 0);
#else
    return z;
#endif
}
__device__ __forceinline__ f32x4 product(const Frag<true> &b, const Frag<true> &a)
{
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int i = 0; i < 4; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[i], a.v[i], d, 0, 0, 0);
#endif
    return d;
}

// Columns n .. n + 3 of one row (those below N). `wide`: N is a multiple of 4, so that a row's start is aligned to four.
__device__ __forceinline__ void store4(_Float16 *row, int n, int N, bool wide, f32x4 v)
{
    const f16x4 o = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    if (wide) {
        if (n < N) *reinterpret_cast<f16x4 *>(row + n) = o;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < N) row[n + r] = o[r];
    }
}
__device__ __forceinline__ void store4(float *row, int n, int N, bool wide, f32x4 v)
{
    if (wide) {
        if (n < N) *reinterpret_cast<f32x4 *>(row + n) = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < N) row[n + r] = v[r];
    }
}
// Columns n .. n + 7 of one row (those below N, a multiple of 4): one store where the row is aligned to it.
__device__ __forceinline__ void store8(_Float16 *row, int n, int N, f32x4 v, f32x4 w)
{
    const f16x8 o = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3], (_Float16)w[0], (_Float16)w[1], (_Float16)w[2], (_Float16)w[3]};
    if (N % 8 == 0) {
        if (n < N) *reinterpret_cast<f16x8 *>(row + n) = o;
    } else {
        store4(row, n, N, true, v);
        store4(row, n + 4, N, true, w);
    }
}
__device__ __forceinline__ void store8(float *row, int n, int N, f32x4 v, f32x4 w)
{
    store4(row, n, N, true, v);
    store4(row, n + 4, N, true, w);
}

Args args(const GemmF8 &L);
// The most tiles of bm rows that the launch's experts can have.
inline long row_tiles(const GemmF8 &L, int bm)
{
    if (!L.off) return (L.M + (long)bm - 1) / bm;
    const long used = L.n_expert < L.M ? L.n_expert : L.M;
    return ((long)L.M + used * (bm - 1)) / bm;
}

}  // namespace f8
}  // namespace rk
