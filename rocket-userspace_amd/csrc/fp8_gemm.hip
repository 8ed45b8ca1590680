// fp8_gemm.hip — products of e4m3 codes with block scales, by tiles: C[m][n] = sum_b sa[m][b] sb[n / 128][b] (A_b B_b^T)[m][n].
//
// A stage is one block of 128 codes: the tile's rows of A and B go by DMA into a ring of LDS slots (chunks swizzled by
// their source address, so that sixteen lanes' 16-byte reads cover all banks once), with the rows' scales beside them. A wave
// multiplies its part of the tile for that block alone and adds the products, times one scale a lane, to its fp32 sums:
// one VALU operation an element and block, behind one MFMA an element block.
#include "f8tile.h"

#include <algorithm>

namespace rk {
namespace f8 {

Args args(const GemmF8 &L)
{
    Args a;
    a.A = L.A; a.B = L.B; a.sa = L.sa; a.sb = L.sb; a.src = L.src; a.off = L.off; a.C = L.C; a.ws = nullptr;
    a.M = L.M; a.K = L.K; a.N = L.N; a.nb = f8_blocks(L.K); a.E = L.n_expert; a.a_rows = L.a_rows;
    a.nbn = a.bm_tiles = 0;
    a.slices = 1;
    a.per = a.nb;
    a.xcds = 8;
    a.band = 8;
    return a;
}

namespace {

// Rows of the weights' tile in the order that a lane's columns become neighbours: MFMA row 4 q + r of block j is row
// 32 (j / 2) + 8 q + 4 (j % 2) + r, so that blocks 2 p and 2 p + 1 give a lane eight neighbours. The swizzle of a tile row:
// sixteen rows of an MFMA operand cover every pair of row parity and slot once.
[[maybe_unused]] __device__ constexpr int sw_a(int row) { return (row >> 1) & 7; }
[[maybe_unused]] __device__ constexpr int sw_b(int row) { return ((row >> 1) & 1) | ((row >> 2) & 6); }

template <int BM_, int BN_, int WGM_, int WGN_, int SLOTS_> struct Cfg {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, SLOTS = SLOTS_;
    static constexpr int NW = WGM * WGN, NT = 64 * NW, WTM = BM / WGM, WTN = BN / WGN, TM = WTM / 16, TN = WTN / 16;
    static constexpr int IA = BM / NW / 8, IB = BN / NW / 8;   // DMA instructions a wave and stage
    static constexpr int RWS = BM / NW;                        // rows whose scales a wave loads
    static constexpr int SLOT = (BM + BN) * 128 + NW * 256;
    static constexpr int NVM = IA + IB + 1;
    static constexpr int SBN = (BN + 127) / 128;               // blocks of 128 columns
    static_assert(IA >= 1 && IB >= 1 && RWS <= 64 && TN % 2 == 0 && (WTN == 128 || 128 % WTN == 0), "tile");
    static constexpr int lds(int per) { return SLOTS * SLOT + SBN * per * 4; }
};

template <class CF, bool WIDE, bool F16> __global__ __launch_bounds__(CF::NT) void k_gemm_fp8(const Args a)
{
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BM = CF::BM, BN = CF::BN, TM = CF::TM, TN = CF::TN, SLOTS = CF::SLOTS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *const sbl = reinterpret_cast<float *>(smem + SLOTS * CF::SLOT);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / CF::WGN, wn = wave % CF::WGN;

    // ---- which tile ----
    const int id = gk::xcd_remap((int)blockIdx.x, (int)gridDim.x, a.xcds);
    const int slice = id % a.slices, tile = id / a.slices;
    int bm, bn;
    {   // bands of `band` row tiles, rows fastest
        const int full = a.band * a.nbn, band = tile / full, r = tile - band * full, rows = min(a.band, a.bm_tiles - band * a.band);
        bm = band * a.band + r % rows;
        bn = r / rows;
    }
    int e, m0, m1;
    tile_rows<BM>(a, bm, e, m0, m1);
    if (m0 >= m1) return;
    const int n0 = bn * BN;
    const int kb0 = slice * a.per, kb1 = min(a.nb, kb0 + a.per);

    // ---- operand streams ----
    const uint8_t *const Bt = a.B + ((size_t)e * a.N + n0) * a.K;
    const uint8_t *const At = a.src ? a.A : a.A + (size_t)m0 * a.K;
    const float *const sat = a.src ? a.sa : a.sa + (size_t)m0 * a.nb;
    const uint32_t arows = a.src ? (uint32_t)a.a_rows : (uint32_t)(m1 - m0);
    const Rsrc rA = gk::rsrc_u(At, arows * (uint32_t)a.K), rB = gk::rsrc_u(Bt, (uint32_t)min(BN, a.N - n0) * (uint32_t)a.K);
    const Rsrc rS = gk::rsrc_u(sat, arows * (uint32_t)a.nb * 4u);
    // (a row of the tile that C does not have, or that has no source, reads zeros)
    auto arow = [&](int r) -> int { return m0 + r < m1 ? (a.src ? source(a, m0 + r) : r) : -1; };
    uint32_t va[CF::IA], vb[CF::IB], ca[CF::IA], cb[CF::IB], vs;
#pragma unroll
    for (int i = 0; i < CF::IA; i++) {
        const int row = (wave * CF::IA + i) * 8 + (lane >> 3), r = arow(row);
        ca[i] = (uint32_t)((lane & 7) ^ sw_a(row)) * 16u;
        va[i] = r < 0 ? kOOB : (uint32_t)r * (uint32_t)a.K + ca[i];
    }
#pragma unroll
    for (int i = 0; i < CF::IB; i++) {
        const int row = (wave * CF::IB + i) * 8 + (lane >> 3);
        cb[i] = (uint32_t)((lane & 7) ^ sw_b(row)) * 16u;
        vb[i] = (uint32_t)row * (uint32_t)a.K + cb[i];
    }
    {
        const int r = arow(wave * CF::RWS + lane % CF::RWS);
        vs = r < 0 ? kOOB : (uint32_t)r * (uint32_t)a.nb * 4u;
    }
    typedef __attribute__((address_space(3))) void *Lds;
    auto load = [&](int b, int slot) __attribute__((always_inline)) {
        char *const at = smem + slot * CF::SLOT;
        const uint32_t k = (uint32_t)b * 128u, left = (uint32_t)a.K - k;
#pragma unroll
        for (int i = 0; i < CF::IA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (Lds)(at + (wave * CF::IA + i) * 1024), 16, (va[i] + k) | (ca[i] < left ? 0u : kOOB), 0, 0, 0);
#pragma unroll
        for (int i = 0; i < CF::IB; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rB, (Lds)(at + BM * 128 + (wave * CF::IB + i) * 1024), 16, (vb[i] + k) | (cb[i] < left ? 0u : kOOB), 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rS, (Lds)(at + (BM + BN) * 128 + wave * 256), 4, vs + (uint32_t)b * 4u, 0, 0, 0);
    };

    // the weights' scales of the tile's columns and the slice's blocks
    for (int i = tid; i < CF::SBN * a.per; i += CF::NT) {
        const int c = i / a.per, b = kb0 + i - c * a.per, n = n0 / 128 + c;
        sbl[i] = b < kb1 && n < (a.N + 127) / 128 ? a.sb[((size_t)e * ((a.N + 127) / 128) + n) * a.nb + b] : 0.f;
    }
    // (waited for before the ring starts: its waits count the DMA's loads alone)
    __syncthreads();

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int s = 0; s < SLOTS - 1; s++) load(min(kb0 + s, kb1 - 1), s);
    const int ra = wm * CF::WTM + (lane & 15);
    const int q = lane >> 4, rb = wn * CF::WTN + 8 * ((lane & 15) >> 2) + (lane & 3);
    const float *const sbw = sbl + (CF::SBN > 1 ? wn * CF::WTN / 128 * a.per : 0);
    int slot = 0;
    for (int b = kb0; b < kb1; b++) {
        gk::wait_vm<(SLOTS - 2) * CF::NVM>();
        gk::lds_barrier();
        // (past the last block the ring loads it again, which nothing reads: the waits' counts stay)
        load(min(b + SLOTS - 1, kb1 - 1), slot == 0 ? SLOTS - 1 : slot - 1);
        const char *const pa = smem + slot * CF::SLOT, *const pb = pa + BM * 128;
        const float *const ps = reinterpret_cast<const float *>(pb + BN * 128);
        const float sb = sbw[b - kb0];
        Frag<WIDE> fb[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int row = rb + 32 * (j / 2) + 4 * (j % 2), f = sw_b(row);
            fb[j].set(*reinterpret_cast<const i32x4 *>(pb + row * 128 + ((q ^ f) << 4)),
                      *reinterpret_cast<const i32x4 *>(pb + row * 128 + (((4 + q) ^ f) << 4)));
        }
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int row = ra + 16 * i, f = sw_a(row);
            Frag<WIDE> fa;
            fa.set(*reinterpret_cast<const i32x4 *>(pa + row * 128 + ((q ^ f) << 4)),
                   *reinterpret_cast<const i32x4 *>(pa + row * 128 + (((4 + q) ^ f) << 4)));
            const float s = ps[row / CF::RWS * 64 + row % CF::RWS] * sb;
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const f32x4 d = product(fb[j], fa);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(d[r], s, acc[i][j][r]);
            }
        }
        slot = slot == SLOTS - 1 ? 0 : slot + 1;
    }
    gk::wait_vm<0>();   // (no DMA is in flight when the workgroup's LDS is given on)

    // ---- results ----
    const bool wide = a.N % 4 == 0;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + ra + 16 * i;
        if (m >= m1) continue;
        using T = std::conditional_t<F16, _Float16, float>;
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int n = n0 + wn * CF::WTN + 32 * (j / 2) + 8 * q + 4 * (j % 2);
            if (a.slices > 1) store4(a.ws + ((size_t)slice * a.M + m) * a.N, n, a.N, wide, acc[i][j]);
            else store4(static_cast<T *>(a.C) + (size_t)m * a.N, n, a.N, wide, acc[i][j]);
        }
    }
#endif
}

template <class CF, bool WIDE, bool F16> hipError_t launch(Args a, const GemmF8 &L, hipStream_t s, uint64_t *blocks)
{
    static std::atomic<uint64_t> opted{0};
    const auto kern = &k_gemm_fp8<CF, WIDE, F16>;
    a.nbn = (L.N + CF::BN - 1) / CF::BN;
    const long tiles = row_tiles(L, CF::BM);
    a.bm_tiles = (int)tiles;
    const long grid = tiles * a.nbn * a.slices;
    if (grid >= (long)1 << 31 || tiles >= (long)1 << 30) return hipErrorInvalidValue;
    const int lds = CF::lds(a.per);
    if (hipError_t e = lds_opt_in(reinterpret_cast<const void *>(kern), CF::lds(kF8MaxK / kF8Block), opted)) return e;
    *blocks = (uint64_t)grid;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(CF::NT), lds, s, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace f8

size_t gemm_fp8_ws(const GemmF8 &L) { (void)L; return 0; }

hipError_t gemm_fp8(const GemmF8 &L, hipStream_t s, uint64_t *blocks)
{
    using namespace f8;
    const Args a = args(L);
    using Base = Cfg<128, 128, 2, 2, 3>;
    return L.f16 ? launch<Base, false, true>(a, L, s, blocks) : launch<Base, true, false>(a, L, s, blocks);
}

}  // namespace rk
