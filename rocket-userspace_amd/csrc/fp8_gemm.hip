// fp8_gemm.hip — products of e4m3 codes with block scales, by tiles: C[m][n] = sum_b sa[m][b] sb[n / 128][b] (A_b B_b^T)[m][n].
//
// A stage is one block of 128 codes: the tile's rows of A and B go by DMA into a ring of LDS slots (chunks swizzled by
// their source address, so that sixteen lanes' 16-byte reads cover all banks once), with the rows' scales beside them. A wave
// multiplies its part of the tile for that block alone and adds the products, times one scale a lane, to its fp32 sums:
// one VALU operation an element and block, behind one MFMA an element block.
//
// Seven tiles, from 256 x 256 (one workgroup a CU, two slots, operands read as they are multiplied) to 32 x 64 (three a CU, four
// slots, operands read a stage ahead); plan() chooses. 4096 x 3840 x 15360 takes 224 us (2160 TFLOP/s; a large library product
// without scales reaches 2830), 8192^3 450 us (2440), 512 x 15360 x 3840 42 us, 4096 tokens of 6 of 64 experts, 2048 -> 2816, 208 us.
// A large tile's matrix units are busy 63% of the time; a workgroup alone takes 1.27 us a stage, with the chip full 1.77, and
// perfect L2s take a tenth off that. What else was measured at 4096 x 3840 x 15360, then at 247 to 251 us: 32 x 32 products 271, scales
// by a DMA of four bytes a lane 305, a second barrier a stage to free B's slot early 257, asking the L2 for the stage after the
// next 285, workgroups that stay and load the next tile's first stage in the last of theirs 265 (33 registers spilled).
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
    a.band = 8;
    return a;
}

namespace {

// Rows of the weights' tile in the order that a lane's columns become neighbours: MFMA row 4 q + r of block j is row
// 32 (j / 2) + 8 q + 4 (j % 2) + r, so that blocks 2 p and 2 p + 1 give a lane eight neighbours. The swizzle of a tile row:
// sixteen rows of an MFMA operand cover every pair of row parity and slot once.
[[maybe_unused]] __device__ constexpr int sw_a(int row) { return (row >> 1) & 7; }
[[maybe_unused]] __device__ constexpr int sw_b(int row) { return ((row >> 1) & 1) | ((row >> 2) & 6); }

template <int BM_, int BN_, int WGM_, int WGN_, int SLOTS_, int WPE_, bool PIPE_> struct Cfg {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, SLOTS = SLOTS_, WPE = WPE_;
    static constexpr bool PIPE = PIPE_;   // operands read a stage ahead
    static constexpr int NW = WGM * WGN, NT = 64 * NW, WTM = BM / WGM, WTN = BN / WGN, TM = WTM / 16, TN = WTN / 16;
    static constexpr int IA = BM / NW / 8, IB = BN / NW / 8;   // DMA instructions a wave and stage
    static constexpr int CH = 4 * NT / BM;                     // stages whose scales of A are loaded at once, four a lane
    static constexpr int SLOT = (BM + BN) * 128;
    static constexpr int NVM = IA + IB;
    static constexpr int SBN = (BN + 127) / 128;               // blocks of 128 columns
    static_assert(IA >= 1 && IB >= 1 && TN % 2 == 0 && TM > 1 && (WTN == 128 || 128 % WTN == 0), "tile");
    static_assert(NT % BM == 0, "whole lanes a row");
    static constexpr int lds(int per) { return SLOTS * SLOT + 2 * BM * CH * 4 + BM * 4 + SBN * per * 4; }
};

template <class CF, bool WIDE, bool F16> __global__ __launch_bounds__(CF::NT) __attribute__((amdgpu_waves_per_eu(CF::WPE))) void k_gemm_fp8(const Args a)
{
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BM = CF::BM, BN = CF::BN, TM = CF::TM, TN = CF::TN, SLOTS = CF::SLOTS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *const sal = reinterpret_cast<float *>(smem + SLOTS * CF::SLOT), *const sbl = sal + 2 * BM * CF::CH + BM;
    int *const none = reinterpret_cast<int *>(sal + 2 * BM * CF::CH);   // rows of C that have no source
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / CF::WGN, wn = wave % CF::WGN;

    // ---- which tile ----
    // Of each 8 * 16 workgroups in the order of their launch an XCD has 16 neighbours, which share what its L2 holds, and
    // all XCDs are near each other in the last cache's. (Runs of an eighth of all on an XCD instead: experts' tiles that
    // there are not, the last ones, left XCDs idle, and 4096 tokens of 6 of 64 experts took 243 us, not 216; 4096 x 3840 x 15360 232, not 227.)
    constexpr int kNear = 16, kRun = 8 * kNear;
    const int run0 = (int)blockIdx.x / kRun * kRun, id = run0 + gk::xcd_remap((int)blockIdx.x - run0, min(kRun, (int)gridDim.x - run0), 8);
    // (a slice's tiles are neighbours, which share rows of A and B; a tile's slices share nothing: 128 x 15360 x 3840 in four slices
    // 18.9 us so, 19.8 with a tile's slices side by side)
    const int tiles = (int)gridDim.x / a.slices, slice = id / tiles, tile = id - slice * tiles;
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
    constexpr int LR = CF::NT / BM;   // lanes that load a row's scales
    // the weights' scales of the tile's columns and the slice's blocks
    auto scale_b = [&](int i) __attribute__((always_inline)) {
        const int c = i / a.per, b = kb0 + i - c * a.per, n = n0 / 128 + c;
        return a.sb[((size_t)e * ((a.N + 127) / 128) + min(n, (a.N - 1) / 128)) * a.nb + min(b, kb1 - 1)];   // (past the last: not used)
    };
    for (int i = tid + CF::NT; i < CF::SBN * a.per; i += CF::NT) sbl[i] = scale_b(i);
    // Where K ends inside its last block, the chunks past K read zeros from that block on.
    const int part = a.K % 128 ? a.nb - 1 : -1;
    const uint32_t left = (uint32_t)a.K % 128u;
    uint32_t va[CF::IA], vb[CF::IB], ca[CF::IA], cb[CF::IB], vs;
#pragma unroll
    for (int i = 0; i < CF::IB; i++) {
        const int row = (wave * CF::IB + i) * 8 + (lane >> 3);
        cb[i] = (uint32_t)((lane & 7) ^ sw_b(row)) * 16u;
        vb[i] = ((uint32_t)row * (uint32_t)a.K + cb[i]) | (kb0 != part || cb[i] < left ? 0u : kOOB);
    }
    typedef __attribute__((address_space(3))) void *Lds;
    char *const pb0 = smem + SLOTS * BM * 128;   // A's slots, then B's
    // Instruction i of the IA + IB that load a stage, whose codes start at byte k of a row.
    auto load1 = [&](int i, int k, int slot) __attribute__((always_inline)) {
        if (i < CF::IA)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (Lds)(smem + slot * BM * 128 + (wave * CF::IA + i) * 1024), 16, va[i], k, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rB, (Lds)(pb0 + slot * BN * 128 + (wave * CF::IB + i - CF::IA) * 1024), 16, vb[i - CF::IA], k, 0, 0);
    };
    auto first_b = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = CF::IA; i < CF::NVM; i++) load1(i, __builtin_amdgcn_readfirstlane(kb0 * 128), 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // Rows of A that the lane loads from, those of the tile's codes and the one of its scales; -1: a row of the tile that C does not have,
    // or that has no source, which reads zeros. All loads of `src` are issued at once (each behind a condition of its own is
    // waited for), and the first stage's weights are on their way behind them.
    int ar[CF::IA + 1];
    auto trow = [&](int i) __attribute__((always_inline)) { return i < CF::IA ? (wave * CF::IA + i) * 8 + (lane >> 3) : tid / LR; };
    if (a.src) {
#pragma unroll
        for (int i = 0; i <= CF::IA; i++) ar[i] = a.src[min(m0 + trow(i), m1 - 1)];
        __builtin_amdgcn_sched_barrier(0);
        first_b();
    } else {
        first_b();
#pragma unroll
        for (int i = 0; i <= CF::IA; i++) ar[i] = trow(i);
    }
#pragma unroll
    for (int i = 0; i <= CF::IA; i++) ar[i] = m0 + trow(i) < m1 && (unsigned)ar[i] < arows ? ar[i] : -1;
#pragma unroll
    for (int i = 0; i < CF::IA; i++) {
        ca[i] = (uint32_t)((lane & 7) ^ sw_a(trow(i))) * 16u;
        va[i] = ar[i] < 0 ? kOOB : (uint32_t)ar[i] * (uint32_t)a.K + ca[i];
    }
    if (a.src && tid % LR == 0) none[tid / LR] = ar[CF::IA] < 0;
    vs = ar[CF::IA] < 0 ? kOOB : ((uint32_t)ar[CF::IA] * (uint32_t)a.nb + (uint32_t)(tid % LR) * 4u) * 4u;
    // The rows' scales of CH stages from stage CH c of the slice on, through registers (a DMA of four bytes a lane, once a
    // stage, cost a fifth of the time), into the half of their LDS that the stages before do not read.
    auto scales = [&](int c) __attribute__((always_inline)) {
        return __builtin_bit_cast(f32x4, gk::ld16(rS, vs + (uint32_t)(kb0 + CF::CH * c) * 4u));   // (zeros past the last row's)
    };
    auto keep = [&](f32x4 v, int c) __attribute__((always_inline)) {
        float *const at = sal + ((c & 1) * CF::CH + tid % LR * 4) * BM + tid / LR;   // ([stage][row]: sixteen rows are neighbours)
#pragma unroll
        for (int i = 0; i < 4; i++) at[i * BM] = v[i];
    };
    // Loads of block b (past the slice's last: the last again, which nothing uses, so that the waits' counts stay).
    auto block = [&](int b) __attribute__((always_inline)) {
        b = min(b, kb1 - 1);
        if (b == part) {
#pragma unroll
            for (int i = 0; i < CF::IA; i++) va[i] |= ca[i] < left ? 0u : kOOB;
#pragma unroll
            for (int i = 0; i < CF::IB; i++) vb[i] |= cb[i] < left ? 0u : kOOB;
        }
        return __builtin_amdgcn_readfirstlane(b * 128);
    };
    {
        __builtin_amdgcn_sched_barrier(0);   // (addresses first: one computed behind the loads can wait for their registers)
        const f32x4 s0 = scales(0);
        const float b0 = scale_b(min(tid, CF::SBN * a.per - 1));
        // the first stages; the scales' loads stand before theirs, so that a wait for the scales leaves them on their way
#pragma unroll
        for (int s = 0; s < (CF::PIPE ? SLOTS : SLOTS - 1); s++) {
            const int k = block(kb0 + s);
#pragma unroll
            for (int i = 0; i < (s ? CF::NVM : CF::IA); i++) load1(i, k, s);
        }
        keep(s0, 0);
        if (tid < CF::SBN * a.per) sbl[tid] = b0;
    }

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int ra = wm * CF::WTM + (lane & 15);
    const int q = lane >> 4, rb = wn * CF::WTN + 8 * ((lane & 15) >> 2) + (lane & 3);
    const float *const sbw = sbl + (CF::SBN > 1 ? wn * CF::WTN / 128 * a.per : 0), *const saw = sal + ra;
    auto codes = [&](const char *plane, int row, int sw) __attribute__((always_inline)) {
        return Codes{*reinterpret_cast<const i32x4 *>(plane + row * 128 + ((q ^ sw) << 4)),
                     *reinterpret_cast<const i32x4 *>(plane + row * 128 + (((4 + q) ^ sw) << 4))};
    };
    auto codes_a = [&](int slot, int i) __attribute__((always_inline)) { return codes(smem + slot * BM * 128, ra + 16 * i, sw_a(ra + 16 * i)); };
    auto codes_b = [&](int slot, int j) __attribute__((always_inline)) {
        const int row = rb + 32 * (j / 2) + 4 * (j % 2);
        return codes(pb0 + slot * BN * 128, row, sw_b(row));
    };
    auto factors = [&](float (&sc)[TM], float &sb, unsigned u) __attribute__((always_inline)) {
        const float *const ps = saw + u % (2 * CF::CH) * BM;
        sb = sbw[u];
#pragma unroll
        for (int i = 0; i < TM; i++) sc[i] = ps[16 * i];
    };
    // A product is added kLag products later, when the matrix unit has it done. A stage's loads are issued between the
    // products of its first half: at once they would hold the wave up, since a CU takes some 43 bytes a clock.
    constexpr int NP = TM * TN, kLag = NP >= 8 ? 3 : 2;
    constexpr int kEvery = NP >= 2 * CF::NVM ? NP / (2 * CF::NVM) : 1, kEach = (CF::NVM * kEvery + NP - 1) / NP;
    auto spread = [&](int t, int k, int slot) __attribute__((always_inline)) {
        if (t % kEvery) return;
#pragma unroll
        for (int e = 0; e < kEach; e++)
            if (t / kEvery * kEach + e < CF::NVM) load1(t / kEvery * kEach + e, k, slot);
    };
    auto add = [&](f32x4 &c, const f32x4 &d, float s) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; r++) c[r] = fmaf(d[r], s, c[r]);
    };
    f32x4 next = {0.f, 0.f, 0.f, 0.f};
    const unsigned n = (unsigned)(kb1 - kb0);
    if constexpr (CF::PIPE) {
        // A stage's operands are read from LDS while the stage before is multiplied from registers, so that the products
        // wait for no read behind a barrier.
        Codes xa[2][TM], xb[2][TN];
        float sc[2][TM], sb[2];
        gk::wait_vm<(SLOTS - 1) * CF::NVM>();
        gk::lds_barrier();
#pragma unroll
        for (int j = 0; j < TN; j++) xb[0][j] = codes_b(0, j);
#pragma unroll
        for (int i = 0; i < TM; i++) xa[0][i] = codes_a(0, i);
        factors(sc[0], sb[0], 0);
        auto stage = [&](auto S, unsigned u) __attribute__((always_inline)) {
            constexpr int slot = S, after = (slot + 1) % SLOTS, now = slot % 2, then = 1 - now;
            gk::wait_vm<(SLOTS - 2) * CF::NVM>();
            if (u % CF::CH == CF::CH / 2) keep(next, (int)(u / CF::CH) + 1);
            gk::lds_barrier();
            if (u % CF::CH == 0) next = scales((int)(u / CF::CH) + 1);
            const int k = block(kb0 + (int)u + SLOTS);
            factors(sc[then], sb[then], min(u + 1, n - 1));
            Frag<WIDE> fb[TN], fa;
#pragma unroll
            for (int j = 0; j < TN; j++) fb[j].set(xb[now][j].lo, xb[now][j].hi);
            f32x4 d[kLag + 1];
#pragma unroll
            for (int t = 0; t < NP + kLag; t++) {
                if (t < NP) {
                    if (t % TN == 0) fa.set(xa[now][t / TN].lo, xa[now][t / TN].hi);
                    d[t % (kLag + 1)] = product(fb[t % TN], fa);
                    spread(t, k, slot);
                    if (t < TN) xb[then][t] = codes_b(after, t);
                    else if (t < TN + TM) xa[then][t - TN] = codes_a(after, t - TN);
                }
                if (t >= kLag) {
                    const int v = t - kLag;
                    if (v % TN == 0) sc[now][v / TN] *= sb[now];
                    add(acc[v / TN][v % TN], d[v % (kLag + 1)], sc[now][v / TN]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        static_assert(NP >= TN + TM && SLOTS % 2 == 0, "a stage has a product for each read of the next");
        for (unsigned u = 0; u < n; u += SLOTS)
            gk::static_for<SLOTS>([&](auto S) __attribute__((always_inline)) {
                if (u + S < n) stage(S, u + S);
            });
    } else {
        auto stage = [&](auto S, unsigned u) __attribute__((always_inline)) {
            constexpr int slot = S, free = (slot + SLOTS - 1) % SLOTS;
            gk::wait_vm<(SLOTS - 2) * CF::NVM>();
            if (u % CF::CH == CF::CH / 2) keep(next, (int)(u / CF::CH) + 1);
            gk::lds_barrier();
            if (u % CF::CH == 0) next = scales((int)(u / CF::CH) + 1);
            const int k = block(kb0 + (int)u + SLOTS - 1);
            Frag<WIDE> fa[2], fb[TN];
            float sc[TM], sb;
            auto set = [](Frag<WIDE> &f, const Codes &c) __attribute__((always_inline)) { f.set(c.lo, c.hi); };
            set(fa[0], codes_a(slot, 0));
#pragma unroll
            for (int j = 0; j < TN; j++) set(fb[j], codes_b(slot, j));
            factors(sc, sb, u);
            f32x4 d[kLag + 1];
            // (ahead of a wave that still reads its operands: 1 to 2% at 256 x 256)
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < NP + kLag; t++) {
                if (t < NP) {
                    const int i = t / TN, j = t % TN;
                    if (j == 0 && i + 1 < TM) set(fa[(i + 1) & 1], codes_a(slot, i + 1));
                    d[t % (kLag + 1)] = product(fb[j], fa[i & 1]);
                    spread(t, k, free);
                }
                if (t >= kLag) {
                    const int v = t - kLag;
                    if (v % TN == 0) sc[v / TN] *= sb;
                    add(acc[v / TN][v % TN], d[v % (kLag + 1)], sc[v / TN]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        };
        for (unsigned u = 0; u < n; u += SLOTS)
            gk::static_for<SLOTS>([&](auto S) __attribute__((always_inline)) {
                if (u + S < n) stage(S, u + S);
            });
    }
    gk::wait_vm<0>();   // (no DMA is in flight when the workgroup's LDS is given on)

    // ---- results ----
    using T = std::conditional_t<F16, _Float16, float>;
    const int n1 = n0 + wn * CF::WTN + 8 * q;
    if (a.slices > 1) {
        const int stride = (a.N + 3) & ~3;   // (columns from N on are zeros: the weights' rows there are)
        float *const ws = a.ws + (size_t)slice * a.M * stride;
#pragma unroll
        for (int i = 0; i < TM; i++)
            if (m0 + ra + 16 * i < m1)
#pragma unroll
                for (int j = 0; j < TN; j++) store4(ws + (size_t)(m0 + ra + 16 * i) * stride, n1 + 32 * (j / 2) + 4 * (j % 2), a.N, true, acc[i][j]);
        return;
    }
    const bool wide = a.N % 4 == 0;
    int gone = 0;   // rows that are not stored: past the last, or without a source
#pragma unroll
    for (int i = 0; i < TM; i++) gone |= (a.src ? none[ra + 16 * i] : m0 + ra + 16 * i >= m1) << i;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + ra + 16 * i;
        if (gone >> i & 1) continue;
        T *const row = static_cast<T *>(a.C) + (size_t)m * a.N;
        if (wide) {
#pragma unroll
            for (int j = 0; j < TN; j += 2) store8(row, n1 + 16 * j, a.N, acc[i][j], acc[i][j + 1]);
        } else {
#pragma unroll 1
            for (int j = 0; j < 4 * TN; j++) {   // (any element of the sums by a chain of selects: 4096 x 3840 x 15359 327 us, x 15360 225)
                float v = 0.f;
#pragma unroll
                for (int u = 0; u < 4 * TN; u++) v = j == u ? acc[i][u / 4][u % 4] : v;
                const int n = n1 + 32 * (j / 8) + j % 8;
                if (n < a.N) row[n] = (T)v;
            }
        }
    }
    // Rows without a source are zeros; their sums are zeros times the weights, NaN where those hold a NaN or an infinite scale. (Zeroed sums
    // instead: 242 us for 4096 tokens of 6 of 64 experts, 208 so.)
    if (a.src && gone) {
#pragma unroll 1
        for (int i = 0; i < TM; i++) {
            const int m = m0 + ra + 16 * i;
            if (!(gone >> i & 1) || m >= m1) continue;
            T *const row = static_cast<T *>(a.C) + (size_t)m * a.N;
#pragma unroll 1
            for (int j = 0; j < 4 * TN; j++) {
                const int n = n1 + 32 * (j / 8) + j % 8;
                if (n < a.N) row[n] = (T)0.f;
            }
        }
    }
#endif
}

// The slices' sums, in order.
template <bool F16> __global__ __launch_bounds__(256) void k_join_fp8(const Args a)
{
    const int stride = (a.N + 3) & ~3, quads = stride / 4;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x, plane = (size_t)a.M * stride;
    if (t >= (size_t)a.M * quads) return;
    f32x4 v = *reinterpret_cast<const f32x4 *>(a.ws + 4 * t);
    for (int s = 1; s < a.slices; s++) v += *reinterpret_cast<const f32x4 *>(a.ws + s * plane + 4 * t);
    using T = std::conditional_t<F16, _Float16, float>;
    const int m = (int)(t / quads), n = (int)(t - (size_t)m * quads) * 4;
    store4(static_cast<T *>(a.C) + (size_t)m * a.N, n, a.N, a.N % 4 == 0, v);
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
    if (hipError_t e = hipGetLastError()) return e;
    if (a.slices > 1) {
        const size_t join = ((size_t)a.M * ((a.N + 3) / 4) + 255) / 256;
        hipLaunchKernelGGL((k_join_fp8<F16>), dim3((unsigned)join), dim3(256), 0, s, a);
        *blocks += join;
    }
    return hipGetLastError();
}

}  // namespace
}  // namespace f8

namespace {

using namespace f8;

// The tiles, what a CU holds of one (cap), and what a stage takes in us: t1 with one workgroup a CU, tc with every CU full (cap 1:
// with few workgroups, and with one a CU); `fixed` is the launch, the first loads and the results, `more` what each further round of
// workgroups adds of these. Fitted to 390 products (17 to 8192 rows, and 8 to 128 experts', K and N from 512 to 15360) with every
// tile and 1 to 8 slices; of 394 timed with the kernels as they are, the chosen ones took 0.9% (fp32 results: 1.1%) longer than the fastest on average,
// 21% at most.
struct Tile {
    int bm, bn, cap;
    float fixed, more, t1, tc;
};
enum Kind { kT256, kT128, kT128Deep, kT64x128, kT64x128Deep, kT64, kT32, kKinds, kRows = kKinds };
constexpr Tile kNarrow[kKinds] = {{256, 256, 1, 8.32f, 4.70f, 0.79f, 1.79f}, {128, 128, 2, 4.89f, 2.67f, 0.64f, 1.11f}, {128, 128, 1, 5.23f, 5.89f, 0.40f, 0.53f},
                                  {64, 128, 2, 3.39f, 2.26f, 0.50f, 0.84f}, {64, 128, 1, 4.14f, 4.10f, 0.29f, 0.37f}, {64, 64, 2, 3.70f, 3.10f, 0.25f, 0.31f},
                                  {32, 64, 3, 3.42f, 2.23f, 0.21f, 0.28f}};
// (widened: no tile of 256, whose codes' fp16 does not fit the registers, none of 128 with four slots, which is no faster, and
// none of 64 x 128, a stage of which takes 0.61 to 0.68: two workgroups of 64 x 64 on a CU have as much done in 0.67)
constexpr Tile kWide[kKinds] = {{}, {128, 128, 2, 4.38f, 6.40f, 1.04f, 1.65f}, {}, {}, {}, {64, 64, 2, 3.51f, 3.01f, 0.41f, 0.67f},
                                {32, 64, 3, 4.05f, 3.14f, 0.35f, 0.64f}};
// Bytes a us: memory, what the CUs take out of the L2s. What joining slices takes: us, and us a slice and value.
constexpr float kCus = 256.f, kMem = 5.2e6f, kL2 = 14e6f;
constexpr float kJoinFixed = 2.1f, kJoin = 1.7e-6f;

// The kernel and the slices of K that are expected to take the least time.
void plan(GemmF8 &L, bool split)
{
    const Tile *const tiles = L.f16 ? kNarrow : kWide;
    const int nb = f8_blocks(L.K);
    const float used = L.off ? (float)std::min(L.n_expert, L.M) : 1.f, mean = (float)L.M / used;
    const float mem = used * (float)L.N * (float)L.K / kMem;
    float best = INFINITY;
    for (int k = 0; k < kKinds; k++) {
        const Tile &t = tiles[k];
        if (!t.bm) continue;
        const float rows = L.off ? used * std::max(1.f, mean / t.bm + 0.5f) : ceilf(mean / t.bm);
        const float w1 = rows * (float)((L.N + t.bn - 1) / t.bn), room = kCus * t.cap;
        for (int s : {1, 2, 3, 4, 6, 8}) {
            if (s > 1 && (!split || L.off || nb < 3 * s || w1 * (s - 1) > room)) break;
            const int per = (nb + s - 1) / s;
            const float w = w1 * s, full = t.cap > 1 ? std::max(0.f, (std::min(w, room) / kCus - 1.f) / (t.cap - 1)) : std::min(1.f, w / kCus);
            const float rounds = ceilf(w / room), stages = rounds * per * (t.t1 + (t.tc - t.t1) * full) + (rounds - 1.f) * t.more;
            const float comp = std::max(stages, w * per * 128.f * (t.bm + t.bn) / kL2);
            float us = t.fixed + sqrtf(comp * comp + mem * mem);
            if (s > 1) us += kJoinFixed + s * (float)L.M * (float)L.N * kJoin;
            if (us < best) best = us, L.kind = k, L.slices = (nb + per - 1) / per;
        }
    }
    const float rows = gemm_fp8_rows_us(L);
    if (rows < best) L.kind = kRows, L.slices = 1;
}

template <class CF> hipError_t start(const Args &a, const GemmF8 &L, hipStream_t s, uint64_t *blocks)
{
    return L.f16 ? launch<CF, false, true>(a, L, s, blocks) : launch<CF, true, false>(a, L, s, blocks);
}

}  // namespace

size_t gemm_fp8_plan(GemmF8 &L)
{
    plan(L, true);
    return L.slices > 1 ? (size_t)L.slices * L.M * ((L.N + 3) & ~3) * sizeof(float) : 0;
}

hipError_t gemm_fp8(const GemmF8 &L0, hipStream_t s, uint64_t *blocks)
{
    GemmF8 L = L0;
    if (L.slices > 1 && !L.ws) plan(L, false);
    Args a = args(L);
    a.ws = L.ws;
    a.per = (a.nb + L.slices - 1) / L.slices;
    a.slices = L.slices;
    switch (L.kind) {
    case kT256: return launch<Cfg<256, 256, 2, 4, 2, 2, false>, false, true>(a, L, s, blocks);
    case kT128: return start<Cfg<128, 128, 2, 2, 2, 2, false>>(a, L, s, blocks);
    case kT128Deep: return launch<Cfg<128, 128, 2, 2, 4, 1, true>, false, true>(a, L, s, blocks);
    case kT64x128: return launch<Cfg<64, 128, 2, 2, 2, 2, true>, false, true>(a, L, s, blocks);
    case kT64x128Deep: return launch<Cfg<64, 128, 2, 2, 4, 2, true>, false, true>(a, L, s, blocks);
    case kT64: return start<Cfg<64, 64, 2, 2, 4, 2, true>>(a, L, s, blocks);
    case kT32: return start<Cfg<32, 64, 1, 2, 4, 2, true>>(a, L, s, blocks);
    default: return gemm_fp8_rows(L, s, blocks);
    }
}

}  // namespace rk
