// serve_tiles.hip — attention of many query rows over the 4-bit cache, and over fp16 keys under a window.
//
// One workgroup = 4 waves = 128 query rows of a KV head (the tokens of all its query heads in a row, so
// that they share each tile), a wave 32 rows. The key axis goes by tiles of 64 keys, those alone that some
// row sees: the sinks' tiles, then from the first window's to the last token's. K tiles [64][D] and V^T
// tiles [D][64] lie in LDS as halves, two of each. fp16 keys arrive by buffer-load DMA. Codes arrive in
// registers a tile ahead and are widened between the MFMAs (two VALU operations a value, shared by
// the 128 rows), then written to LDS, a key as the two halves that hold it exactly (kv4_widen.h), one K tile of each.
//
// The loop is software-pipelined: an iteration runs the previous tile's PV products with this tile's
// score arithmetic between them, then the next tile's QK products with this tile's exponentials between
// them; K runs a tile ahead of V^T. Scores are transposed, S^T = K Q^T (v_mfma_f32_32x32x16_f16), so a lane
// holds one row's scores and P stays in registers: rounded to fp16 (over codes as two halves) and swapped between the
// half-waves it is the second product's operand. O is rescaled only when some running maximum grows by more than 5.5 (log2
// units).
//
// Roundings beside the result's: over halves the weights' to fp16 (summed as rounded); over codes the values', to the halves
// that the cache's reading gives. Scores, maxima, sums, outputs and shares' outputs are fp32. Measured: 2048 tokens under a
// window of 1024, 16 / 8 heads of 256, 55.0 us (630 TFLOP/s); 512 over 16384 fp16 keys of those heads 155 (870); 512 over 4096
// codes 88 (365; with keys and weights rounded to one half each 69, and results 4.0e-4 of their size off, not 2.8e-4); 2048
// over 8192 fp16 keys, 32 / 8 heads of 128, 274 (880). Heads of 256 have one wave a SIMD, which issues in order: by counters
// a tile of halves is 240 VALU operations of 4 cycles and 64 MFMAs of 32 in 4900 cycles, an instruction issued in 46% of
// them, 28% waiting to issue and 26% for LDS, loads or the other waves (LDS itself is busy a fifth of the time). Of codes a tile
// is twice the products and the widening: 820 VALU operations and 130 MFMAs in 9350 cycles, an instruction issued in 58%.
#include "kv4_widen.h"
#include "lds_optin.h"
#include "serve.h"
#include "softcap.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace rk {
namespace {

typedef int      i32x2  __attribute__((ext_vector_type(2)));
typedef int      i32x4  __attribute__((ext_vector_type(4)));
typedef float    f32x2  __attribute__((ext_vector_type(2)));
typedef float    f32x4  __attribute__((ext_vector_type(4)));
typedef float    f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4  __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t Rsrc;

constexpr uint32_t kOOB = 0x80000000u;   // an offset past every range: loads return 0
constexpr int BQ = 128, BK = 64, NW = 4;

[[maybe_unused]] __device__ __forceinline__ Rsrc rsrc(const void *base, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void wait_vm0()
{
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));
#endif
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// (a wave's LDS operations are served in order: the compiler alone has to keep it)
__device__ __forceinline__ void wave_lds_order()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// eight halves at any 2-byte address
struct __attribute__((packed, aligned(2))) Halves8 { i32x4 v; };

struct TileArgs {
    ServeAttn a;
    int nsplit, nqb;   // shares of the key tiles; row blocks of a KV head
    int len, per;      // rows of a run that is cut into blocks of BQ: a head's T or all of a KV head's; blocks of a run
    float *part;       // [split][row][dv] outputs (divided by the split's sum), then [split][row] (max, sum); rounded to fp16
                       // they would be a third rounding beside the weights' and the result's
};

// D: 64, 128 or 256. 16-byte chunk c of an LDS row lies at slot c ^ x(row): the sixteen lanes that one
// LDS cycle serves (consecutive rows, one chunk) hit all banks once.
template <int D> struct Cfg {
    static constexpr int KC = D / 16;            // score MFMA steps
    static constexpr int KCPR = D / 8;           // 16-byte chunks a K row
    static constexpr int KINS = D / 32, VINS = D / 32;   // DMA instructions a wave and tile
    static constexpr int KBYTES = BK * D * 2, VBYTES = D * BK * 2, STAGE = KBYTES + VBYTES;
    static constexpr int DB = D / 32;            // 32-row blocks of output dims
    static constexpr int SUMS = BK * 16;         // 4-bit: the minimums of a tile's keys, eight groups each
    static constexpr int LDS = 2 * STAGE + SUMS + 16;   // + the flag of a tile with non-finite values
    // 4-bit: a thread's runs of a tile's key codes and value codes, and the 16-byte writes they make
    static constexpr int ITEMS = D == 256 ? 2 : 1, KW = D == 64 ? 2 : 4, VD = D == 64 ? 2 : 4;
    static constexpr int KU = ITEMS * KW, VU = ITEMS * VD;
    __device__ static int kx(int row) { return (D * 2) % 256 == 0 ? (row & 15) : ((row >> 1) & 7); }
};
__device__ __forceinline__ int vx(int row) { return (row >> 1) & 7; }   // V^T rows: 128 bytes

// Where keys and values come from: fp16 rows by DMA; the same with V^T rows that are no whole 16-byte chunks, whose values
// go through registers; codes.
enum Src { kHalves, kRagged, kCodes };

template <int D, Src SRC, Cap CAP>
__global__ __launch_bounds__(256, D <= 64 || (D == 128 && SRC != kCodes) ? 2 : 1) void k_serve_tiles(const TileArgs ta)
{
    constexpr bool C4 = SRC == kCodes, RV = SRC == kRagged, CAPPED = CAP != kUncapped;
    const ServeAttn &a = ta.a;
    using CF = Cfg<D>;
    constexpr int KC = CF::KC, KCPR = CF::KCPR, DB = CF::DB;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    [[maybe_unused]] _Float16 *const mins = reinterpret_cast<_Float16 *>(smem + 2 * CF::STAGE);   // [key][8]
    int *const bad_tile = reinterpret_cast<int *>(smem + 2 * CF::STAGE + CF::SUMS);
    // Halves: two slots of a K tile and a V^T tile. Codes: one K tile as the halves that its products take first and second
    // (kv4_widen.h), and two V^T tiles.
    auto k_tile = [&](int slot) __attribute__((always_inline)) { return C4 ? smem + slot * CF::KBYTES : smem + slot * CF::STAGE; };
    auto v_tile = [&](int slot) __attribute__((always_inline)) { return C4 ? smem + 2 * CF::KBYTES + slot * CF::VBYTES : smem + slot * CF::STAGE + CF::KBYTES; };

    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int T = a.n_tokens, kvh = a.n_head / a.gqa;
    // Workgroup w runs on XCD w % 8; each XCD gets a contiguous range of logical ids, and consecutive ids are
    // the row blocks that read the same keys.
    int qb, hk, zs, s;
    {
        const int total = (int)gridDim.x, w = (int)blockIdx.x;
        const int xcd = w % 8, idx = w / 8, per = total / 8, rem = total % 8;
        int lid = xcd * per + (xcd < rem ? xcd : rem) + idx;
        qb = ta.nqb - 1 - lid % ta.nqb;   // the last rows, which see the most keys, first
        lid /= ta.nqb;
        zs = lid % ta.nsplit;
        lid /= ta.nsplit;
        hk = lid % kvh;
        s = lid / kvh;
    }
    const int n = a.seq_len ? a.seq_len[s] : a.max_kv;
    const bool served = n >= 1 && n <= a.max_kv;
    // the block's rows r0 .. r1 of the KV head's (head r / T of it, token r % T); the lane's row and its position
    const int run0 = qb / ta.per * ta.len, r0 = run0 + qb % ta.per * BQ, r1 = min(run0 + ta.len, r0 + BQ) - 1;
    const int r = r0 + wave * 32 + l32;
    const bool qok = r <= r1;
    const bool one = r0 / T == r1 / T;
    const int p_lo = n - T + (one ? r0 % T : 0), p_hi = n - T + (one ? r1 % T : T - 1);
    const int pos = n - T + r % T;
    const size_t row0 = ((size_t)s * a.n_head + (size_t)hk * a.gqa) * T;

    // the tiles that some row of the block sees, v -> tile: the sinks', then from the first window's on
    const int first = a.window ? max(0, p_lo - a.window + 1) : 0, sinks = min(a.sinks, first);
    const int ns = (sinks + BK - 1) / BK, f0 = max(first / BK, ns);
    const int count = served && p_hi >= 0 ? ns + p_hi / BK - f0 + 1 : 0;
    const int tps = (count + ta.nsplit - 1) / ta.nsplit;
    const int kb0 = min(zs * tps, count), kb1 = min(count, kb0 + tps);
    auto key_of = [&](int kb) __attribute__((always_inline)) { return (kb < ns ? kb : kb - ns + f0) * BK; };
    // every row of the block sees every key of the tile
    auto whole = [&](int key0) __attribute__((always_inline)) {
        return key0 + BK - 1 <= p_lo && (!a.window || key0 > p_hi - a.window || key0 + BK <= a.sinks);
    };
    // no row of the block sees the key
    auto dead = [&](int key) __attribute__((always_inline)) { return (bool)((key > p_hi) | ((key < first) & (key >= sinks))); };
    const int behind = a.window ? pos - a.window : -1;   // the last key behind the row's window
    auto sees = [&](int key) __attribute__((always_inline)) { return (bool)((key <= pos) & ((key > behind) | (key < a.sinks))); };

    // the lane's query row as the B operand of the score MFMAs: step c takes dims 16 c + 8 hh .. + 8 (in the order in
    // which widened codes lie)
    f16x8 qf[KC];
    {
        const _Float16 *qrow = a.Q + (row0 + min(r, r1)) * a.dk + 8 * hh;   // (rows behind the last repeat it)
#pragma unroll
        for (int c = 0; c < KC; c++) {
            f16x8 x = *reinterpret_cast<const f16x8 *>(qrow + min(16 * c, a.dk - 16));
            if (16 * c >= a.dk || a.scale == 0.f) x = f16x8{};
            if (a.scale < 0.f) x = -x;
            qf[c] = C4 ? kv4_query_order(x) : x;
        }
    }
    // 4-bit: the query's sums over the groups, first halves in half-wave 0 and second ones in 1, as the operand that meets the
    // groups' minimums
    [[maybe_unused]] f16x8 qsum = {};
    [[maybe_unused]] float qback = 1.f;
    [[maybe_unused]] bool back = false;
    if constexpr (C4) {
        float sum[D / 32], most = 0.f;
#pragma unroll
        for (int g = 0; g < D / 32; g++) {
            const float own = kv4_sum(qf[2 * g + 1], kv4_sum(qf[2 * g], 0.f));
            sum[g] = own + __shfl_xor(own, 32, 64);
            most = fmaxf(most, fabsf(sum[g]));
        }
        const int e = kv4_sum_exponent(most);
        qback = __builtin_amdgcn_ldexpf(1.f, e);
        back = __any(e != 0);
#pragma unroll
        for (int g = 0; g < D / 32; g++) {
            const f16x2 h = kv4_sum_halves(sum[g], e);
            qsum[g] = hh ? h[1] : h[0];
        }
        if (D < 256 && tid < BK) *reinterpret_cast<i32x4 *>(mins + 8 * tid) = i32x4{0, 0, 0, 0};   // (groups that there are not)
    }

    // ---- tiles into LDS: K tile at smem + slot * STAGE, V^T tile right behind it ----
    // fp16: DMA. Lane slot g of a tile -> (row, chunk), the global chunk the swizzled one; an instruction moves
    // 256 / KCPR rows on where those are a multiple of the swizzle's period.
    constexpr bool KSEP = 256 % KCPR == 0 && (256 / KCPR) % 16 == 0;
    constexpr int KN = KSEP ? 1 : CF::KINS;
    [[maybe_unused]] uint32_t kvo[KN], vvo = 0, kstep = 0, vstep = 0;
    [[maybe_unused]] int vkey = 0, vrow = 0;
    [[maybe_unused]] const _Float16 *Kh = nullptr, *Vh = nullptr;
    if constexpr (!C4) {
#pragma unroll
        for (int i = 0; i < KN; i++) {
            const int g = (i * NW + wave) * 64 + lane, row = g / KCPR, lc = (g % KCPR) ^ CF::kx(row);
            kvo[i] = lc * 8 < a.dk ? (uint32_t)(row * a.dk + lc * 8) * 2u : kOOB;
        }
        const int g = wave * 64 + lane, row = g >> 3, lc = (g & 7) ^ vx(row);
        vvo = (uint32_t)((long)row * a.stride + lc * 8) * 2u;
        vkey = lc * 8;
        vrow = row;
        kstep = (uint32_t)((256 / KCPR) * a.dk * 2);
        vstep = (uint32_t)(32 * a.stride * 2);
        Kh = a.Kf + (size_t)hk * a.k_hs;
        Vh = a.Vf + (size_t)hk * a.dv * a.stride;
    }
    auto dma_k = [&](int kb, int slot) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int k0 = key_of(kb);
        const Rsrc rk = rsrc(Kh + (size_t)k0 * a.dk, (uint32_t)((long)max(n - k0, 0) * a.dk * 2));
        char *ks = k_tile(slot);
#pragma unroll
        for (int i = 0; i < CF::KINS; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void *)(ks + (i * NW + wave) * 1024), 16,
                                                     KSEP ? kvo[0] + i * kstep : kvo[i < KN ? i : 0], 0, 0, 0);
#else
        (void)kb; (void)slot;
#endif
    };
    auto dma_v = [&](int kb, int slot) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int k0 = key_of(kb);
        const Rsrc rv = rsrc(Vh + k0, (uint32_t)((long)a.dv * a.stride * 2 - (long)k0 * 2));
        char *vs = v_tile(slot);
        const uint32_t past = k0 + vkey < a.stride ? 0u : kOOB;   // past a row's end lies the next row
#pragma unroll
        for (int i = 0; i < CF::VINS; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void *)(vs + (i * NW + wave) * 1024), 16,
                                                     (vvo + i * vstep) | past, 0, 0, 0);
#else
        (void)kb; (void)slot;
#endif
    };
    // Ragged V^T rows: the thread's chunks (those of its DMA slots) at any 2-byte address, a tile ahead; the last ones of a
    // row lie at its last eight keys, and are moved into place, zeros behind them, on their way to LDS.
    [[maybe_unused]] i32x4 rv[CF::VINS];
    auto load_rv = [&](int kb) __attribute__((always_inline)) {
        const int key = min(key_of(min(kb, kb1 - 1)) + vkey, (int)a.stride - 8);
#pragma unroll
        for (int i = 0; i < CF::VINS; i++)
            rv[i] = reinterpret_cast<const Halves8 *>(Vh + (size_t)min(32 * i + vrow, a.dv - 1) * a.stride + key)->v;
    };
    auto put_rv = [&](int kb, int slot) __attribute__((always_inline)) {
        const int past = key_of(kb) + vkey + 8 - (int)a.stride;   // halves of the chunk behind the row's end
        char *vs = v_tile(slot) + (wave * 64 + lane) * 16;
        if (key_of(kb) + BK > a.stride) {
#pragma unroll
            for (int i = 0; i < CF::VINS; i++) {
                i32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; e++) {   // half e of the chunk is half e + past of the eight that were loaded
                    int h = 0;
#pragma unroll
                    for (int f = 0; f < 8; f++) h = f == e + max(past, 0) ? (rv[i][f >> 1] >> (16 * (f & 1))) & 0xFFFF : h;
                    x[e >> 1] |= h << (16 * (e & 1));
                }
                *reinterpret_cast<i32x4 *>(vs + i * NW * 1024) = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < CF::VINS; i++) *reinterpret_cast<i32x4 *>(vs + i * NW * 1024) = rv[i];
        }
    };
    // 4-bit: a thread's runs of codes. Keys: key tid / 4, words 4 g + i of run g (D 64: 2 (tid % 4) + i). Values: block
    // tid % 8 of eight keys, VD nibbles of word w.
    [[maybe_unused]] int kw[CF::ITEMS][CF::KW];
    [[maybe_unused]] f16x2 ksm[CF::ITEMS];
    [[maybe_unused]] i32x4 vw[CF::ITEMS][2], vsm[CF::ITEMS][2];
    [[maybe_unused]] unsigned vp[4];                 // of one run: pairs of keys, the thread's nibbles lowest
    [[maybe_unused]] f16x2 vsc[4], vmi[4];
    [[maybe_unused]] const int vpart = D == 64 ? (tid >> 3) & 3 : (tid >> 3) & 1, vword = D == 64 ? tid >> 5 : tid >> 4;
    [[maybe_unused]] const Widen widen;
    [[maybe_unused]] const size_t hr = C4 ? (size_t)s * a.c.heads + hk : 0;
    // (No load stands under a condition: its registers would be copied, and so waited for, where the paths meet. Past the
    // last tile the last one's loads are repeated; past the capacity, which a tile may end 32 keys behind, and past
    // dk or dv others of the tile are loaded: hidden keys, dims that Q has as 0, rows that are not stored.)
    auto load_k = [&](int kb) __attribute__((always_inline)) {
        const int key = min(key_of(min(kb, kb1 - 1)) + (tid >> 2), a.c.cap - 1);
        const char *codes = a.c.kc + (hr * a.c.cap + key) * (a.dk / 2), *sms = a.c.ks + (hr * a.c.cap + key) * (a.dk / 8);
#pragma unroll
        for (int i = 0; i < CF::ITEMS; i++) {
            const int p = tid & 3, d = D == 64 ? min(16 * p, a.dk - 16) : min(32 * (p + 4 * i), a.dk - 32);
            if constexpr (D == 64) {
                const i32x2 x = *reinterpret_cast<const i32x2 *>(codes + d / 2);
                kw[i][0] = x[0];
                kw[i][1] = x[1];
            } else {
                const i32x4 x = *reinterpret_cast<const i32x4 *>(codes + d / 2);
#pragma unroll
                for (int e = 0; e < 4; e++) kw[i][e] = x[e];
            }
            ksm[i] = *reinterpret_cast<const f16x2 *>(sms + d / 32 * 4);
        }
    };
    auto load_v = [&](int kb, int i) __attribute__((always_inline)) {
        const int key = min(key_of(min(kb, kb1 - 1)) + 8 * (tid & 7), a.c.cap - 8);
        const size_t block = hr * (a.c.cap / 8) + key / 8;
        const int w = min(vword + 16 * i, a.dv / 8 - 1);
        const char *p = a.c.vc + (block * (a.dv / 8) + w) * 32, *m = a.c.vs + (block * (a.dv / 32) + w / 4) * 32;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            vw[i][e] = *reinterpret_cast<const i32x4 *>(p + 16 * e);
            vsm[i][e] = *reinterpret_cast<const i32x4 *>(m + 16 * e);
        }
    };
    // unit u of a thread's key words: eight dims of its key, a 16-byte write into each half's tile
    auto put_k = [&](int u) __attribute__((always_inline)) {
        const int i = u / CF::KW, w = u % CF::KW, key = tid >> 2;
        const int chunk = D == 64 ? 2 * (tid & 3) + w : 4 * ((tid & 3) + 4 * i) + w;
        const HiLo x = kv4_keys(kw[i][w], KeyScale(ksm[i][0]));
        const int at = key * (D * 2) + ((chunk ^ CF::kx(key)) << 4);
        *reinterpret_cast<f16x8 *>(k_tile(0) + at) = x.hi;
        *reinterpret_cast<f16x8 *>(k_tile(1) + at) = x.lo;
        if (w == 0) mins[8 * key + chunk / 4] = ksm[i][1];   // (D 64: two threads the same)
    };
    // pairs of keys of run i of the thread's value words; keys that no row sees get scale and minimum 0
    auto pair_v = [&](int kb, int i) __attribute__((always_inline)) {
        const int key0 = key_of(kb);
        if (!whole(key0)) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (dead(key0 + 8 * (tid & 7) + e)) vsm[i][e >> 2][e & 3] = 0;
        }
        const unsigned half = D == 64 ? vpart >> 1 : vpart;
        const unsigned sel = half ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned w0 = vw[i][k >> 1][2 * (k & 1)], w1 = vw[i][k >> 1][2 * (k & 1) + 1];
            const unsigned s0 = vsm[i][k >> 1][2 * (k & 1)], s1 = vsm[i][k >> 1][2 * (k & 1) + 1];
            vp[k] = __builtin_amdgcn_perm(w1, w0, sel) >> (D == 64 ? 8 * (vpart & 1) : 0);
            vsc[k] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x05040100u));
            vmi[k] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x07060302u));
        }
    };
    // (Two runs, heads of 256: each where its first unit is written, so that the pairs of one take registers alone: 4% of
    // 2048 tokens' time. One run: in front of QK, 6% of it for heads of 128, whose loads then have longer.)
    auto next_v = [&](int kb, int i) __attribute__((always_inline)) {
        pair_v(max(kb, kb0), i);
        load_v(kb + 1, i);
    };
    // unit u: eight keys of one dim, one 16-byte write
    auto put_v = [&](int kb, int slot, int u) __attribute__((always_inline)) {
        const int i = u / CF::VD, j = u % CF::VD, d = 8 * (vword + 16 * i) + CF::VD * vpart + j;
        if (CF::ITEMS > 1 && j == 0) next_v(kb, i);
        f16x8 x;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const f16x2 y = widen.at(vp[k], j, vsc[k], vmi[k]);
            x[2 * k] = y[0];
            x[2 * k + 1] = y[1];
        }
        *reinterpret_cast<f16x8 *>(v_tile(slot) + d * 128 + (((tid & 7) ^ vx(d)) << 4)) = x;
    };

    constexpr int PH = C4 ? 2 : 1;       // halves of a weight
    float m_run = -1e30f, l_run = 0.f;   // (finite: a row may see nothing of a tile)
    f32x16 O[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) O[d] = f32x16{};

    // S^T for the 64 keys of the K tile in slot `slot`: two 32-key blocks; fragments are read two steps ahead. Codes: steps take
    // first and second halves in turn, and the minimums' product stands in front.
    constexpr int QKS = C4 ? 2 * KC : KC;
    auto qk = [&](int slot, f32x16 (&Sx)[2], auto &&beside) __attribute__((always_inline)) {
        auto kfrag = [&](int t, int sb) __attribute__((always_inline)) {
            const int row = 32 * sb + l32, lc = 2 * (C4 ? t / 2 : t) + hh;
            return *reinterpret_cast<const f16x8 *>(k_tile(C4 ? t & 1 : slot) + row * (D * 2) + ((lc ^ CF::kx(row)) << 4));
        };
        f16x8 kf[3][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            kf[t][0] = kfrag(t, 0);
            kf[t][1] = kfrag(t, 1);
        }
#pragma unroll
        for (int sb = 0; sb < 2; sb++) {
            Sx[sb] = f32x16{};
            if constexpr (C4)
                Sx[sb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8 *>(mins + 8 * (32 * sb + l32)), qsum, Sx[sb], 0, 0, 0);
        }
        if constexpr (C4) {
            if (__builtin_expect(back, 0)) {
                Sx[0] *= qback;
                Sx[1] *= qback;
            }
        }
#pragma unroll
        for (int t = 0; t < QKS; t++) {
            if (t + 2 < QKS) {
                kf[(t + 2) % 3][0] = kfrag(t + 2, 0);
                kf[(t + 2) % 3][1] = kfrag(t + 2, 1);
            }
#pragma unroll
            for (int sb = 0; sb < 2; sb++) {
                Sx[sb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[t % 3][sb], qf[C4 ? t / 2 : t], Sx[sb], 0, 0, 0);
                beside(2 * t + sb);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // Scores stay products, and the factor to log2 units joins the exponential's subtraction (Q carries the scale's sign, so
    // that the largest product is the largest score; a scale of 0: Q is 0 and the factor 1, so that hidden keys'
    // -infinity stays one). A score under a cap up to kNarrowCap, c tanh(y) = 2 c sigmoid(2 y) - c, is kept as its sigmoid: 2 c is
    // the factor, and the constant leaves the softmax unchanged (hardware exponential and reciprocal: within c 2^-22 of the
    // score; four operations for six, 2048 tokens over 8192 keys, heads of 128, 361 us, 342). One under a larger cap is
    // kept as it is.
    const float unit = CAP == kWide ? 1.4426950408889634f : CAP == kNarrow ? 2.f * 1.4426950408889634f * fabsf(a.softcap) : a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    [[maybe_unused]] const float slope = -cap_slope(fabsf(a.scale), fabsf(a.softcap));
    auto cap1 = [&](f32x16 (&Sx)[2], int e) __attribute__((always_inline)) {
        if constexpr (CAP == kWide) Sx[e >> 4][e & 15] = softcap_wide(Sx[e >> 4][e & 15] * fabsf(a.scale), 1.f / a.softcap, a.softcap);
        else if constexpr (CAP == kNarrow) Sx[e >> 4][e & 15] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(Sx[e >> 4][e & 15] * slope));
    };
    auto mask = [&](int kb, f32x16 (&Sx)[2]) __attribute__((always_inline)) {
        const int key0 = key_of(kb);
        const int k0 = key0 + 4 * hh, after = pos - k0, before = behind - k0;
        auto hide = [&](auto &&hidden) __attribute__((always_inline)) {
#pragma unroll
            for (int sb = 0; sb < 2; sb++)
#pragma unroll
                for (int e = 0; e < 16; e++) Sx[sb][e] = hidden(32 * sb + 8 * (e >> 2) + (e & 3)) ? -INFINITY : Sx[sb][e];
        };
        if (key0 + BK - 1 > p_lo) hide([&](int k) __attribute__((always_inline)) { return k > after; });
        if (a.window && key0 <= p_hi - a.window) {
            if (key0 >= a.sinks) hide([&](int k) __attribute__((always_inline)) { return k <= before; });
            else if (key0 + BK > a.sinks) hide([&](int k) __attribute__((always_inline)) { return ((k - before - 1) & (a.sinks - 1 - k0 - k)) < 0; });
        }
    };
    auto highest = [&](float mloc) __attribute__((always_inline)) {
        const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, mloc), __builtin_bit_cast(unsigned, mloc), false, false);
        const unsigned x0 = x[0], x1 = x[1];
        return fmaxf(__builtin_bit_cast(float, x0), __builtin_bit_cast(float, x1));
    };
    // Weights are 2^(score - m_run), with m_run 10 (in log2 units) below the largest score, and it moves when some row's
    // scores pass it by more than 15.5: then a weight stays inside fp16 and one is lost to it only below 2^-35 of the
    // largest (around the maximum itself 2^-25, which 2^17 such keys made 2e-3 of a result). The division by the sum
    // makes the result independent of m_run. Both go by the product that the exponential takes, unrounded, so that no
    // rounding of a large score (2^27 is rounded by 4) carries a weight past fp16.
    auto rescale = [&](float m_new) __attribute__((always_inline)) {
        const float alpha = exp2f(m_run - m_new);
        m_run = m_new;
#pragma unroll
        for (int d = 0; d < DB; d++) O[d] *= alpha;
        return alpha;
    };
    auto grows = [&](float mloc) __attribute__((always_inline)) { return (bool)__any(fmaf(mloc, unit, -m_run) > 15.5f); };
    auto raised = [&](float mloc) __attribute__((always_inline)) { return fmaxf(m_run, fmaf(mloc, unit, -10.f)); };
    // Weights of halves are rounded to one, and the sum takes them as rounded, two at a time in fp32: weights and their sum round
    // alike. Those of codes are two halves.
    auto prob1 = [&](const f32x16 (&Sx)[2], f16x8 (&pb)[PH][2][2], float m, float &psum, int e) __attribute__((always_inline)) {
        const int sb = e >> 4, i = e & 15;
        const float p = __builtin_amdgcn_exp2f(fmaf(Sx[sb][i], unit, -m));
        const _Float16 h = (_Float16)p;
        pb[0][sb][i >> 3][i & 7] = h;
        if constexpr (C4) {
            pb[PH - 1][sb][i >> 3][i & 7] = (_Float16)(p - (float)h);
            psum += p;
        } else if (i & 1) {
            psum = __builtin_amdgcn_fdot2(f16x2{pb[0][sb][i >> 3][(i & 7) - 1], pb[0][sb][i >> 3][i & 7]}, f16x2{(_Float16)1.f, (_Float16)1.f}, psum, false);
        }
    };
    // P to natural key order: of 16 keys, half-wave 0 holds 0-3 and 8-11 and takes 0-7
    auto reorder = [&](f16x8 (&pb)[PH][2][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < PH; h++)
#pragma unroll
            for (int sb = 0; sb < 2; sb++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    i32x4 w = __builtin_bit_cast(i32x4, pb[h][sb][t]);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const auto x = __builtin_amdgcn_permlane32_swap((unsigned)w[e], (unsigned)w[2 + e], false, false);
                        w[e] = (int)x[0];
                        w[2 + e] = (int)x[1];
                    }
                    pb[h][sb][t] = __builtin_bit_cast(f16x8, w);
                }
    };
    // O^T += V^T P^T for the V^T tile in slot `slot`
    auto pv = [&](int slot, const f16x8 (&pb)[PH][2][2], auto &&beside) __attribute__((always_inline)) {
        const char *vs = v_tile(slot);
        auto vfrag = [&](int j, int db) __attribute__((always_inline)) {   // keys 16 j + 8 hh .. + 8
            const int d = 32 * db + l32;
            return *reinterpret_cast<const f16x8 *>(vs + d * 128 + (((2 * j + hh) ^ vx(d)) << 4));
        };
        f16x8 vf[2][DB];
#pragma unroll
        for (int db = 0; db < DB; db++) vf[0][db] = vfrag(0, db);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int db = 0; db < DB; db++) {
                if (j + 1 < 4) vf[(j + 1) & 1][db] = vfrag(j + 1, db);
#pragma unroll
                for (int h = 0; h < PH; h++) {
                    O[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[j & 1][db], pb[h][j >> 1][j & 1], O[db], 0, 0, 0);
                    beside((j * DB + db) * PH + h);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
    };
    // fp16 values of a tile that is not seen whole, before its products (0 times an infinity or a NaN would reach rows
    // that do not see its key): dead keys become 0; where a key that some rows see holds a non-finite value, the rows
    // that see it take it here, and the products take 0.
    auto clean_v = [&](int kb, int slot) __attribute__((always_inline)) {
        if constexpr (!C4) {
            const int key0 = key_of(kb);
            if (whole(key0)) return;
            char *vs = v_tile(slot);
            // an exponent of all ones carries into the sign's place
            auto not_finite = [](unsigned w) __attribute__((always_inline)) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; };
            // (a thread's chunks, 32 rows apart, hold the same eight keys)
            const int key = key0 + 8 * ((tid & 7) ^ vx(tid >> 3));
            unsigned live[4];
#pragma unroll
            for (int i = 0; i < 4; i++) live[i] = (dead(key + 2 * i) ? 0u : 0xFFFFu) | (dead(key + 2 * i + 1) ? 0u : 0xFFFF0000u);
            const bool edge = (live[0] & live[1] & live[2] & live[3]) != 0xFFFFFFFFu;
            auto each = [&](bool finite) __attribute__((always_inline)) {
                unsigned bad = 0;
#pragma unroll
                for (int g = 0; g < D / 32; g++) {
                    i32x4 *const p = reinterpret_cast<i32x4 *>(vs + (tid + 256 * g) * 16);
                    i32x4 x = *p;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[i] &= (int)live[i];
                        const unsigned nf = not_finite(x[i]);
                        bad |= nf;
                        if (finite) x[i] &= ~(int)((nf >> 15) * 0xFFFFu);
                    }
                    if (edge || finite) *p = x;
                }
                return bad != 0;
            };
            if (each(false)) *bad_tile = kb;
            lds_barrier();
            if (__builtin_expect(*bad_tile == kb, 0)) {
#pragma unroll 1
                for (int i = 0; i < DB * 16; i++) {   // (rolled, and the register picked by comparison: this is rare)
                    const int d = 32 * (i >> 4) + 8 * (i >> 2 & 3) + 4 * hh + (i & 3);
                    float x = 0.f;
#pragma unroll 1
                    for (int j = 0; j < BK; j++) {
                        const int w = *reinterpret_cast<const uint16_t *>(vs + d * 128 + (((j >> 3) ^ vx(d)) << 4) + 2 * (j & 7));
                        if ((w & 0x7C00) == 0x7C00 && sees(key0 + j)) x += (float)__builtin_bit_cast(_Float16, (uint16_t)w);
                    }
#pragma unroll
                    for (int db = 0; db < DB; db++)
#pragma unroll
                        for (int e = 0; e < 16; e++) O[db][e] = i == 16 * db + e ? O[db][e] + x : O[db][e];
                }
                lds_barrier();
                each(true);
                lds_barrier();
            }
        }
    };

    // Iteration kb: PV of tile kb - 1 beside the score arithmetic of tile kb (soft-caps, the maximum), then QK of tile kb + 1
    // beside the exponentials of tile kb. K tile kb + 2 goes into the K slot that tile kb left, V^T tile kb into the V^T slot that tile
    // kb - 2 left; both are read an iteration on. (Codes: K tile kb + 1 into the one slot that tile kb left, in front of its QK, with a
    // barrier between.) The first iteration (kb0 - 1) has the first QK alone and the last
    // (kb1) the last PV, so that there is one copy of the products' code. Codes are loaded a whole iteration before they are
    // widened, keys beside PV and values beside QK, each beside its first half, so that the writes are through at the barrier (also where there is no such tile: into slots that nothing reads again
    // before they are written).
    constexpr int QKM = 2 * QKS, PVM = 4 * DB * PH;
    // With one wave a SIMD a phase takes its instructions' issue or its MFMAs, whichever is longer: over halves of heads of 256
    // QK's is the former and PV's the latter, so half of the exponentials go beside PV, whose first half then finds the
    // maximum (512 tokens over 16384 keys 161 us, 155; 8 of the 32 159, 24 156). Over codes, whose widening fills PV, and at two
    // waves a SIMD it was slower.
    constexpr int EARLY = !CAPPED && !C4 && D == 256 ? 16 : 0, MXM = EARLY ? PVM / 2 : PVM;
    f32x16 S[2] = {};
    f16x8 P[PH][2][2] = {};
    if (kb0 < kb1) {
        if constexpr (C4) {
            load_k(kb0);
#pragma unroll
            for (int i = 0; i < CF::ITEMS; i++) load_v(kb0, i);
        } else {
            dma_k(kb0, 0);
            if (tid == 0) *bad_tile = -1;
        }
#pragma unroll 1
        for (int kb = kb0 - 1;; kb++) {
            const int cur = (kb - kb0) & 1;
            // (Q in the accumulators' registers, where the MFMAs read it as well: else the compiler moves 70 others a tile, 3%)
            if constexpr (D == 256) {
#pragma unroll
                for (int c = 0; c < KC; c++) asm volatile("" : "+a"(qf[c]));
            }
            const bool tile = kb >= kb0 && kb < kb1;
            if constexpr (!C4) wait_vm0();
            lds_barrier();
            if constexpr (!C4) {
                if (kb + 2 < kb1) dma_k(kb + 2, cur);
                if constexpr (!RV) {
                    if (tile) dma_v(kb, cur);
                } else {
                    if (tile) put_rv(kb, cur);
                    load_rv(kb + 1);
                }
            }
            if constexpr (!CAPPED) {
                if (tile) mask(kb, S);
            }
            float mloc = -INFINITY, psum = 0.f;
            [[maybe_unused]] float m_next = m_run;
            [[maybe_unused]] bool up = false;
            f16x8 Pm[PH][2][2], (&Pn)[PH][2][2] = EARLY > 0 ? Pm : P;
            if (kb > kb0) {
                clean_v(kb - 1, cur ^ 1);
                pv(cur ^ 1, P, [&](int m) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = m * 32 / MXM; e < min(32, (m + 1) * 32 / MXM); e++) {
                        cap1(S, e);
                        mloc = fmaxf(mloc, S[e >> 4][e & 15]);
                    }
                    if constexpr (EARLY > 0) {
                        if (m == MXM) {
                            mloc = highest(mloc);
                            up = tile && grows(mloc);
                            m_next = up ? raised(mloc) : m_run;
                        }
                        if (m >= MXM) {
#pragma unroll
                            for (int e = (m - MXM) * EARLY / (PVM - MXM); e < (m + 1 - MXM) * EARLY / (PVM - MXM); e++) prob1(S, Pn, m_next, psum, e);
                        }
                    }
                    if constexpr (C4) {
#pragma unroll
                        for (int u = m * CF::KU / (PVM / 2); u < min(CF::KU, (m + 1) * CF::KU / (PVM / 2)); u++) put_k(u);
                    }
                });
                if (kb == kb1) break;
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    cap1(S, e);
                    mloc = fmaxf(mloc, S[e >> 4][e & 15]);
                }
                if constexpr (EARLY > 0) {
                    mloc = highest(mloc);
                    up = tile && grows(mloc);
                    m_next = up ? raised(mloc) : m_run;
#pragma unroll
                    for (int e = 0; e < EARLY; e++) prob1(S, Pn, m_next, psum, e);
                }
                if constexpr (C4) {
#pragma unroll
                    for (int u = 0; u < CF::KU; u++) put_k(u);
                }
            }
            if constexpr (C4) load_k(kb + 2);
            if constexpr (CAPPED) {   // (a hidden key's capped score would not be -infinity: masks come behind it)
                if (tile && !whole(key_of(kb))) {
                    mask(kb, S);
                    mloc = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; e++) mloc = fmaxf(mloc, S[e >> 4][e & 15]);
                }
            }
            float alpha = 1.f;
            if constexpr (EARLY > 0) {
                if (__builtin_expect(up, 0)) alpha = rescale(m_next);
            } else if (tile) {
                mloc = highest(mloc);
                if (__builtin_expect(grows(mloc), 0)) alpha = rescale(raised(mloc));
            }
            if constexpr (C4 && CF::ITEMS == 1) next_v(kb, 0);
            if constexpr (C4) lds_barrier();   // (the K tile is whole; the barrier above let it be written)
            if (kb + 1 < kb1) {
                f32x16 Sn[2];
                qk(cur ^ 1, Sn, [&](int m) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = EARLY + m * (32 - EARLY) / QKM; e < EARLY + (m + 1) * (32 - EARLY) / QKM; e++) prob1(S, Pn, m_run, psum, e);
                    if constexpr (C4) {
#pragma unroll
                        for (int u = m * CF::VU / (QKM / 2); u < min(CF::VU, (m + 1) * CF::VU / (QKM / 2)); u++) put_v(kb, cur, u);
                    }
                });
                S[0] = Sn[0];
                S[1] = Sn[1];
            } else {
                float m = m_run;
                asm("" : "+v"(m));   // (or the compiler takes both branches' subtractions out in front of the products)
#pragma unroll
                for (int e = EARLY; e < 32; e++) prob1(S, Pn, m, psum, e);
                if constexpr (C4) {
#pragma unroll
                    for (int u = 0; u < CF::VU; u++) put_v(kb, cur, u);
                }
            }
            if (tile) {
                reorder(Pn);
                if constexpr (EARLY > 0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) P[0][i >> 1][i & 1] = Pn[0][i >> 1][i & 1];
                }
                l_run = l_run * alpha + psum;
            }
        }
    }

    // lane holds dims 32 db + 8 b + 4 hh + c of its row
    const float l = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = l == 0.f ? 0.f : 1.f / l;   // (a row that sees nothing; NaN stays)
    // Results go through LDS, a wave's 32 rows by themselves, so that they are stored as they lie, 16 bytes a lane side by
    // side: lanes that store their own rows' pieces of 8 bytes took 6 us of a call's 21 (2048 rows of two tiles each,
    // heads of 256). A pass takes as many dims as the tiles' room holds.
    auto store_rows = [&](auto *base) __attribute__((always_inline)) {
        typedef std::remove_reference_t<decltype(*base)> E;
        typedef E E4 __attribute__((ext_vector_type(4)));
        constexpr int EC = 16 / sizeof(E), DP = D * 2 / sizeof(E), RS = D * 2 + 16;   // (16 bytes of padding: rows start on other banks)
        static_assert(NW * 32 * RS <= 2 * CF::STAGE, "the rows fit the tiles' room");
        char *const mine = smem + wave * 32 * RS;
        const int first_row = r0 + wave * 32, n_rows = min(32, r1 + 1 - first_row);
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += DP) {
#pragma unroll
            for (int db = d0 / 32; db < (d0 + DP) / 32; db++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    E4 v;
#pragma unroll
                    for (int c = 0; c < 4; c++) v[c] = (E)(O[db][4 * b + c] * inv);
                    *reinterpret_cast<E4 *>(mine + l32 * RS + (32 * db + 8 * b + 4 * hh - d0) * (int)sizeof(E)) = v;
                }
            wave_lds_order();
            const int chunks = (min(a.dv, d0 + DP) - d0) / EC;   // of a row
            if (chunks > 0) {
                int row = lane / chunks, c = lane - row * chunks;
                const int rows_on = 64 / chunks, c_on = 64 - rows_on * chunks;
                while (row < n_rows) {
                    *reinterpret_cast<i32x4 *>(base + (size_t)(first_row + row) * a.dv + d0 + c * EC) =
                        *reinterpret_cast<const i32x4 *>(mine + row * RS + c * 16);
                    row += rows_on;
                    c += c_on;
                    if (c >= chunks) {
                        c -= chunks;
                        row++;
                    }
                }
            }
            wave_lds_order();
        }
    };
    lds_barrier();   // (the tiles are read no more)
    if (ta.nsplit > 1) {
        const size_t rows = (size_t)a.n_seq * a.n_head * T, prow = zs * rows + row0;
        if (qok && hh == 0) reinterpret_cast<f32x2 *>(ta.part + ta.nsplit * rows * a.dv)[prow + r] = f32x2{m_run, l};
        store_rows(ta.part + prow * a.dv);
    } else {
        store_rows(a.out + row0 * a.dv);
    }
}

// Merges the splits: out = sum_s w_s O_s / sum_s w_s with w_s = 2^(m_s - m) l_s, m the largest of the m_s, for four output
// dims of a row a thread; every split's pair and outputs are loaded before the first is used.
template <int MAXS>
__global__ __launch_bounds__(256) void k_serve_combine(const float *__restrict__ part, _Float16 *__restrict__ out, long rows, int dv, int nsplit)
{
    const int dq = dv / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, row = i / dq;
    if (row >= rows) return;
    const int d0 = (int)(i - row * dq) * 4;
    const f32x2 *const ml = reinterpret_cast<const f32x2 *>(part + nsplit * rows * dv);
    f32x2 x[MAXS];
    f32x4 o[MAXS];
#pragma unroll
    for (int s = 0; s < MAXS; s++)
        if (s < nsplit) {
            x[s] = ml[s * rows + row];
            o[s] = *reinterpret_cast<const f32x4 *>(part + (s * rows + row) * dv + d0);
        }
    float m = -1e30f;
#pragma unroll
    for (int s = 0; s < MAXS; s++)
        if (s < nsplit) m = fmaxf(m, x[s][0]);
    float l = 0.f;
    f32x4 acc = {};
#pragma unroll
    for (int s = 0; s < MAXS; s++)
        if (s < nsplit) {
            const float w = __builtin_amdgcn_exp2f(x[s][0] - m) * x[s][1];
            l += w;
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] += w * o[s][c];
        }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const f16x4 h = {(_Float16)(acc[0] * inv), (_Float16)(acc[1] * inv), (_Float16)(acc[2] * inv), (_Float16)(acc[3] * inv)};
    *reinterpret_cast<f16x4 *>(out + row * dv + d0) = h;
}

void combine(const TileArgs &ta, long rows, long blocks, hipStream_t s)
{
    auto *kern = ta.nsplit <= 4 ? k_serve_combine<4> : ta.nsplit <= 8 ? k_serve_combine<8> : ta.nsplit <= 16 ? k_serve_combine<16> : k_serve_combine<32>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, s, ta.part, ta.a.out, rows, ta.a.dv, ta.nsplit);
}

template <int D, Src SRC, Cap CAP> hipError_t launch_c(const TileArgs &ta, unsigned wgs, hipStream_t s)
{
    auto kern = k_serve_tiles<D, SRC, CAP>;
    static_assert(Cfg<D>::LDS <= 160 * 1024, "LDS budget");
    static std::atomic<uint64_t> opted{0};
    if (const hipError_t e = lds_opt_in(reinterpret_cast<const void *>(kern), Cfg<D>::LDS, opted)) return e;
    hipLaunchKernelGGL(kern, dim3(wgs), dim3(256), Cfg<D>::LDS, s, ta);
    return hipGetLastError();
}
template <int D, Src SRC> hipError_t launch_s(const TileArgs &ta, unsigned wgs, hipStream_t s)
{
    switch (cap_of(ta.a.softcap)) {
    case kUncapped: return launch_c<D, SRC, kUncapped>(ta, wgs, s);
    case kNarrow: return launch_c<D, SRC, kNarrow>(ta, wgs, s);
    default: return launch_c<D, SRC, kWide>(ta, wgs, s);
    }
}
template <int D> hipError_t launch(const TileArgs &ta, unsigned wgs, hipStream_t s)
{
    if (!ta.a.Kf) return launch_s<D, kCodes>(ta, wgs, s);
    return ta.a.stride % 8 ? launch_s<D, kRagged>(ta, wgs, s) : launch_s<D, kHalves>(ta, wgs, s);
}

// Row blocks of a KV head: its rows in a row, or each head's tokens by themselves, which takes more blocks where the
// tokens are no multiple of one, but leaves none with rows of two heads, the first tokens of one and the last of the
// other, which between them see every tile of the call: whichever has fewer tiles to visit.
struct Blocks {
    long len, per, all;
};
Blocks row_blocks(const ServeAttn &a)
{
    const long T = a.n_tokens, R = (long)a.gqa * T, w = a.window ? std::min(a.window, a.max_kv) : a.max_kv;
    const long flat = (R + BQ - 1) / BQ, head = (T + BQ - 1) / BQ, mixed = T % BQ ? std::min<long>(a.gqa - 1, flat) : 0;
    const long seen = a.window ? BQ + w : w;
    if (a.window && T > BQ && head * a.gqa * seen < (flat - mixed) * seen + mixed * (T + w)) return {T, head, head * a.gqa};
    return {R, flat, flat};
}

int splits(const ServeAttn &a)
{
    // enough workgroups for every CU (256), and two on one where the registers allow it, each split keeping at least 2 of
    // the tiles that a block may see, more than 16 at least 4 (128 rows, heads of 128: 8 KV heads over 16000 codes 39.1 us with
    // 16 splits, 32 29.1; over 4000 19.0 with 16 of 4 tiles, 21.3 with 31 of 2)
    const int d = std::max(a.dk, a.dv);
    const long wgs = row_blocks(a).all * (a.n_head / a.gqa) * a.n_seq, want = d <= 64 || (d <= 128 && a.Kf) ? 512 : 256;
    long tiles = (a.max_kv + BK - 1) / BK;
    if (a.window) tiles = std::min<long>(tiles, (std::min(a.sinks, a.max_kv) + BK - 1) / BK + ((long)std::min(a.n_tokens, BQ) + a.window - 2) / BK + 2);
    const long most = std::max(std::min(tiles / 2, 16L), std::min((tiles + 3) / 4, 32L));
    return (int)std::max<long>(1, std::min((want + wgs - 1) / wgs, most));
}

}  // namespace

size_t serve_tiles_ws(const ServeAttn &a)
{
    const int ns = splits(a);
    return ns > 1 ? (size_t)ns * a.n_seq * a.n_head * a.n_tokens * (a.dv + 2) * sizeof(float) : 0;
}

hipError_t serve_tiles(const ServeAttn &a, hipStream_t s, uint64_t *blocks)
{
    if (a.Kf && a.stride % 8 && a.stride < 8) return hipErrorInvalidValue;
    TileArgs ta;
    ta.a = a;
    ta.nsplit = a.ws && a.ws_bytes >= serve_tiles_ws(a) ? splits(a) : 1;
    ta.part = a.ws;
    const Blocks b = row_blocks(a);
    const long wgs = b.all * (a.n_head / a.gqa) * a.n_seq * ta.nsplit;
    if (wgs > 0x7FFFFFFFL) return hipErrorInvalidValue;
    ta.nqb = (int)b.all;
    ta.len = (int)b.len;
    ta.per = (int)b.per;
    const int d = std::max(a.dk, a.dv);
    const hipError_t e = d <= 64 ? launch<64>(ta, (unsigned)wgs, s) : d <= 128 ? launch<128>(ta, (unsigned)wgs, s) : launch<256>(ta, (unsigned)wgs, s);
    *blocks = (uint64_t)wgs;
    if (e != hipSuccess || ta.nsplit == 1) return e;
    const long rows = (long)a.n_seq * a.n_head * a.n_tokens, n = (rows * (a.dv / 4) + 255) / 256;
    combine(ta, rows, n, s);
    *blocks += (uint64_t)n;
    return hipGetLastError();
}

}  // namespace rk
