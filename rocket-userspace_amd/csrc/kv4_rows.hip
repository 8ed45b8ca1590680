// kv4_rows.hip — attention of few query rows (decode steps, drafts) over the 4-bit cache.
//
// What bounds it is how fast the codes arrive, and about as much the VALU that widens them: some three
// operations a pair of values or keys, whatever the number of query rows, and the MFMAs beside it. So all rows of a KV head (its query heads'
// tokens, at most 64, in blocks of 16) share one widening (of heads above 128 each 32). A workgroup owns a place of the
// batch, a KV head and a range of its keys; each of its four waves takes chunks of 32 keys and loads them straight into registers as
// they lie in the cache, the next chunk's while this one's are widened.
//
// Scores are transposed, S^T = K Q^T (v_mfma_f32_16x16x32_f16, K the first operand): lane (c, q) =
// (l % 16, l / 16) holds query c and keys 8 q .. 8 q + 7 of the chunk, as the second product takes them.
// The order of the summed dims is free as long as Q has the same: quarter q takes whole groups, so a
// lane's sixteen bytes of a key share one scale. In O^T += V^T P^T the rows (dims) are free: lane c
// takes a word of eight dims of each of its eight keys, product j their nibbles j, which a byte permute brings
// side by side as pairs of keys.
//
// Keys and weights go into the products as two halves each (kv4_widen.h), so beside the result's there is one rounding: a widened
// value's, to the half that rocket_kv4_read_fp16 gives; scores, maxima, sums and outputs are fp32. The result is within
// 2.8e-4 of its size (the rounded result alone 2.1e-4). Of up to eight rows the weights' second halves take the product's other
// eight columns (32 / 8 heads of 128, one token of 32 sequences: 52.6 us, with products of their own 58). Measured by trace: 32
// sequences of up to 8192 keys, 32 / 8 heads of 128, one token, 249 MB, 52.6 us (4.7 TB/s; a large copy's rate is 5.1, which keys
// and weights of one half reached) and 4.7 for the merge; one sequence of 3000 keys, 16 / 8 heads of 256, 7.0 and 3.8: two
// launches, each a chain of loads that nothing else hides.
#include "kv4_widen.h"
#include "lds_optin.h"
#include "serve.h"
#include "softcap.h"

#include <algorithm>
#include <atomic>

namespace rk {
namespace {

typedef int      i32x2 __attribute__((ext_vector_type(2)));
typedef int      i32x4 __attribute__((ext_vector_type(4)));
typedef float    f32x2 __attribute__((ext_vector_type(2)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 32, kWaves = 4, kMaxSplit = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4RowArgs {
    ServeAttn a;
    int nsplit;   // workgroups a place and KV head, which share the chunks that its length has
    float *part;       // [place][split][head][token][dv] outputs, then (max, sum) pairs
};

// The chunks of a sequence of n keys that some of its last T tokens sees: those of the sinks, then from the
// first window's on. v -> the v-th of them.
struct Chunks {
    int first, sinks, ns, skip, count;
    __device__ Chunks(const ServeAttn &a, int n)
    {
        first = a.window ? max(0, n - a.n_tokens - a.window + 1) : 0;   // (n and n_tokens below 2^24)
        sinks = min(a.sinks, first);
        ns = (sinks + kChunk - 1) / kChunk;
        const int f = max(first / kChunk, ns);
        skip = f - ns;
        count = ns + (n - 1) / kChunk - f + 1;
    }
    __device__ int at(int v) const { return v < ns ? v : v + skip; }
};

// Chunks a workgroup: the length's own share, so that a long bound costs a short sequence nothing (one a wave at least).
__device__ __forceinline__ int share(int count, int nsplit) { return max(kWaves, (count + nsplit - 1) / nsplit); }

// D: head sizes up to this (64, 128, 256). ROWS: at most this many (8, or blocks of 16). FULL: dk and dv are D.
template <int D, int ROWS, Cap CAP, bool FULL>
__global__ __launch_bounds__(kWaves * 64, D <= 128 && ROWS <= 16 ? 4 : D == 64 && ROWS == 64 ? 2 : 1) void k_kv4_rows(const Kv4RowArgs ra)
{
    const ServeAttn &a = ra.a;
    constexpr bool FOLD = ROWS == 8;
    constexpr int NQ = FOLD ? 1 : ROWS / 16;
    constexpr int U = D == 256 ? 2 : 1, KW = D == 64 ? 2 : 4, KS = U * KW;   // key words of a lane: U runs of KW
    constexpr int NJ = D == 64 ? 4 : 8, VB = U * NJ, LROW = D + 4;          // output blocks of 16 dims; LDS row (floats)
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the workgroup's R rows of the KV head's, from row0 on (heads above 128: blocks of 32 rows, a split's on one XCD where the
    // heads are a multiple of 8, whose L2 gives the second block the codes)
    constexpr bool BLOCKS = D == 256 && NQ == 2;
    const int hk = blockIdx.x, zs = BLOCKS ? blockIdx.y % ra.nsplit : blockIdx.y, s = blockIdx.z;
    const int T = a.n_tokens, row0 = BLOCKS ? blockIdx.y / ra.nsplit * 16 * NQ : 0;
    const int R = BLOCKS ? min(16 * NQ, a.gqa * T - row0) : a.gqa * T;
    const int n = a.seq_len[s];
    const size_t head0 = ((size_t)s * a.n_head + (size_t)hk * a.gqa) * T + row0;   // row of the first query
    f16x8 qf[NQ][KS];
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        const _Float16 *qrow = a.Q + (head0 + min(FOLD ? c & 7 : 16 * x + c, R - 1)) * a.dk;   // (rows behind the last repeat it)
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const int d = D == 64 ? 16 * q + 8 * i : 128 * (i / 4) + 32 * q + 8 * (i % 4);
            f16x8 y = *reinterpret_cast<const f16x8 *>(qrow + (FULL ? d : min(d, a.dk - 8)));
            if ((!FULL && d >= a.dk) || (CAP == kUncapped && a.scale == 0.f)) y = f16x8{};
            if (CAP == kUncapped && a.scale < 0.f) y = -y;
            qf[x][i] = kv4_query_order(y);
        }
    }
    asm volatile("" ::: "memory");   // (the queries' loads are sent before the length is there)
    // the sums of this lane's queries over its runs, a group's (D 64: half of one's) dims each, as the operand that meets the
    // groups' minimums: halves 2 u and 2 u + 1 for run u. (Beside the length's load, as the queries: behind the first chunk's
    // loads it was no faster, and took registers.)
    f16x4 qsum[NQ] = {};
    float qback[NQ];
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        float sum[U], most = 0.f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            sum[u] = 0.f;
#pragma unroll
            for (int i = 0; i < KW; i++) sum[u] = kv4_sum(qf[x][KW * u + i], sum[u]);
            most = fmaxf(most, fabsf(sum[u]));
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        const int e = kv4_sum_exponent(most);
        qback[x] = __builtin_amdgcn_ldexpf(1.f, e);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const f16x2 h = kv4_sum_halves(sum[u], e);
            qsum[x][2 * u] = h[0];
            qsum[x][2 * u + 1] = h[1];
        }
    }
    const bool served = n >= 1 && n <= a.max_kv;
    const Chunks list(a, served ? n : 1);
    const int count = served ? list.count : 0;
    const int cps = ra.nsplit > 1 ? share(count, ra.nsplit) : max(count, 1);
    if (zs > 0 && zs * cps >= count) return;   // (the merge knows)
    // this lane's queries: row 16 x + c of the workgroup's (a KV head's row r: head r / T of it, token r % T), and its position
    bool qok[NQ];
    int pos[NQ], behind[NQ];                      // (the last key behind its window)
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        const int r = FOLD ? c & 7 : 16 * x + c;
        qok[x] = 16 * x + c < R;
        pos[x] = n - T + (row0 + r) % T;
        behind[x] = a.window ? pos[x] - a.window : -1;
    }
    const int p_lo = n - T, p_hi = n - 1;

    const size_t hr = (size_t)s * a.c.heads + hk;
    const int dk = FULL ? D : a.dk, dv = FULL ? D : a.dv;
    const char *const kc = a.c.kc + hr * a.c.cap * (dk / 2), *const ks = a.c.ks + hr * a.c.cap * (dk / 8);
    const char *const vc = a.c.vc + hr * a.c.cap * (dv / 2), *const vs = a.c.vs + hr * a.c.cap * (dv / 8);
    // (a head's part is 2^30 bytes at most: 32-bit offsets, which leave the addresses' upper halves in scalar registers)
    int kw[2][KS];        // block b's key of this lane: 8 (c / 4) + 4 b + c % 4
    f16x2 ksm[2][U];
    i32x4 vw[U][2];       // a word of each of the keys 8 q .. 8 q + 7
    i32x4 vsm[U][2];      // their (scale, minimum)
    auto load_k = [&](int key0) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t key = key0 + 8 * (c >> 2) + 4 * b + (c & 3);
#pragma unroll
            for (int u = 0; u < U; u++) {
                [[maybe_unused]] const int g = 4 * u + q;   // the run: a group (D 64: half of one)
                // (past dk another run of the key: Q has those dims as 0)
                const int run = FULL ? (D == 64 ? q : g) : D == 64 ? min(q, dk / 16 - 1) : min(g, dk / 32 - 1);
                if constexpr (D == 64) {
                    const i32x2 x = *reinterpret_cast<const i32x2 *>(kc + (uint32_t)(key * (dk / 2) + 8 * run));
                    kw[b][0] = x[0];
                    kw[b][1] = x[1];
                    ksm[b][u] = *reinterpret_cast<const f16x2 *>(ks + (uint32_t)(key * (dk / 8) + 4 * (run >> 1)));
                } else {
                    const i32x4 x = *reinterpret_cast<const i32x4 *>(kc + (uint32_t)(key * (dk / 2) + 16 * run));
#pragma unroll
                    for (int i = 0; i < 4; i++) kw[b][4 * u + i] = x[i];
                    ksm[b][u] = *reinterpret_cast<const f16x2 *>(ks + (uint32_t)(key * (dk / 8) + 4 * run));
                }
            }
        }
    };
    auto load_v = [&](int key0) __attribute__((always_inline)) {
        const uint32_t block = key0 / 8 + q;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int word = D == 64 ? c >> 1 : 16 * u + c;   // the lane's word: dims 8 w .. 8 w + 7
            const int w = FULL ? word : min(word, dv / 8 - 1);   // (results past dv are not stored)
            const char *p = vc + (uint32_t)((block * (dv / 8) + w) * 32), *m = vs + (uint32_t)((block * (dv / 32) + w / 4) * 32);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                vw[u][i] = *reinterpret_cast<const i32x4 *>(p + 16 * i);
                vsm[u][i] = *reinterpret_cast<const i32x4 *>(m + 16 * i);
            }
        }
    };

    const Widen widen;
    [[maybe_unused]] const float rest = c >= 8 ? 1.f : 0.f;   // (FOLD: this lane's column is of the weights' second halves)
    // Uncapped scores stay products, and the factor to log2 units joins the exponential's subtraction. (Q carries the scale's
    // sign, so that the largest product is the largest score; a scale of 0: Q is 0 and the factor 1, so that hidden keys'
    // -infinity stays one.)
    const float unit = CAP != kUncapped || a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
    float m_run[NQ], l_run[NQ];
    f32x4 O[NQ][VB];
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        m_run[x] = -1e30f;
        l_run[x] = 0.f;
#pragma unroll
        for (int j = 0; j < VB; j++) O[x][j] = f32x4{};
    }
    const int c1 = min(count, (zs + 1) * cps);
    int ch = zs * cps + wave;
    if (ch < c1) {
        load_k(list.at(ch) * kChunk);
        load_v(list.at(ch) * kChunk);
    }
    for (; ch < c1; ch += kWaves) {
        const int key0 = list.at(ch) * kChunk;
        f32x4 S[NQ][2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            f16x4 mf = {};
#pragma unroll
            for (int u = 0; u < U; u++) mf[2 * u] = mf[2 * u + 1] = ksm[b][u][1];
#pragma unroll
            for (int x = 0; x < NQ; x++) S[x][b] = __builtin_amdgcn_mfma_f32_16x16x16f16(mf, qsum[x], f32x4{}, 0, 0, 0) * qback[x];
        }
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const HiLo kf = kv4_keys(kw[b][i], KeyScale(ksm[b][i / KW][0]));
#pragma unroll
                for (int x = 0; x < NQ; x++) S[x][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf.hi, qf[x][i], S[x][b], 0, 0, 0);
#pragma unroll
                for (int x = 0; x < NQ; x++) S[x][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf.lo, qf[x][i], S[x][b], 0, 0, 0);
            }
        const bool more = ch + kWaves < c1;
        const int next = list.at(more ? ch + kWaves : ch) * kChunk;
        if (more) load_k(next);
        // every row sees every key of the chunk, or the rows differ (uniform)
        const bool whole = key0 + kChunk - 1 <= p_lo && (!a.window || key0 > p_hi - a.window || key0 + kChunk <= a.sinks);
        if (!whole) {
            // keys that no row sees: their values count as 0, whatever the memory holds
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 8 * q + i;
                    if ((bool)((key > p_hi) | ((key < list.first) & (key >= list.sinks)))) vsm[u][i >> 2][i & 3] = 0;
                }
        }
        f16x8 p[NQ];
        [[maybe_unused]] f16x8 pl[NQ];
#pragma unroll
        for (int x = 0; x < NQ; x++) {
            float v[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = S[x][i >> 2][i & 3];
                if constexpr (CAP != kUncapped) v[i] = softcap_log2<CAP>(y, a.scale, a.softcap);
                else v[i] = y;
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 8 * q + i;
                    v[i] = (bool)((key <= pos[x]) & ((key > behind[x]) | (key < a.sinks))) ? v[i] : -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, v[i]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__any(fmaf(mx, unit, -m_run[x]) > 15.5f)) {
                const float m_new = fmaxf(m_run[x], lifted(mx, unit)), alpha = __builtin_amdgcn_exp2f(m_run[x] - m_new);
                m_run[x] = m_new;
                l_run[x] *= alpha;
#pragma unroll
                for (int j = 0; j < VB; j++) O[x][j] *= alpha;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(v[i], unit, -m_run[x]));
                l_run[x] += e;
                const _Float16 h = (_Float16)e;
                if constexpr (FOLD) p[x][i] = (_Float16)fmaf(-(float)h, rest, e);
                else {
                    p[x][i] = h;
                    pl[x][i] = (_Float16)(e - (float)h);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            int x[2][4];      // low and high halves of the words of two keys each
            f16x2 sc[4], mi[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const unsigned w0 = vw[u][k >> 1][2 * (k & 1)], w1 = vw[u][k >> 1][2 * (k & 1) + 1];
                const unsigned s0 = vsm[u][k >> 1][2 * (k & 1)], s1 = vsm[u][k >> 1][2 * (k & 1) + 1];
                if constexpr (D == 64) {   // lane c has the low or the high half of its word
                    x[0][k] = (int)__builtin_amdgcn_perm(w1, w0, c & 1 ? 0x07060302u : 0x05040100u);
                } else {
                    x[0][k] = (int)__builtin_amdgcn_perm(w1, w0, 0x05040100u);
                    x[1][k] = (int)__builtin_amdgcn_perm(w1, w0, 0x07060302u);
                }
                sc[k] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x05040100u));
                mi[k] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x07060302u));
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                f16x8 f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const f16x2 y = widen.at(x[j >> 2][k], j & 3, sc[k], mi[k]);
                    f[2 * k] = y[0];
                    f[2 * k + 1] = y[1];
                }
#pragma unroll
                for (int b = 0; b < NQ; b++) O[b][u * NJ + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[b], O[b][u * NJ + j], 0, 0, 0);
                if constexpr (!FOLD) {
#pragma unroll
                    for (int b = 0; b < NQ; b++) O[b][u * NJ + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, pl[b], O[b][u * NJ + j], 0, 0, 0);
                }
            }
        }
        if (more) load_v(next);
    }

    // merge the waves: [wave][row][LROW] outputs, then [wave][row] (max, sum)
    float *const Ol = reinterpret_cast<float *>(smem);
    f32x2 *const ml = reinterpret_cast<f32x2 *>(Ol + kWaves * R * LROW);
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        l_run[x] += __shfl_xor(l_run[x], 16, 64);
        l_run[x] += __shfl_xor(l_run[x], 32, 64);
        if constexpr (FOLD) {   // the columns of the second halves, eight lanes on
#pragma unroll
            for (int j = 0; j < VB; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = O[x][j][e];   // (bit_cast of a vector's element itself takes the first)
                    O[x][j][e] = y + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), 0x128, 0xF, 0xF, true));   // row_ror:8
                }
        }
        if (!qok[x]) continue;
        float *const row = Ol + (wave * R + 16 * x + c) * LROW;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++)   // block row 4 q + e: dims NJ (4 q + e) + j
#pragma unroll
                for (int j = 0; j < NJ; j += 4)
                    *reinterpret_cast<f32x4 *>(row + 128 * u + NJ * (4 * q + e) + j) =
                        f32x4{O[x][u * NJ + j][e], O[x][u * NJ + j + 1][e], O[x][u * NJ + j + 2][e], O[x][u * NJ + j + 3][e]};
        if (q == 0) ml[wave * R + 16 * x + c] = f32x2{m_run[x], l_run[x]};
    }
    __syncthreads();
    const int dq = dv / 4;
    for (int i = tid; i < R * dq; i += kWaves * 64) {
        const int r = i / dq, d0 = (i - r * dq) * 4;
        float m = -1e30f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) m = fmaxf(m, ml[w * R + r][0]);
        float l = 0.f;
        f32x4 o = {};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const f32x2 x = ml[w * R + r];
            const float f = __builtin_amdgcn_exp2f(x[0] - m);
            l += f * x[1];
            o += f * *reinterpret_cast<const f32x4 *>(Ol + (w * R + r) * LROW + d0);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;   // (a row that sees nothing; NaN stays)
        if (ra.nsplit > 1) {
            const size_t row = ((size_t)s * ra.nsplit + zs) * a.n_head * T + (size_t)hk * a.gqa * T + row0 + r;
            *reinterpret_cast<f32x4 *>(ra.part + row * dv + d0) = o * inv;
            if (d0 == 0) reinterpret_cast<f32x2 *>(ra.part + (size_t)a.n_seq * ra.nsplit * a.n_head * T * dv)[row] = f32x2{m, l};
        } else {
            f16x4 out;
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = (_Float16)(o[e] * inv);
            *reinterpret_cast<f16x4 *>(a.out + (head0 + r) * dv + d0) = out;
        }
    }
}

// Merges the splits that a sequence's length has, one (head, token) row of a place a workgroup: out = sum_s
// w_s On_s / sum_s w_s with w_s = 2^(m_s - m) l_s, outputs in fp32 (a rounding of each to fp16 would be a third
// one beside the probabilities' and the result's). Pairs and outputs of every split that there may be are loaded beside the
// length, which then says how many count (the others' hold anything).
__global__ __launch_bounds__(256) void k_kv4_merge(const Kv4RowArgs ra)
{
    const ServeAttn &a = ra.a;
    __shared__ float sum[8 * 256];
    const int tid = threadIdx.x, row = blockIdx.x, s = blockIdx.y, dv = a.dv;
    const size_t rows = (size_t)a.n_head * a.n_tokens, base = (size_t)s * ra.nsplit * rows + row;
    const int dq = dv / 8, sg = tid / dq, d0 = (tid - sg * dq) * 8, ng = min(8, 256 / dq);   // dv <= 256: 8
    f32x4 os[8][2];
    if (sg < ng)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int sp = sg + i * ng;
            if (sp < ra.nsplit)
#pragma unroll
                for (int j = 0; j < 2; j++) os[i][j] = reinterpret_cast<const f32x4 *>(ra.part + (base + sp * rows) * dv + d0)[j];
        }
    const f32x2 pair = reinterpret_cast<const f32x2 *>(ra.part + (size_t)a.n_seq * ra.nsplit * rows * dv)[base + min(tid & 63, ra.nsplit - 1) * rows];
    const int n = a.seq_len[s];
    const int count = n >= 1 && n <= a.max_kv ? Chunks(a, n).count : 0;
    const int cps = share(count, ra.nsplit), nsplit = max(1, (count + cps - 1) / cps);
    // (every wave makes the weights, lane i split i's: that is shorter than one that hands them out)
    const f32x2 x = (tid & 63) < nsplit ? pair : f32x2{-1e30f, 0.f};
    float m = x[0];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float w = __builtin_amdgcn_exp2f(x[0] - m) * x[1];
    float l = w;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
    const float wt = l == 0.f ? 0.f : w / l;
    float ws[8];
#pragma unroll
    for (int i = 0; i < 8; i++) ws[i] = __shfl(wt, sg + i * ng, 64);
    if (sg < ng) {
        float acc[8] = {};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int sp = sg + i * ng;
            if (sp < nsplit)
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] += ws[i] * os[i][e >> 2][e & 3];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) sum[sg * dv + d0 + e] = acc[e];
    }
    __syncthreads();
    for (int d = tid; d < dv; d += 256) {
        float o = 0.f;
        for (int sp = 0; sp < ng; sp++) o += sum[sp * dv + d];
        a.out[((size_t)s * rows + row) * dv + d] = (_Float16)o;
    }
}

// Blocks of 16 rows that a KV head's queries make; of heads above 128 a workgroup takes two at most, whose outputs its
// registers hold.
int row_blocks(const ServeAttn &a) { return (a.gqa * a.n_tokens + 15) / 16; }
int row_groups(const ServeAttn &a) { return std::max(a.dk, a.dv) <= 128 ? 1 : (row_blocks(a) + 1) / 2; }

template <int D, int ROWS, Cap CAP, bool FULL> hipError_t launch_f(const Kv4RowArgs &ra, hipStream_t s)
{
    auto kern = k_kv4_rows<D, ROWS, CAP, FULL>;
    const ServeAttn &a = ra.a;
    const int R = std::min(ROWS, a.gqa * a.n_tokens);
    const size_t lds = (size_t)kWaves * R * ((D + 4) * 4 + 8);
    if (lds > 64 * 1024) {
        static std::atomic<uint64_t> opted{0};
        constexpr int most = kWaves * ROWS * ((D + 4) * 4 + 8);
        static_assert(most <= 160 * 1024, "LDS budget");
        if (const hipError_t e = lds_opt_in(reinterpret_cast<const void *>(kern), most, opted)) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)a.c.heads, (unsigned)(ra.nsplit * row_groups(a)), (unsigned)a.n_seq), dim3(kWaves * 64), lds, s, ra);
    return hipGetLastError();
}
template <int D, int ROWS> hipError_t launch_q(const Kv4RowArgs &ra, hipStream_t s)
{
    const bool full = ra.a.dk == D && ra.a.dv == D;
    switch (cap_of(ra.a.softcap)) {
    case kUncapped: return full ? launch_f<D, ROWS, kUncapped, true>(ra, s) : launch_f<D, ROWS, kUncapped, false>(ra, s);
    case kNarrow: return full ? launch_f<D, ROWS, kNarrow, true>(ra, s) : launch_f<D, ROWS, kNarrow, false>(ra, s);
    default: return launch_f<D, ROWS, kWide, false>(ra, s);   // (rare: one kernel for all heads)
    }
}
template <int D> hipError_t launch(const Kv4RowArgs &ra, hipStream_t s)
{
    const int nq = row_blocks(ra.a);
    if constexpr (D <= 128) {
        if (nq > 2) return launch_q<D, 64>(ra, s);
    }
    if (ra.a.gqa * ra.a.n_tokens <= 8) return launch_q<D, 8>(ra, s);
    return nq == 1 ? launch_q<D, 16>(ra, s) : launch_q<D, 32>(ra, s);
}

// Chunks that a sequence of up to max_kv keys may have to visit.
int most_chunks(const ServeAttn &a)
{
    const int all = (a.max_kv + kChunk - 1) / kChunk;
    if (!a.window) return all;
    const long seen = (std::min<long>(a.sinks, a.max_kv) + kChunk - 1) / kChunk + ((long)a.n_tokens + a.window - 2) / kChunk + 2;
    return (int)std::min<long>(all, seen);
}

int splits(const ServeAttn &a)
{
    const int chunks = most_chunks(a);
    // As many workgroups as the CUs hold at once, a wave of each a SIMD: one more round, or a few workgroups of one, costs
    // more than longer shares (1024 for all: 16 sequences of 4000 keys, heads of 256, one row 33.4 us, so 31.3; 24 rows
    // 75.7, 59.8; heads of 128, 20 rows 34.7, 32.7).
    const int d = std::max(a.dk, a.dv), nq = row_blocks(a);
    const long resident = 256 * (nq == 1 ? (d <= 128 ? 4 : 2) : nq == 2 ? (d <= 64 ? 3 : d <= 128 ? 2 : 1) : d <= 64 ? 2 : 1);
    const long wgs = (long)a.c.heads * a.n_seq * row_groups(a), waves = (chunks + kWaves - 1) / kWaves;
    const long n = std::min<long>({waves, resident / wgs, kMaxSplit});
    if (n < 2) return 1;
    // Where that saves more than the merge costs: a wave's chunks less, at what one takes a wave (ns, measured unsplit), against
    // a launch of some 3.5 us and 2 + dv / 100 ns a row of the batch, a workgroup each. (Over 250 shapes of 1 to 64 rows the better
    // of the two but for 0.2% of the time, 20% at worst; always split 12%: 32 sequences of 300 keys, 8 heads of 64,
    // 64 rows 46.1 us, unsplit 11.6; 16 of 1000, heads of 128, 24 rows 22.1 and 17.3; one token of one sequence of 300, heads
    // of 64, 7.2 and 5.2, of 1000 7.2 and 8.7.)
    static const long chunk_ns[3][3] = {{700, 1100, 1700}, {950, 1400, 2600}, {1600, 2400, 2400}};
    const long saved = (waves - (chunks + n * kWaves - 1) / (n * kWaves)) * chunk_ns[d <= 64 ? 0 : d <= 128 ? 1 : 2][std::min(nq, 3) - 1];
    const long rows = (long)a.n_seq * a.n_head * a.n_tokens;
    return saved < 3500 + rows * (200 + a.dv) / 100 ? 1 : (int)n;
}

}  // namespace

// Up to 64 rows. In tiles of 128 rows, at 16000 keys of one sequence, 8 KV heads of 128: 20 rows 31.8 us, here 16.9; 64 rows
// 34.9 and 27.7; at 16 sequences of 4000 keys 80.7 and 32.7, 84.5 and 73.6. Heads of 256, 64 rows: 16000 keys of one sequence
// 51.5 and 36.0, 8 sequences of 4000 81.5 and 63.3, 32 of 2000 137 and 97; a third block would lose there what it gains at
// one. (64 rows of a few dozen short sequences are even, 32 of 1000 keys, 2 heads of 64, 20.4 and 20.7, or lose a little, heads
// of 128 there 24.4 and 28.5.)
bool kv4_few_rows(const ServeAttn &a) { return (long)a.gqa * a.n_tokens <= 64; }

size_t kv4_rows_ws(const ServeAttn &a)
{
    const int n = splits(a);
    return n > 1 ? (size_t)a.n_seq * n * a.n_head * a.n_tokens * (a.dv + 2) * sizeof(float) : 0;
}

hipError_t kv4_rows(const ServeAttn &a, hipStream_t s, uint64_t *blocks)
{
    if (a.n_seq > 65535) return hipErrorInvalidValue;
    Kv4RowArgs ra;
    ra.a = a;
    ra.nsplit = a.ws && a.ws_bytes >= kv4_rows_ws(a) ? splits(a) : 1;
    ra.part = a.ws;
    const int d = std::max(a.dk, a.dv);
    const hipError_t e = d <= 64 ? launch<64>(ra, s) : d <= 128 ? launch<128>(ra, s) : launch<256>(ra, s);
    *blocks = (uint64_t)a.c.heads * ra.nsplit * row_groups(a) * a.n_seq;
    if (e != hipSuccess || ra.nsplit == 1) return e;
    const unsigned rows = (unsigned)(a.n_head * a.n_tokens);
    hipLaunchKernelGGL(k_kv4_merge, dim3(rows, (unsigned)a.n_seq), dim3(256), 0, s, ra);
    *blocks += (uint64_t)rows * a.n_seq;
    return hipGetLastError();
}

}  // namespace rk
