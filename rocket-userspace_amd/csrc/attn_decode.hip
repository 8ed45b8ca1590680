// attn_decode.hip — attention of few query rows (decode steps) for gfx950.
//
// A KV head's query rows, the tokens of every query head that reads it, are at most 16 here (under
// a window up to 64, in blocks of 16), so the tiled kernel's 128-query workgroups (attn.hip) would be mostly padding; what bounds the
// call is how fast K and V arrive. A workgroup owns a KV head and a range of its keys; each of
// its 4 waves takes chunks of 32 keys and loads their K rows and V^T columns straight into
// registers as MFMA fragments, 32 KB of them in flight a wave at head size 256, next chunk's K
// while this chunk's scores and outputs are formed. All of a KV head's query rows share one
// read of its keys. V^T rows of any length are read in place: no padded copy. (Rows at
// 4-byte addresses cost nothing here; an odd number of keys, rows at 2-byte ones, up to twice the time of a
// chunk.)
//
// Scores are transposed, S^T = K Q^T (v_mfma_f32_16x16x32_f16, K the first operand): lane l
// holds query l % 16. The 16 rows of K block b are keys 8 (i / 4) + 4 b + i % 4, so that lane
// quarter q ends up with keys 8 q .. 8 q + 7 of the chunk, which is what the second product's
// operand takes: O^T += V^T P^T, P rounded to fp16 in registers. The waves' outputs merge in
// LDS, the workgroups' in k_fa_merge; a short cache is one workgroup's, and has no merge.
//
// Measured (sets of operands in turn; before, with attn.hip; after):
//   1 x 3000 keys, 16 / 8 heads of 256    31.6 -> 10.8 us  (24.6 MB of K and V; 8.0 us the kernel, 3.1 TB/s)
//   1 x 4096 keys, 32 / 8 heads of 128    18.2 ->  8.8
//   8 x 3000 keys, 16 / 8 heads of 256    33.5 -> 14.2     (with a mask)
#include "attn.h"
#include "lds_optin.h"
#include "softcap.h"

#include <algorithm>
#include <atomic>

namespace rk {
namespace {

typedef int      i32x4  __attribute__((ext_vector_type(4)));
typedef float    f32x2  __attribute__((ext_vector_type(2)));
typedef float    f32x4  __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2  __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4  __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8  __attribute__((ext_vector_type(8)));
typedef __amdgpu_buffer_rsrc_t Rsrc;
// eight halves at any 2-byte address
struct __attribute__((packed, aligned(2))) Halves8 { i32x4 v; };

constexpr int kRows = 16, kChunk = 32, kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ Rsrc rsrc(const void *base, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ i32x4 ld16(Rsrc r, uint32_t off)
{
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

struct RowArgs {
    const _Float16 *Q, *K, *Vt, *mask;
    _Float16 *O;
    long q_hs, q_rs, k_hs, k_rs, v_hs, v_rs, o_hs, o_rs, m_rs;
    int T, n_kv, dk, dv, gqa, n_head;
    float scale, softcap;
    int nsplit, cps;   // workgroups a KV head, chunks a workgroup
    float *part;       // [split][head][T][dv] outputs, then [split][head][T] (max, sum)
    // WIN: the chunks that some token sees, v -> v below ns, v + skip from there on, count of them; keys
    // [sinks, first) are seen by none
    int window, sinks, first, ns, skip, count;
};

// Halves key .. key + 8 of a row of n (n >= 8), zeros past the row: the last eight are loaded
// and shifted where the row ends inside. No branch: one around each of a chunk's loads made them wait
// for each other (1 x 255 keys in one workgroup a head, heads of 256: 20.8 -> 18.8 us).
__device__ __forceinline__ i32x4 row8(const _Float16 *row, int key, int n)
{
    const i32x4 v = reinterpret_cast<const Halves8 *>(row + min(key, n - 8))->v;
    const int past = max(key + 8 - n, 0), s = 16 * (past & 3);   // halves past the row's end
    unsigned long lo = (unsigned)v[0] | ((unsigned long)(unsigned)v[1] << 32);
    unsigned long hi = (unsigned)v[2] | ((unsigned long)(unsigned)v[3] << 32);
    lo = past >= 8 ? 0 : (past >= 4 ? hi : lo);
    hi = past >= 4 ? 0 : hi;
    lo = (lo >> s) | ((hi << 1) << (63 - s));
    hi >>= s;
    return i32x4{(int)(unsigned)lo, (int)(lo >> 32), (int)(unsigned)hi, (int)(hi >> 32)};
}

// Merges the splits, one (head, token) row a workgroup: out = sum_s w_s On_s / sum_s w_s with
// w_s = 2^(m_s - m) l_s, for up to 64 splits. The outputs are fp32, as one workgroup without splits
// holds them: caches from 257 keys on are split here, and a rounding of each split's output to fp16
// beside those of the probabilities and of the result would cost a quarter more error (448 keys, heads
// of 256: 2.5e-4 of the result, with it 3.2e-4). The splits spread over
// the workgroup's 256 threads (dv / 8 threads a split), whose sums add in LDS. (A merge by each KV
// head's last workgroup instead of this launch, on an arrival counter, measured 15.5 against 11.1
// us at 3000 keys: the counter's release and acquire write back and invalidate the XCD's L2, and
// one workgroup walks all rows.)
__global__ __launch_bounds__(256) void k_fa_merge(const float *__restrict__ part, _Float16 *__restrict__ O, long o_hs, long o_rs,
                                                  int n_head, int T, int dv, int nsplit)
{
    __shared__ float wt[64], sum[8 * 256];
    const int tid = threadIdx.x, row = blockIdx.x, h = row / T, t = row - h * T;
    const size_t rows = (size_t)n_head * T;
    const int dq = dv / 8, sg = tid / dq, d0 = (tid - sg * dq) * 8, ng = min(8, 256 / dq);   // dv <= 256: 8
    f32x4 os[8][2];
    if (sg < ng)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int s = sg + i * ng;
            if (s < nsplit)
#pragma unroll
                for (int j = 0; j < 2; j++) os[i][j] = reinterpret_cast<const f32x4 *>(part + ((size_t)s * rows + row) * dv + d0)[j];
        }
    if (tid < 64) {
        const f32x2 x = tid < nsplit ? reinterpret_cast<const f32x2 *>(part + (size_t)nsplit * rows * dv)[(size_t)tid * rows + row]
                                     : f32x2{-INFINITY, 0.f};
        float m = x[0];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const float w = __builtin_amdgcn_exp2f(x[0] - m) * x[1];
        float l = w;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
        wt[tid] = l > 0.f ? w / l : 0.f;
    }
    __syncthreads();
    if (sg < ng) {
        float acc[8] = {};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int s = sg + i * ng;
            if (s < nsplit)
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] += wt[s] * os[i][e >> 2][e & 3];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) sum[sg * dv + d0 + e] = acc[e];
    }
    __syncthreads();
    for (int d = tid; d < dv; d += 256) {
        float o = 0.f;
        for (int s = 0; s < ng; s++) o += sum[s * dv + d];
        O[(size_t)h * o_hs + (size_t)t * o_rs + d] = (_Float16)o;
    }
}

// D: head sizes up to this (64, 128, 256); dk a multiple of 32, dv of 16. FULL: both are D, so
// that no load or product carries a test of its dims. WIN: token t sees the keys up to its own, n_kv - T + t, that
// lie in its window or among the sinks; no mask and no clamp. There a row may see nothing of a chunk (a
// finite first maximum), and values of keys that a row does not see must not reach it as 0 times an infinity. NQ:
// blocks of 16 rows that share a chunk's fragments.
template <int D, int NQ, Cap CAP, bool FULL, bool WIN>
__global__ __launch_bounds__(kWaves * 64) void k_fa_rows(const RowArgs a)
{
    constexpr int KS = D / 32, VB = D / 16, LROW = D + 4;   // score steps, output blocks, LDS row (floats)
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x, zs = blockIdx.y;
    const int R = a.gqa * a.T;
    // this lane's queries: row 16 x + c, head hk gqa + row / T, token row % T
    bool qok[NQ];
    int t[NQ], pos[NQ], behind[NQ];                         // (position; the last key behind the token's window)
    i32x4 qf[NQ][KS];
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        const int r = 16 * x + c, hg = r / a.T;
        t[x] = r - hg * a.T;
        qok[x] = r < R;
        pos[x] = a.n_kv - a.T + t[x];
        behind[x] = a.window ? pos[x] - a.window : -1;
        const _Float16 *qrow = a.Q + (size_t)(hk * a.gqa + (qok[x] ? hg : 0)) * a.q_hs + (size_t)(qok[x] ? t[x] : 0) * a.q_rs;
#pragma unroll
        for (int s = 0; s < KS; s++)
            qf[x][s] = (qok[x] && (FULL || 32 * s < a.dk)) ? *reinterpret_cast<const i32x4 *>(qrow + 32 * s + 8 * q) : i32x4{0, 0, 0, 0};
    }
    const Rsrc rk = rsrc(a.K + (size_t)hk * a.k_hs, (uint32_t)((long)a.n_kv * a.k_rs * 2));   // keys past n_kv: zeros
    const _Float16 *const Vh = a.Vt + (size_t)hk * a.v_hs + (size_t)c * a.v_rs;              // rows 16 j + c
    const _Float16 *const mrow = !WIN && a.mask ? a.mask + (size_t)t[0] * a.m_rs : nullptr;
    auto key_of = [&](int ch) __attribute__((always_inline)) { return (WIN && ch >= a.ns ? ch + a.skip : ch) * kChunk; };
    // (no short circuits: a branch a score takes longer, and the compiler lost a lane's mask among them)
    auto sees = [&](int x, int key) __attribute__((always_inline)) { return (bool)((key <= pos[x]) & ((key > behind[x]) | (key < a.sinks))); };

    i32x4 kf[2][KS], vf[VB];
    const uint32_t ko = (uint32_t)((8 * (c >> 2) + (c & 3)) * a.k_rs + 8 * q) * 2u, k4 = (uint32_t)(4 * a.k_rs) * 2u;
    auto load_k = [&](int key0) __attribute__((always_inline)) {
        const uint32_t o = ko + (uint32_t)((long)key0 * a.k_rs * 2);
#pragma unroll
        for (int s = 0; s < KS; s++)
            if (FULL || 32 * s < a.dk) {
                kf[0][s] = ld16(rk, o + 64u * s);
                kf[1][s] = ld16(rk, o + k4 + 64u * s);
            }
    };
    auto load_v = [&](int key0) __attribute__((always_inline)) {
        const int key = key0 + 8 * q;
        if (key0 + kChunk <= a.n_kv) {   // uniform: whole chunks
#pragma unroll
            for (int j = 0; j < VB; j++)
                if (FULL || 16 * j < a.dv) vf[j] = reinterpret_cast<const Halves8 *>(Vh + (size_t)(16 * j) * a.v_rs + key)->v;
        } else {
#pragma unroll
            for (int j = 0; j < VB; j++)
                if (FULL || 16 * j < a.dv) vf[j] = row8(Vh + (size_t)(16 * j) * a.v_rs, key, a.n_kv);
        }
    };

    float m_run[NQ], l_run[NQ];
    f32x4 O[NQ][VB];
#pragma unroll
    for (int x = 0; x < NQ; x++) {
        m_run[x] = WIN ? -1e30f : -INFINITY;
        l_run[x] = 0.f;
#pragma unroll
        for (int j = 0; j < VB; j++) O[x][j] = f32x4{};
    }
    const int chunks = WIN ? a.count : (a.n_kv + kChunk - 1) / kChunk;
    const int c1 = min(chunks, (zs + 1) * a.cps);
    int ch = zs * a.cps + wave;
    if (ch < c1) {
        load_k(key_of(ch));
        load_v(key_of(ch));
    }
    for (; ch < c1; ch += kWaves) {
        const int key0 = key_of(ch);
        f32x4 S[NQ][2] = {};
#pragma unroll
        for (int s = 0; s < KS; s++)
            if (FULL || 32 * s < a.dk) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int x = 0; x < NQ; x++)
                        S[x][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kf[b][s]),
                                                                         __builtin_bit_cast(f16x8, qf[x][s]), S[x][b], 0, 0, 0);
            }
        const bool more = ch + kWaves < c1;
        const int next = WIN ? key_of(more ? ch + kWaves : ch) : key0 + kWaves * kChunk;
        if (more) load_k(next);
        // every row sees every key of the chunk (uniform)
        [[maybe_unused]] const bool whole = key0 + kChunk <= a.n_kv - a.T + 1 && (!a.window || key0 > a.n_kv - 1 - a.window || key0 + kChunk <= a.sinks);
        // the reference's score steps in log2 units; lane holds keys key0 + 8 q + 4 b + e
        i32x4 mw = {0, 0, 0, 0};
        if (mrow) mw = row8(mrow, key0 + 8 * q, a.n_kv);
        const f16x8 mv = __builtin_bit_cast(f16x8, mw);
        if constexpr (WIN) {
            if (!whole) {
                // keys that no row sees: their values count as 0
                i32x4 live = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 8 * q + i;
                    if (key < a.n_kv && !(key < a.first && key >= a.sinks)) live[i >> 1] |= 0xFFFF << (16 * (i & 1));
                }
#pragma unroll
                for (int j = 0; j < VB; j++) vf[j] &= live;
            }
        }
        f16x8 p[NQ];
#pragma unroll
        for (int x = 0; x < NQ; x++) {
            float v[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = S[x][i >> 2][i & 3];
                if constexpr (WIN && CAP != kUncapped) v[i] = softcap_log2<CAP>(y, a.scale, a.softcap);
                else if constexpr (WIN) v[i] = y * (a.scale * kLog2e);
                else if constexpr (CAP != kUncapped) v[i] = fmaxf(a.softcap * tanhf(y * a.scale / a.softcap) + (float)mv[i], -30000.f) * kLog2e;
                else v[i] = fmaxf(fmaf((float)mv[i], kLog2e, y * (a.scale * kLog2e)), -30000.f * kLog2e);
                if constexpr (!WIN) {
                    if (key0 + 8 * q + i >= a.n_kv) v[i] = -INFINITY;   // weighs 0
                    mx = fmaxf(mx, v[i]);
                }
            }
            if constexpr (WIN) {
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = sees(x, key0 + 8 * q + i) ? v[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) mx = fmaxf(mx, v[i]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if constexpr (WIN) mx = lifted(mx);
            if (__any(mx > m_run[x])) {   // (a chunk has a key below n_kv, so without a window the new maximum is finite)
                const float m_new = fmaxf(m_run[x], mx), alpha = __builtin_amdgcn_exp2f(m_run[x] - m_new);
                m_run[x] = m_new;
                l_run[x] *= alpha;
#pragma unroll
                for (int j = 0; j < VB; j++) O[x][j] *= alpha;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(v[i] - m_run[x]);
                p[x][i] = (_Float16)e;
                if constexpr (!WIN) l_run[x] += e;
                // (under a window the sum of the rounded weights, two at a time: weights and their sum round alike)
                else if (i & 1) l_run[x] = __builtin_amdgcn_fdot2(f16x2{p[x][i - 1], p[x][i]}, f16x2{(_Float16)1.f, (_Float16)1.f}, l_run[x], false);
            }
        }
        if constexpr (WIN) {
            // a non-finite value of a key that some rows see: those take it here, the products take 0
            if (!whole && a.T > 1) {
                bool bad = false;
#pragma unroll
                for (int j = 0; j < VB; j++)
                    if (FULL || 16 * j < a.dv) {   // (the others were not loaded)
#pragma unroll
                        for (int i = 0; i < 8; i++) bad |= (vf[j][i >> 1] >> (16 * (i & 1)) & 0x7C00) == 0x7C00;
                    }
                if (__builtin_expect(__any(bad), 0)) {
                    const uint16_t *const vr = reinterpret_cast<const uint16_t *>(a.Vt + (size_t)hk * a.v_hs);
#pragma unroll
                    for (int x = 0; x < NQ; x++)
#pragma unroll 1
                        for (int i = 0; i < VB * 4; i++) {   // (rolled, and the register picked by comparison: this is rare)
                            const int d = 16 * (i >> 2) + 4 * q + (i & 3);
                            float y = 0.f;
#pragma unroll 1
                            for (int j = 0; d < a.dv && j < kChunk && key0 + j < a.n_kv; j++) {
                                const uint16_t w = vr[(size_t)d * a.v_rs + key0 + j];
                                if ((w & 0x7C00) == 0x7C00 && sees(x, key0 + j)) y += (float)__builtin_bit_cast(_Float16, w);
                            }
#pragma unroll
                            for (int j = 0; j < VB; j++)
#pragma unroll
                                for (int e = 0; e < 4; e++) O[x][j][e] = i == 4 * j + e ? O[x][j][e] + y : O[x][j][e];
                        }
#pragma unroll
                    for (int j = 0; j < VB; j++)
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if ((vf[j][i >> 1] >> (16 * (i & 1)) & 0x7C00) == 0x7C00) vf[j][i >> 1] &= 0xFFFF << (16 * (~i & 1));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < VB; j++)
            if (FULL || 16 * j < a.dv) {
#pragma unroll
                for (int x = 0; x < NQ; x++)
                    O[x][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, vf[j]), p[x], O[x][j], 0, 0, 0);
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
        if (!qok[x]) continue;
        const int row = wave * R + 16 * x + c;
#pragma unroll
        for (int j = 0; j < VB; j++)
            if (FULL || 16 * j < a.dv) *reinterpret_cast<f32x4 *>(Ol + row * LROW + 16 * j + 4 * q) = O[x][j];
        if (q == 0) ml[row] = f32x2{m_run[x], l_run[x]};
    }
    __syncthreads();
    const int dq = a.dv / 4;
    for (int i = tid; i < R * dq; i += kWaves * 64) {
        const int r = i / dq, d0 = (i - r * dq) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; w++) m = fmaxf(m, ml[w * R + r][0]);
        float l = 0.f;
        f32x4 o = {};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const f32x2 x = ml[w * R + r];
            // (a wave without keys: 2^-inf = 0)
            const float f = __builtin_amdgcn_exp2f(x[0] - m);
            l += f * x[1];
            o += f * *reinterpret_cast<const f32x4 *>(Ol + (w * R + r) * LROW + d0);
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const int g = r / a.T, tt = r - g * a.T, h = hk * a.gqa + g;
        if (a.nsplit > 1) {
            const size_t row = ((size_t)zs * a.n_head + h) * a.T + tt;
            *reinterpret_cast<f32x4 *>(a.part + row * a.dv + d0) = o * inv;
            if (d0 == 0) reinterpret_cast<f32x2 *>(a.part + (size_t)a.nsplit * a.n_head * a.T * a.dv)[row] = f32x2{m, l};
        } else {
            f16x4 out;
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = (_Float16)(o[e] * inv);
            *reinterpret_cast<f16x4 *>(a.O + (size_t)h * a.o_hs + (size_t)tt * a.o_rs + d0) = out;
        }
    }
}

template <int D, int NQ, Cap CAP, bool FULL, bool WIN> hipError_t launch_rows_f(const RowArgs &a, int kv_heads, hipStream_t s)
{
    auto kern = k_fa_rows<D, NQ, CAP, FULL, WIN>;
    const int R = a.gqa * a.T;
    const size_t lds = (size_t)kWaves * R * ((D + 4) * 4 + 8);
    if (lds > 64 * 1024) {
        static std::atomic<uint64_t> opted{0};
        constexpr int most = kWaves * 16 * NQ * ((D + 4) * 4 + 8);
        static_assert(most <= 160 * 1024, "LDS budget");
        if (const hipError_t e = lds_opt_in(reinterpret_cast<const void *>(kern), most, opted)) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)kv_heads, (unsigned)a.nsplit), dim3(kWaves * 64), lds, s, a);
    return hipGetLastError();
}

template <int D, int NQ, bool WIN> hipError_t launch_rows_q(const RowArgs &a, int kv_heads, hipStream_t s)
{
    const bool full = a.dk == D && a.dv == D;
    const Cap cap = cap_of(a.softcap);
    if (cap == kUncapped) return full ? launch_rows_f<D, NQ, kUncapped, true, WIN>(a, kv_heads, s) : launch_rows_f<D, NQ, kUncapped, false, WIN>(a, kv_heads, s);
    if constexpr (WIN) {   // (without one, tanhf takes any cap)
        if (cap == kWide) return launch_rows_f<D, NQ, kWide, false, WIN>(a, kv_heads, s);   // (rare: one kernel for all heads)
    }
    return full ? launch_rows_f<D, NQ, kNarrow, true, WIN>(a, kv_heads, s) : launch_rows_f<D, NQ, kNarrow, false, WIN>(a, kv_heads, s);
}
template <int D, bool WIN> hipError_t launch_rows(const RowArgs &a, int kv_heads, hipStream_t s)
{
    if constexpr (WIN) {
        const int nq = (a.gqa * a.T + 15) / 16;
        if constexpr (D <= 64) {
            if (nq > 2) return launch_rows_q<D, 4, WIN>(a, kv_heads, s);
        }
        if (nq > 1) return launch_rows_q<D, 2, WIN>(a, kv_heads, s);
    }
    return launch_rows_q<D, 1, WIN>(a, kv_heads, s);
}
template <bool WIN> hipError_t launch_rows(const RowArgs &a, int kv_heads, hipStream_t s)
{
    const int d = std::max(a.dk, a.dv);
    return d <= 64 ? launch_rows<64, WIN>(a, kv_heads, s) : d <= 128 ? launch_rows<128, WIN>(a, kv_heads, s) : launch_rows<256, WIN>(a, kv_heads, s);
}

// The chunks to visit: all, or those that some token sees.
int chunk_list(const FaLaunch &L, RowArgs *a)
{
    const int all = (L.n_kv + kChunk - 1) / kChunk;
    const int first = L.win && L.window ? std::max(0, L.n_kv - L.T - L.window + 1) : 0, sinks = std::min(L.sinks, first);
    const int ns = (sinks + kChunk - 1) / kChunk, f = std::max(first / kChunk, ns), count = all - (f - ns);
    if (a) {
        a->window = L.window; a->sinks = L.sinks; a->first = first;
        a->ns = ns; a->skip = f - ns; a->count = count;
    }
    return count;
}

// Workgroups a KV head: one chunk a wave while the workgroups stay near three a CU; one workgroup for
// short caches, where the merge's launch costs more than the waves' further chunks (one token, 32 heads
// of 64, 192 keys 4.3 us, split 7.0; 512 keys 6.4 and 7.1; heads of 128, 320 keys 7.5 and 8.3, 384 keys
// 8.1 and 8.3; heads of 256, 256 keys 10.2 and 10.5, 320 keys 12.2 and 10.5); fewer chunks with an odd
// number of keys, whose loads take longer (heads of 64, 319 keys 7.7 and 8.1, 383 keys 8.7 and 8.3; heads of
// 128, 255 keys 10.6 and 10.4, 319 keys 12.6 and 10.2; heads of 256, 159 keys 9.8 and 10.6, 191 keys 15.0
// and 12.8, 255 keys 18.8 and 14.6).
void split_of(const FaLaunch &L, int *nsplit, int *cps)
{
    const int kvh = L.n_head / L.gqa, chunks = chunk_list(L, nullptr);
    const int d = std::max(L.dk, L.dv), odd = L.n_kv & 1;
    const int whole = d <= 64 ? (odd ? 10 : 16) : d <= 128 ? (odd ? 8 : 10) : odd ? 5 : 8;
    // under a window no more than the CUs hold at once, where the registers leave room for fewer than three: a second round of
    // them cost more than longer shares (8 KV heads of 256 over 6000 keys, 24 rows 28.8 us, here 19.1, one token of two heads
    // each 18.1 and 13.9; 16 KV heads, 32 rows 47.8 and 28.5; 64 rows of 16 heads of 64 21.9 and 18.7)
    const int nq = (L.gqa * L.T + 15) / 16;
    const int resident = 256 * (!L.win ? 3 : d > 128 ? 1 : nq == 1 ? 3 : d > 64 ? 2 : nq == 2 ? 3 : 2);
    const int n = chunks <= whole ? 1 : std::min({(chunks + kWaves - 1) / kWaves, std::max(1, resident / kvh), 64});
    *cps = (chunks + n - 1) / n;
    *nsplit = (chunks + *cps - 1) / *cps;
}

}  // namespace

bool flash_attn_few_rows(const FaLaunch &L)
{
    if (L.n_kv < 8 || L.dk % 32 || L.dv % 16) return false;
    // Under a window up to 32 rows, of heads of up to 64 up to 64 (in tiles of 128 rows, 8 KV heads: 20 rows of heads of 128,
    // 4001 keys 16.0 us, here 12.4, 16000 keys 24.1 and 20.0; 24 rows of heads of 256, 2000 keys 19.1 and 16.9, 16000 keys 36.2
    // and 34.2; 64 rows of heads of 64, 1000 keys 11.0 and 11.5, 16000 keys 20.1 and 17.8).
    if (L.win) return (long)L.gqa * L.T <= (std::max(L.dk, L.dv) <= 64 ? 4 : 2) * kRows;
    if ((long)L.gqa * L.T > kRows) return false;
    // One query head a KV head and long caches: the tiled kernel reads V^T in whole 128-byte lines (64
    // keys a tile, 32 here), and where its workgroups fill the CUs and nothing has to be padded it is the
    // faster one while the cache is not far larger than the memory-side cache (heads of 256, 16 x 8192
    // keys 28.9 us, here 33.0; 32 x 8192 54.8 and 62.8, 32 x 32768 212 and 200; heads of 128, 32 x 8192 28.3
    // and 30.7; 24 heads, whose 264 workgroups are two rounds, 8192 keys 69 and 48.6).
    const int d = std::max(L.dk, L.dv);
    const size_t kv = (size_t)L.n_head / L.gqa * L.n_kv * (L.dk + L.dv) * sizeof(_Float16);
    return !(L.gqa == 1 && d > 64 && L.n_kv % 8 == 0 && kv >= ((size_t)(d > 128 ? 64 : 96) << 20) && kv <= ((size_t)512 << 20) &&
             flash_attn_tiles_fill(L));
}

size_t flash_attn_rows_ws(const FaLaunch &L)
{
    int n, cps;
    split_of(L, &n, &cps);
    return n > 1 ? (size_t)n * L.n_head * L.T * (L.dv + 2) * sizeof(float) : 0;
}

hipError_t flash_attn_rows(const FaLaunch &L, hipStream_t s, uint64_t *blocks)
{
    RowArgs a;
    a.Q = L.Q; a.K = L.K; a.Vt = L.Vt; a.mask = L.mask; a.O = L.O;
    a.q_hs = L.q_hs; a.q_rs = L.q_rs; a.k_hs = L.k_hs; a.k_rs = L.k_rs; a.v_hs = L.v_hs; a.v_rs = L.v_rs;
    a.o_hs = L.o_hs; a.o_rs = L.o_rs; a.m_rs = L.m_rs;
    a.T = L.T; a.n_kv = L.n_kv; a.dk = L.dk; a.dv = L.dv; a.gqa = L.gqa; a.n_head = L.n_head;
    a.scale = L.scale; a.softcap = L.softcap;
    split_of(L, &a.nsplit, &a.cps);
    if (a.nsplit > 1 && (!L.ws || L.ws_bytes < flash_attn_rows_ws(L))) {
        a.nsplit = 1;
        a.cps = chunk_list(L, nullptr);
    }
    (void)chunk_list(L, &a);
    a.part = L.ws;
    const int kvh = L.n_head / L.gqa;
    const hipError_t e = L.win ? launch_rows<true>(a, kvh, s) : launch_rows<false>(a, kvh, s);
    if (blocks) *blocks = (uint64_t)kvh * a.nsplit;
    if (e != hipSuccess || a.nsplit == 1) return e;
    const unsigned rows = (unsigned)(L.n_head * L.T);
    hipLaunchKernelGGL(k_fa_merge, dim3(rows), dim3(256), 0, s, a.part, L.O, L.o_hs, L.o_rs, L.n_head, L.T, L.dv, a.nsplit);
    if (blocks) *blocks += rows;
    return hipGetLastError();
}

}  // namespace rk
