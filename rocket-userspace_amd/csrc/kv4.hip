// kv4.hip — new keys and values into the 4-bit cache, and the values that it stands for.
//
// Four lanes take a group of 32 values of one row, eight values each: 16 bytes in (or out) a lane, a word of
// codes, and the group's scale. The lanes of a wave are laid out as the bytes lie: a key row's groups end to end, and of
// values eight tokens of a group side by side, whose words the cache keeps together. (A thread a group, which found its row
// by three 64-bit divisions and divided 32 times, took 25 us for the prompt below; its reading 18.) 4096 tokens of 8 heads of
// 256, 44 MB each: append 14.0 us by trace (3.1 TB/s), read 10.5 us (4.2 TB/s); one token of 32 sequences 4.0 and 3.0.
// The issue of VALU operations bounds append: by counters 210 a wave, 26 a value with the addresses, the extremes and the
// scale, 26.8 thousand cycles of a SIMD, 11.2 us. Reading has 107 a wave, 5.7 us, and is bound by memory.
#include "serve.h"

namespace rk {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct RowsArgs {
    Kv4View c;
    const _Float16 *K, *V;
    long k_ss, k_hs, k_rs, v_ss, v_hs, v_rs;
    _Float16 *Ko, *Vo;
    const int32_t *seq_len;
    int n_tokens, k_blocks;   // workgroups of a head that take key rows; the others take values
};

// A quad's group, and where its codes and scale lie in the cache.
struct Item {
    int s, h, t, g, e;   // place, head, token, group, the lane's word of the group
    bool value;
    long j;              // position
    size_t code, sm;     // word and scale, in words from the part's start
};
__device__ __forceinline__ bool item(const RowsArgs &a, Item &x)
{
    x.value = (int)blockIdx.x >= a.k_blocks;
    const unsigned q = (blockIdx.x - (x.value ? a.k_blocks : 0)) * 64 + (threadIdx.x >> 2);
    const unsigned groups = (x.value ? a.c.dv : a.c.dk) / 32;
    x.s = blockIdx.z;
    x.h = blockIdx.y;
    x.e = threadIdx.x & 3;
    if (x.value) {
        const unsigned y = q >> 3, tb = y / groups;
        x.g = (int)(y - tb * groups);
        x.t = (int)(8 * tb + (q & 7));
    } else {
        x.t = (int)(q / groups);
        x.g = (int)(q - x.t * groups);
    }
    if (x.t >= a.n_tokens) return false;
    x.j = (long)a.seq_len[x.s] - a.n_tokens + x.t;
    const size_t hr = (size_t)x.s * a.c.heads + x.h;
    if (x.value) {
        const size_t block = hr * (a.c.cap / 8) + x.j / 8;
        x.code = (block * (a.c.dv / 8) + 4 * x.g + x.e) * 8 + x.j % 8;
        x.sm = (block * groups + x.g) * 8 + x.j % 8;
    } else {
        const size_t row = hr * a.c.cap + x.j;
        x.code = row * (a.c.dk / 8) + 4 * x.g + x.e;
        x.sm = row * groups + x.g;
    }
    return true;
}

// A value of the four lanes' that share a group.
template <class F> __device__ __forceinline__ float quad(float x, F f)
{
    x = f(x, __shfl_xor(x, 1, 64));
    return f(x, __shfl_xor(x, 2, 64));
}

__global__ __launch_bounds__(256) void k_kv4_append(const RowsArgs a)
{
    Item x;
    if (!item(a, x) || x.j < 0 || x.j >= a.c.capacity) return;   // (the same for a group's four lanes)
    const _Float16 *src = x.value ? a.V + x.s * a.v_ss + x.h * a.v_hs + x.t * a.v_rs : a.K + x.s * a.k_ss + x.h * a.k_hs + x.t * a.k_rs;
    f16x8 w = *reinterpret_cast<const f16x8 *>(src + 32 * x.g + 8 * x.e);
    const u32x4 bits = __builtin_bit_cast(u32x4, w);
    unsigned odd = 0;   // an exponent of all ones carries into the sign's place
#pragma unroll
    for (int i = 0; i < 4; i++) odd |= ((bits[i] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
    if (odd) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (_Float16)kv4_finite((float)w[i]);
    }
    float v[8], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = (float)w[i];
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
    lo = quad(lo, [](float p, float q) { return fminf(p, q); }) + 0.f;   // (-0 becomes 0)
    hi = quad(hi, [](float p, float q) { return fmaxf(p, q); });
    const _Float16 s = kv4_scale(lo, hi);
    // Codes by the hardware's reciprocal: (x - lo) / s to 2^-18, rounded as the sum with 2^23 rounds (to even), whose low
    // bits are the code. That is the division's code wherever the quotient is not within 2^-14 of a half; there, and
    // for a subnormal scale (its rounding may reach past 15), the division itself.
    const float r = __builtin_amdgcn_rcpf((float)s);
    float far = 0.f;
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float d = v[i] - lo, c = fmaf(d, r, 0x1p23f);
        far = fmaxf(far, fabsf(fmaf(d, r, 0x1p23f - c)));
        word |= (__builtin_bit_cast(unsigned, c) & 15u) << (4 * i);
    }
    if (!(far < 0.5f - 0x1p-14f) || (float)s < 0x1p-14f) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) word |= (unsigned)kv4_code(v[i], lo, (float)s) << (4 * i);
    }
    reinterpret_cast<unsigned *>(x.value ? a.c.vc : a.c.kc)[x.code] = word;
    if (x.e == 0) reinterpret_cast<f16x2 *>(x.value ? a.c.vs : a.c.ks)[x.sm] = f16x2{s, (_Float16)lo};
}

__global__ __launch_bounds__(256) void k_kv4_read(const RowsArgs a)
{
    Item x;
    if (!item(a, x)) return;
    _Float16 *dst = x.value ? a.Vo : a.Ko;
    if (!dst) return;
    unsigned w = 0;
    f16x2 y = {(_Float16)0.f, (_Float16)0.f};
    if (x.j >= 0 && x.j < a.c.capacity) {
        w = reinterpret_cast<const unsigned *>(x.value ? a.c.vc : a.c.kc)[x.code];
        y = reinterpret_cast<const f16x2 *>(x.value ? a.c.vs : a.c.ks)[x.sm];
    }
    f16x8 o;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = __builtin_fmaf16((_Float16)(float)(w >> (4 * i) & 15), y[0], y[1]);
    const size_t row = ((size_t)x.s * a.c.heads + x.h) * a.n_tokens + x.t;
    *reinterpret_cast<f16x8 *>(dst + row * (x.value ? a.c.dv : a.c.dk) + 32 * x.g + 8 * x.e) = o;
}

// The arguments and the grid: key workgroups then value workgroups of 64 groups, heads, places.
bool fill(const Kv4View &c, const Kv4Rows &r, RowsArgs &a, dim3 *grid)
{
    a.c = c;
    a.K = r.K; a.V = r.V; a.Ko = r.Ko; a.Vo = r.Vo; a.seq_len = r.seq_len; a.n_tokens = r.n_tokens;
    a.k_ss = r.k_ss; a.k_hs = r.k_hs; a.k_rs = r.k_rs; a.v_ss = r.v_ss; a.v_hs = r.v_hs; a.v_rs = r.v_rs;
    const long kg = (long)r.n_tokens * (c.dk / 32), vg = ((long)r.n_tokens + 7) / 8 * 8 * (c.dv / 32);   // at most 2^26 each
    a.k_blocks = (int)((kg + 63) / 64);
    *grid = dim3((unsigned)(a.k_blocks + (vg + 63) / 64), (unsigned)c.heads, (unsigned)c.n_seq);
    return c.heads <= 65535 && c.n_seq <= 65535;
}

}  // namespace

hipError_t kv4_append(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks)
{
    RowsArgs a;
    dim3 grid;
    if (!fill(c, r, a, &grid)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv4_append, grid, dim3(256), 0, s, a);
    *blocks = (uint64_t)grid.x * grid.y * grid.z;
    return hipGetLastError();
}

hipError_t kv4_read(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks)
{
    RowsArgs a;
    dim3 grid;
    if (!fill(c, r, a, &grid)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv4_read, grid, dim3(256), 0, s, a);
    *blocks = (uint64_t)grid.x * grid.y * grid.z;
    return hipGetLastError();
}

}  // namespace rk
