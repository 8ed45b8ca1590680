// kv4.hip — new keys and values into the 4-bit cache, and the values that it stands for.
//
// A thread takes one group of 32 values of one row: 64 bytes in (or out), and a group's 16 bytes of
// codes and its scale. Key codes of a row lie end to end; value codes come in blocks of eight keys, whose
// words (eight dims of a key) stand side by side, as the attention kernels' second product takes them.
#include "serve.h"

namespace rk {
namespace {

typedef int      i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct RowsArgs {
    Kv4View c;
    const _Float16 *K, *V;
    long k_ss, k_hs, k_rs, v_ss, v_hs, v_rs;
    _Float16 *Ko, *Vo;
    const int32_t *seq_len;
    int n_tokens, gk, g;   // groups of a key row, of both rows
    long total;
};

// One thread's group: its place, head, token, position and group (value: of the value row).
struct Item {
    int s, h, t, g;
    long j;
    bool value;
};
__device__ __forceinline__ bool item(const RowsArgs &a, Item &x)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total) return false;
    const long row = i / a.g;   // (place * heads + head) * tokens + token
    x.g = (int)(i - row * a.g);
    x.value = x.g >= a.gk;
    if (x.value) x.g -= a.gk;
    const long hr = row / a.n_tokens;
    x.t = (int)(row - hr * a.n_tokens);
    x.s = (int)(hr / a.c.heads);
    x.h = (int)(hr - (long)x.s * a.c.heads);
    x.j = (long)a.seq_len[x.s] - a.n_tokens + x.t;
    return true;
}
// The four words of the group's codes and its scale.
__device__ __forceinline__ void at(const Kv4View &c, const Item &x, int *&code, int &step, f16x2 *&sm)
{
    const size_t hr = (size_t)x.s * c.heads + x.h;
    if (x.value) {
        const size_t block = hr * (c.cap / 8) + x.j / 8;
        code = reinterpret_cast<int *>(c.vc) + (block * (c.dv / 8) + 4 * x.g) * 8 + x.j % 8;
        step = 8;
        sm = reinterpret_cast<f16x2 *>(c.vs) + (block * (c.dv / 32) + x.g) * 8 + x.j % 8;
    } else {
        const size_t row = hr * c.cap + x.j;
        code = reinterpret_cast<int *>(c.kc) + row * (c.dk / 8) + 4 * x.g;
        step = 1;
        sm = reinterpret_cast<f16x2 *>(c.ks) + row * (c.dk / 32) + x.g;
    }
}

__global__ __launch_bounds__(256) void k_kv4_append(const RowsArgs a)
{
    Item x;
    if (!item(a, x) || x.j < 0 || x.j >= a.c.capacity) return;
    const _Float16 *src = x.value ? a.V + x.s * a.v_ss + x.h * a.v_hs + x.t * a.v_rs : a.K + x.s * a.k_ss + x.h * a.k_hs + x.t * a.k_rs;
    float v[32], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f16x8 w = reinterpret_cast<const f16x8 *>(src + 32 * x.g)[i];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[8 * i + e] = kv4_finite((float)w[e]);
            lo = fminf(lo, v[8 * i + e]);
            hi = fmaxf(hi, v[8 * i + e]);
        }
    }
    lo += 0.f;   // (-0 becomes 0)
    const _Float16 s = kv4_scale(lo, hi);
    int *code, step;
    f16x2 *sm;
    at(a.c, x, code, step, sm);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        int w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= kv4_code(v[8 * i + e], lo, (float)s) << (4 * e);
        code[i * step] = w;
    }
    *sm = f16x2{s, (_Float16)lo};
}

__global__ __launch_bounds__(256) void k_kv4_read(const RowsArgs a)
{
    Item x;
    if (!item(a, x)) return;
    _Float16 *dst = x.value ? a.Vo : a.Ko;
    if (!dst) return;
    const size_t row = ((size_t)x.s * a.c.heads + x.h) * a.n_tokens + x.t;
    dst += row * (x.value ? a.c.dv : a.c.dk) + 32 * x.g;
    const bool in = x.j >= 0 && x.j < a.c.capacity;
    int *code = nullptr, step = 0;
    f16x2 *sm = nullptr, y = {(_Float16)0.f, (_Float16)0.f};
    if (in) {
        at(a.c, x, code, step, sm);
        y = *sm;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int w = in ? code[i * step] : 0;
        f16x8 o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = __builtin_fmaf16((_Float16)(float)(w >> (4 * e) & 15), y[0], y[1]);
        reinterpret_cast<f16x8 *>(dst)[i] = o;
    }
}

bool fill(const Kv4View &c, const Kv4Rows &r, RowsArgs &a, unsigned *blocks)
{
    a.c = c;
    a.K = r.K; a.V = r.V; a.Ko = r.Ko; a.Vo = r.Vo; a.seq_len = r.seq_len; a.n_tokens = r.n_tokens;
    a.k_ss = r.k_ss; a.k_hs = r.k_hs; a.k_rs = r.k_rs; a.v_ss = r.v_ss; a.v_hs = r.v_hs; a.v_rs = r.v_rs;
    a.gk = c.dk / 32;
    a.g = a.gk + c.dv / 32;
    a.total = (long)c.n_seq * c.heads * r.n_tokens * a.g;
    const long n = (a.total + 255) / 256;
    *blocks = (unsigned)n;
    return n <= 0x7FFFFFFFL;
}

}  // namespace

hipError_t kv4_append(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks)
{
    RowsArgs a;
    unsigned n;
    if (!fill(c, r, a, &n)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv4_append, dim3(n), dim3(256), 0, s, a);
    *blocks = n;
    return hipGetLastError();
}

hipError_t kv4_read(const Kv4View &c, const Kv4Rows &r, hipStream_t s, uint64_t *blocks)
{
    RowsArgs a;
    unsigned n;
    if (!fill(c, r, a, &n)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv4_read, dim3(n), dim3(256), 0, s, a);
    *blocks = n;
    return hipGetLastError();
}

}  // namespace rk
