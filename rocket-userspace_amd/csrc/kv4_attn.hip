// kv4_attn.hip — attention over the 4-bit cache and over fp16 keys under a window: one workgroup a
// token and head walks the keys it sees, 256 at a time, with the running maximum and sum of the softmax in
// fp32. Keys that it does not see are not read.
#include "serve.h"

#include <algorithm>

namespace rk {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ float block_reduce(float x, bool mx, float *tmp)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float y = __shfl_xor(x, o, 64);
        x = mx ? fmaxf(x, y) : x + y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = x;
    __syncthreads();
    return mx ? fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3])) : tmp[0] + tmp[1] + tmp[2] + tmp[3];
}

__device__ __forceinline__ float dequant(int code, f16x2 sm) { return (float)__builtin_fmaf16((_Float16)(float)code, sm[0], sm[1]); }

__global__ __launch_bounds__(256) void k_serve_row(const ServeAttn a)
{
    __shared__ float q[256], p[256], tmp[4];
    const int tid = threadIdx.x, t = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const size_t row = ((size_t)s * a.n_head + h) * a.n_tokens + t;
    const int n = a.seq_len ? a.seq_len[s] : a.max_kv;
    const int pos = n >= 1 && n <= a.max_kv ? n - a.n_tokens + t : -1;
    const int hk = h / a.gqa;
    const size_t hr = (size_t)s * (a.n_head / a.gqa) + hk;
    if (tid < a.dk) q[tid] = (float)a.Q[row * a.dk + tid];
    __syncthreads();
    const int lo = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0, sinks = min(a.sinks, lo);
    const int seen = pos < 0 ? 0 : sinks + pos + 1 - lo;
    float m = -1e30f, l = 0.f, o = 0.f;
    for (int i0 = 0; i0 < seen; i0 += 256) {
        const int i = i0 + tid, j = i < sinks ? i : lo + i - sinks;
        float x = -INFINITY;
        if (i < seen) {
            x = 0.f;
            if (a.Kf) {
                const _Float16 *k = a.Kf + ((size_t)hk * a.stride + j) * a.dk;
                for (int d = 0; d < a.dk; d++) x += q[d] * (float)k[d];
            } else {
                const int *code = reinterpret_cast<const int *>(a.c.kc) + (hr * a.c.cap + j) * (a.dk / 8);
                const f16x2 *sm = reinterpret_cast<const f16x2 *>(a.c.ks) + (hr * a.c.cap + j) * (a.dk / 32);
                for (int d = 0; d < a.dk; d++) x += q[d] * dequant(code[d >> 3] >> (4 * (d & 7)) & 15, sm[d >> 5]);
            }
            x *= a.scale;
            if (a.softcap != 0.f) x = a.softcap * tanhf(x / a.softcap);
        }
        const float m_new = fmaxf(m, block_reduce(x, true, tmp)), alpha = expf(m - m_new), e = expf(x - m_new);
        m = m_new;
        p[tid] = e;
        l = l * alpha + block_reduce(e, false, tmp);   // (its barriers order p too)
        o *= alpha;
        if (tid < a.dv)
            for (int c = 0; c < min(256, seen - i0); c++) {
                const int jj = i0 + c < sinks ? i0 + c : lo + i0 + c - sinks;
                float v;
                if (a.Kf) {
                    v = (float)a.Vf[((size_t)hk * a.dv + tid) * a.stride + jj];
                } else {
                    const size_t block = hr * (a.c.cap / 8) + jj / 8;
                    const int w = reinterpret_cast<const int *>(a.c.vc)[(block * (a.dv / 8) + tid / 8) * 8 + jj % 8];
                    v = dequant(w >> (4 * (tid & 7)) & 15, reinterpret_cast<const f16x2 *>(a.c.vs)[(block * (a.dv / 32) + tid / 32) * 8 + jj % 8]);
                }
                o += p[c] * v;
            }
        __syncthreads();
    }
    if (tid < a.dv) a.out[row * a.dv + tid] = (_Float16)(l == 0.f ? 0.f : o / l);
}

}  // namespace

size_t serve_attn_ws(const ServeAttn &a) { return !a.Kf && kv4_few_rows(a) ? kv4_rows_ws(a) : 0; }

hipError_t serve_attn(const ServeAttn &a, hipStream_t s, uint64_t *blocks)
{
    if (!a.Kf && kv4_few_rows(a)) return kv4_rows(a, s, blocks);
    if (a.n_seq > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_serve_row, dim3((unsigned)a.n_tokens, (unsigned)a.n_head, (unsigned)a.n_seq), dim3(256), 0, s, a);
    *blocks = (uint64_t)a.n_tokens * a.n_head * a.n_seq;
    return hipGetLastError();
}

}  // namespace rk
