// kv4_widen.h — codes of the 4-bit cache as the halves that matrix products take.
//
// A cached value is code * scale + minimum. Rounded to a half each, keys and values put results of attention 3.4e-4 of their
// size off, and the weights' own rounding 4e-4, where 2.1e-4 is the fp16 result's. So of the three only values are
// rounded (2.8e-4): as rocket_kv4_read_fp16 gives them, three operations a pair. A weight goes as two halves, itself and what its rounding
// left, into two products. And so does a key's code times its scale, 4 bits by 11, which two halves hold
// exactly: the product rounded, and the rest, which a fused operation gives. Keys' minimums, one for 32 dims, make a small product of their
// own: q . minimum is the sum over the groups of their minimum times the query's sum there.
#pragma once

#include <hip/hip_runtime.h>

namespace rk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short    i16x2 __attribute__((ext_vector_type(2)));

// ---- values ----
// Two codes a step, at the same place of a word's two halves: bits 0-3 (E = 0) or 4-7 (E = 1; a word moved down by eight
// has its other two there). Or-ing in the bits of 1024 makes the half 1024 + c, or 1024 + 16 c, which an exact
// packed operation turns into c; then times the scale plus the minimum, one rounding: three operations for two
// values, and a move for eight. (The masks are kept in vector registers: as literals and and or were two operations.)
struct Widen {
    unsigned low = 0x000F000Fu, high = 0x00F000F0u, base = 0x64006400u;
    __device__ __forceinline__ Widen() { asm volatile("" : "+v"(low), "+v"(high), "+v"(base)); }
    template <int E> __device__ __forceinline__ f16x2 two(unsigned w, f16x2 s, f16x2 m) const
    {
        const unsigned bits = (w & (E ? high : low)) | base;
        const f16x2 x = __builtin_bit_cast(f16x2, bits);
        const f16x2 c = E ? __builtin_elementwise_fma(x, f16x2{(_Float16)0.0625f, (_Float16)0.0625f}, f16x2{(_Float16)-64.f, (_Float16)-64.f})
                          : x - f16x2{(_Float16)1024.f, (_Float16)1024.f};
        return __builtin_elementwise_fma(c, s, m);
    }
    // The same with the place as a number that unrolling makes constant: 0 to 3 of a half.
    __device__ __forceinline__ f16x2 at(unsigned w, int place, f16x2 s, f16x2 m) const
    {
        const unsigned x = place & 2 ? w >> 8 : w;
        return place & 1 ? two<1>(x, s, m) : two<0>(x, s, m);
    }
};

// ---- keys ----
struct HiLo { f16x8 hi, lo; };
// A key's scale, and that which hi is made with: half of it where a code times the scale may pass the largest fp16 (15 * 4364
// does not). hi and lo are then about equal, and lo's rounding, half a step of half the product, stays.
struct KeyScale {
    f16x2 s, first;
    __device__ __forceinline__ explicit KeyScale(_Float16 x) : s{x, x}
    {
        const _Float16 y = x > (_Float16)4364.f ? x * (_Float16)0.5f : x;
        first = f16x2{y, y};
    }
};
// A word's eight codes in the order 0 2 4 6 1 3 5 7: hi + lo = code * scale. A byte of 0 to 15 is, as an 8-bit float (e4m3, whose
// subnormals and first normals are one line), 2^-9 times itself: one conversion makes two halves of two bytes.
__device__ __forceinline__ HiLo kv4_keys(unsigned w, const KeyScale &k)
{
    HiLo r;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const unsigned bytes = (e < 2 ? w : w >> 4) & 0x0F0F0F0Fu;
        const f16x2 c = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, false);
        const f16x2 hi = c * k.first, lo = __builtin_elementwise_fma(c, k.s, -hi);
        r.hi[2 * e] = hi[0];
        r.hi[2 * e + 1] = hi[1];
        r.lo[2 * e] = lo[0];
        r.lo[2 * e + 1] = lo[1];
    }
    return r;
}
__device__ __forceinline__ f16x8 kv4_query_order(f16x8 q) { return __builtin_shufflevector(q, q, 0, 2, 4, 6, 1, 3, 5, 7); }

// A query's sums as two halves, for the products with the minimums: hi + lo = 2^-e sum, to 2^-22 of `most`, the largest of their
// sizes. e is 0 where halves hold them so, else it takes `most` to just below 2^14. The product is taken back by 2^e.
__device__ __forceinline__ float kv4_sum(f16x8 q, float sum)
{
#pragma unroll
    for (int i = 0; i < 8; i += 2) sum = __builtin_amdgcn_fdot2(f16x2{q[i], q[i + 1]}, f16x2{(_Float16)1.f, (_Float16)1.f}, sum, false);
    return sum;
}
__device__ __forceinline__ int kv4_sum_exponent(float most) { return most >= 0.125f && most < 16384.f ? 0 : __builtin_amdgcn_frexp_expf(most) - 14; }
__device__ __forceinline__ f16x2 kv4_sum_halves(float sum, int e)
{
    const float x = __builtin_amdgcn_ldexpf(sum, -e);
    const _Float16 hi = (_Float16)x;
    return f16x2{hi, (_Float16)(x - (float)hi)};
}

}  // namespace rk
