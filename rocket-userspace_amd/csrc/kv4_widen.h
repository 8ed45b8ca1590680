// kv4_widen.h — codes of the 4-bit cache as halves, the values that rocket_kv4_read_fp16 gives.
#pragma once

#include <hip/hip_runtime.h>

namespace rk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

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
    // A word's eight codes in the order 0 4 1 5 2 6 3 7, with one scale and minimum.
    __device__ __forceinline__ f16x8 eight(unsigned w, f16x2 sm) const
    {
        const f16x2 s = {sm[0], sm[0]}, m = {sm[1], sm[1]};
        f16x8 r;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const f16x2 x = at(w, e, s, m);
            r[2 * e] = x[0];
            r[2 * e + 1] = x[1];
        }
        return r;
    }
};

}  // namespace rk
