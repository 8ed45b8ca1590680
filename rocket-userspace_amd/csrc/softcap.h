// softcap.h — scores of the serving kernels: soft-caps, softcap tanh(score / softcap), and what maxima are lifted by.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

namespace rk {

// tanh y = 1 - 2 / (1 + e^2y) from the hardware's exponential and reciprocal is within 2^-22 of 1, so a capped score is off
// by up to softcap 2^-22, however small it is itself: 2^-16 at this cap, well below the weights' 2^-11, and
// without bound above it. Caps up to it take that form (a library tanh, a branch and some 40 operations a score, was
// half of a call's time where every score is capped); larger ones softcap_wide().
constexpr float kNarrowCap = 64.f;
enum Cap { kUncapped, kNarrow, kWide };
inline Cap cap_of(float softcap) { return softcap == 0.f ? kUncapped : fabsf(softcap) <= kNarrowCap ? kNarrow : kWide; }

// What takes a product q . k to 2 y log2 e (finite, so that a product of 0 stays one under a cap next to 0).
__device__ __forceinline__ float cap_slope(float scale, float softcap)
{
    const float k = 2.f * 1.4426950408889634f * scale / softcap;
    return fmaxf(fminf(k, 3e38f), -3e38f);
}

// A scaled score under a cap above kNarrowCap (inv = 1 / cap), to 2^-20 of itself: below |y| = 0.35 by tanh's series,
// y - y^3 / 3 + 2 y^5 / 15 - 17 y^7 / 315 + 62 y^9 / 2835 (the next term 2.5e-7 of it), which leaves a score far below its
// cap as it is, and from there on by the form above (terms that round to 1.7 2^-23, of 0.336 or more).
__device__ __forceinline__ float softcap_wide(float s, float inv, float cap)
{
    const float y = s * inv, y2 = y * y;
    const float series = fmaf(s * y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3), s);
    const float far = cap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * 2.885390081777927f)));
    return fabsf(y) < 0.35f ? series : far;
}

// A product q . k as a capped score in log2 units, for the few-row kernels (the tiles leave out the constant).
template <Cap CAP> __device__ __forceinline__ float softcap_log2(float x, float scale, float softcap)
{
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (CAP == kWide) return softcap_wide(x * scale, 1.f / softcap, softcap) * kLog2e;
    const float e = __builtin_amdgcn_exp2f(x * cap_slope(scale, softcap));
    return (softcap * kLog2e) * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e));
}

// The same for a row's largest product, times `unit` the score, by the product that the exponential takes, unrounded: 15 or 10
// below it, whichever is within what a weight may grow to, or (from scores of 2^27 on, maybe) the score itself.
__device__ __forceinline__ float lifted(float mx, float unit)
{
    float m = fmaf(mx, unit, -15.f);
    if (fmaf(mx, unit, -m) > 15.25f) {
        m = fmaf(mx, unit, -10.f);
        if (fmaf(mx, unit, -m) > 15.25f) m = mx * unit;
    }
    return m;
}

// What a row's largest score, in log2 units, is taken down by so that its weight is 2^15: fp16 then loses those alone
// below 2^-40 of the largest. (Not taken down where the difference would round to more, from scores of 2^24 on.)
__device__ __forceinline__ float lifted(float mx)
{
    const float m = mx - 15.f;
    return mx - m > 15.5f ? mx : m;
}

}  // namespace rk
