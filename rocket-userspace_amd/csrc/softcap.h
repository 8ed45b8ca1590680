// softcap.h — a soft-capped score in log2 units, for the few-row serving kernels (the tiles leave out its constant).
#pragma once

#include <hip/hip_runtime.h>

namespace rk {

// softcap tanh(x scale / softcap) log2 e, with tanh y = 1 - 2 / (1 + e^2y) from the hardware's exponential and
// reciprocal: within 2^-22 of 1, so within softcap 2^-22 of the score (a library tanh, a branch and some 40
// operations a score, was half of a call's time where every score is capped).
__device__ __forceinline__ float softcap_log2(float x, float scale, float softcap)
{
    constexpr float kLog2e = 1.4426950408889634f;
    const float e = __builtin_amdgcn_exp2f(x * (2.f * kLog2e * scale / softcap));
    return (softcap * kLog2e) * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e));
}

}  // namespace rk
