// f8codes.h — eight fp32 values to e4m3 codes on the GPU, shared by the kernels that write them.
#pragma once

#include "layer.h"

namespace rk {

// The codes of v * s, clamped, rounded to nearest even.
__device__ __forceinline__ uint2 f8_codes(const float (&v)[8], float s)
{
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int d = __builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(v[4 * i] * s), f8_clamp(v[4 * i + 1] * s), 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(v[4 * i + 2] * s), f8_clamp(v[4 * i + 3] * s), d, true);
    }
    return make_uint2(w[0], w[1]);
}

// The largest size of a group's values, eight a lane over 16 lanes (NaN passed over), at least 2^-100.
__device__ __forceinline__ float f8_group_amax(const float (&v)[8])
{
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) x = fmaxf(x, fabsf(v[e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return f8_amax(x);
}

}  // namespace rk
