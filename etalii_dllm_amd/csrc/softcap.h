// The soft cap's tanh.
#pragma once

#include <hip/hip_runtime.h>

namespace dllm_hip {

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// tanh to about 6 x 2^-24 of itself: z (945 + 105 z^2 + z^4) / (945 + 420 z^2 + 15 z^4), Lambert's continued fraction cut after
// five levels, where |z| < 1/2 (off by 2^-27), else 1 - 2 / (1 + e^2|z|); and its derivative, right where |tanh| is near one too.
__device__ __forceinline__ float tanh_of_any_size(float z, float& derivative) {
    const float w = z * z;
    const float near = z * fmaf(w + 105.0f, w, 945.0f) * __builtin_amdgcn_rcpf(fmaf(fmaf(15.0f, w, 420.0f), w, 945.0f));
    const float tail = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(2.0f * kLog2E * fabsf(z)));  // (1 - tanh |z|) / 2
    const bool is_near = fabsf(z) < 0.5f;
    derivative = is_near ? fmaf(-near, near, 1.0f) : 4.0f * fmaf(-tail, tail, tail);
    return is_near ? near : copysignf(fmaf(-2.0f, tail, 1.0f), z);
}

}  // namespace dllm_hip
