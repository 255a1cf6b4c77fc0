// cap tanh(s / cap) of a score s, as cap (1 - 2 / (1 + exp(2 s / cap))). That is good to 2^-22 of the cap, which is nothing beside a score of its
// size and everything beside a small one: where the cap is above kCapNear (2^-16 at most: a thirtieth of what rounding a weight to fp16 costs),
// scores of up to kCapSmall of it go by a polynomial, whose error goes with the score.
#pragma once
#include <cuda_runtime.h>

namespace tdist {

// tanh(z) / z = sum of kCapC[i] z^(2 i) for |z| <= kCapSmall: fitted to the least largest relative error, 9.1e-8 (1.8e-7 with fp32's roundings)
constexpr float kCapNear = 64.f, kCapSmall = 0.6f;
constexpr float kCapC0 = 0.9999999403953552f, kCapC1 = -0.33332309126853943f, kCapC2 = 0.13310173153877258f, kCapC3 = -0.05210148170590401f,
                kCapC4 = 0.01547542680054903f;

// z = s / cap, |z| <= kCapSmall; `s` in any unit
__device__ __forceinline__ float soft_cap_small(float s, float z) {
    const float u = z * z;
    return s * fmaf(fmaf(fmaf(fmaf(u, kCapC4, kCapC3), u, kCapC2), u, kCapC1), u, kCapC0);
}
// by the exponential; `cap` in the unit wanted. NaN stays NaN.
__device__ __forceinline__ float soft_cap_far(float z, float cap) {
    return cap - __fdividef(2.f * cap, 1.f + exp2f(z * (2.f * 1.4426950408889634f)));
}
// any z
__device__ __forceinline__ float soft_cap(float s, float z, float cap) {
    const float far = soft_cap_far(z, cap);
    return fabsf(z) <= kCapSmall ? soft_cap_small(s, z) : far;
}

}  // namespace tdist
