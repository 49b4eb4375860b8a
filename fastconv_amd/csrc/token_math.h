// Activations that the state-space operators share, in fp32.
#pragma once

#include "token_types.h"

__device__ __forceinline__ float fc_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float fc_silu(float z) { return z * fc_sigmoid(z); }
__device__ __forceinline__ float fc_silu_slope(float z) {
    const float s = fc_sigmoid(z);
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
}

// e^v good to a last place or two: the product's rounding error, which a large v makes large, goes into the result.
__device__ __forceinline__ float fc_exp(float v) {
    const float p = v * 1.44269502f, low = __builtin_fmaf(v, 1.44269502f, -p) + v * 1.92596299e-8f;      // log2(e) in two floats
    const float e = __builtin_amdgcn_exp2f(p);
    return __builtin_fabsf(p) < 130.f ? __builtin_fmaf(e, low * 0.693147181f, e) : e;      // beyond, 0 and infinity stay
}

// log(1 + e^v), exact in proportion down to e^v itself: max(v, 0) + log(1 + e), e = e^-|v| <= 1, and with s = e / (2 + e) <= 1/3
//   log(1 + e) = 2 atanh(s) = 2 s P(s^2),
// P fitted to atanh(s)/s over s^2 <= 1/9 so that the largest relative error is least: 8e-9 with these five terms.
__device__ __forceinline__ float fc_softplus(float v) {
    const float e = fc_exp(-__builtin_fabsf(v)), s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float r = __builtin_fmaf(0.140891671f, q, 0.139803007f);
    r = __builtin_fmaf(r, q, 0.200124547f);
    r = __builtin_fmaf(r, q, 0.333331585f);
    r = __builtin_fmaf(r, q, 1.f);
    return __builtin_fmaf(2.f * s, r, fmaxf(v, 0.f));      // NaN comes through s
}
