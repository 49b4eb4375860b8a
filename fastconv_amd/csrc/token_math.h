// Activations that the state-space operators share, in fp32.
#pragma once

#include "token_types.h"

__device__ __forceinline__ float fc_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float fc_silu(float z) { return z * fc_sigmoid(z); }
__device__ __forceinline__ float fc_silu_slope(float z) {
    const float s = fc_sigmoid(z);
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
}

// log(1 + e^v), exact in proportion down to e^v itself: max(v, 0) + log(1 + e), e = e^-|v| <= 1, and with s = e / (2 + e) <= 1/3
//   log(1 + e) = 2 atanh(s) = 2 s P(s^2),
// P fitted to atanh(s)/s over s^2 <= 1/9 so that the largest relative error is least: 8e-9 with these five terms.  The exponent of e is formed in two floats: its
// rounding, which a large v makes large, would go into the result.
__device__ __forceinline__ float fc_softplus(float v) {
    const float a = fminf(__builtin_fabsf(v), 150.f);      // e^-150 is 0 already
    const float p = a * -1.44269502f, low = __builtin_fmaf(a, -1.92596299e-8f, __builtin_fmaf(a, -1.44269502f, -p));      // log2(e) in two floats
    const float e0 = __builtin_amdgcn_exp2f(p), e = __builtin_fmaf(e0, low * 0.693147181f, e0);
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float r = __builtin_fmaf(0.140891671f, q, 0.139803007f);
    r = __builtin_fmaf(r, q, 0.200124547f);
    r = __builtin_fmaf(r, q, 0.333331585f);
    r = __builtin_fmaf(r, q, 1.f);
    return __builtin_fmaf(2.f * s, r, v < 0.f ? 0.f : v);      // NaN stays
}
