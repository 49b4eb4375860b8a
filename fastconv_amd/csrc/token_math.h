// Activations that the state-space operators share, in fp32.
#pragma once

#include "token_types.h"

__device__ __forceinline__ float fc_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float fc_silu(float z) { return z * fc_sigmoid(z); }
__device__ __forceinline__ float fc_silu_slope(float z) {
    const float s = fc_sigmoid(z);
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
}

// log(1 + e^v), exact in proportion down to e^v itself (within 2.8e-7): max(v, 0) + log(1 + e), e = e^-|v| <= 1.  With u = 1 + e rounded to a float, log(1 + e) is
// log(u) + (e - (u - 1)) / u, and where what the rounding lost is of any weight, u is near 1.  v_log_f32 over all floats from 1 to 2 is off by at most 1.15e-7 of
// its result, also next to 1.  The exponent of e is formed in two floats: its rounding, which a large v makes large, would go into the result.
__device__ __forceinline__ float fc_softplus(float v) {
    const float a = fminf(__builtin_fabsf(v), 150.f);      // e^-150 is 0 already
    const float p = a * -1.44269502f, low = __builtin_fmaf(a, -1.92596299e-8f, __builtin_fmaf(a, -1.44269502f, -p));      // log2(e) in two floats
    const float e0 = __builtin_amdgcn_exp2f(p), e = __builtin_fmaf(e0, low * 0.693147181f, e0);
    const float u = 1.f + e, lost = e - (u - 1.f);
    return __builtin_fmaf(__builtin_amdgcn_logf(u), 0.693147181f, lost) + (v < 0.f ? 0.f : v);      // NaN stays
}
