// Element types of the operators on tokens: fp32, bf16 and IEEE half in memory, fp32 in registers.
#pragma once

#include <hip/hip_runtime.h>

#include "fc_internal.h"

template <int DT>
struct fc_elem;
template <>
struct fc_elem<FC_F32> {
    typedef float type;
};
template <>
struct fc_elem<FC_BF16> {
    typedef __bf16 type;
};
template <>
struct fc_elem<FC_F16> {
    typedef _Float16 type;
};

// VEC elements that lie side by side, aligned to their whole size: one access.
template <int DT, int VEC>
struct alignas(VEC * sizeof(typename fc_elem<DT>::type)) fc_vec {
    typename fc_elem<DT>::type v[VEC];
    __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
    // round to nearest, ties to even: the one rounding of a result
    __device__ __forceinline__ void set(int i, float x) { v[i] = (typename fc_elem<DT>::type)x; }
};

// Accesses of global memory through a pointer that the compiler cannot follow to a kernel argument, and would take for one that may point
// into LDS.
template <class V>
__device__ __forceinline__ V fc_load_global(const void *p) {
    typedef __attribute__((address_space(1))) const V global;
    return *(const V *)(global *)(uintptr_t)p;
}
template <class V>
__device__ __forceinline__ void fc_store_global(void *p, const V &v) {
    typedef __attribute__((address_space(1))) V global;
    *(V *)(global *)(uintptr_t)p = v;
}

static inline size_t fc_elem_size(int dtype) { return dtype == FC_F32 ? 4 : 2; }
static inline bool fc_dtype_ok(int dtype) { return dtype == FC_F32 || dtype == FC_BF16 || dtype == FC_F16; }

// The widest access, in elements, up to 16 bytes, that `bits` (element counts and strides joined by or) and the byte addresses
// `addr` (joined by or) are multiples of.
static inline int fc_widest(int dtype, uint64_t bits, uint64_t addr) {
    const int es = (int)fc_elem_size(dtype);
    int v = 16 / es;
    while (v > 1 && ((bits & (uint64_t)(v - 1)) || (addr & (uint64_t)(v * es - 1)))) v >>= 1;
    return v;
}

// a * b * c as a count that fits 62 bits, or -1
static inline long fc_count(long a, long b, long c = 1) {
    const __int128 p = (__int128)a * b * c;
    return p < 0 || p > ((__int128)1 << 62) ? -1 : (long)p;
}

// Rows of so many elements, n of them a stride apart, share none.
static inline bool fc_apart(long n, long stride, long row) { return n < 2 || stride >= row; }

__device__ __forceinline__ float fc_wave_sum(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
