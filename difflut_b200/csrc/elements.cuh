// Element types (fp32 / bf16 / fp16) and aligned vectors shared by the kernels that take more than one type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

// N elements of T that are loaded and stored as one access (N * sizeof(T) is 2, 4, 8 or 16 bytes; 32 are two)
template <typename T, int N>
struct __align__(sizeof(T) * N < 16 ? sizeof(T) * N : 16) DlVec {
    T v[N];
};

__device__ __forceinline__ float dl_to_float(float x) { return x; }
__device__ __forceinline__ float dl_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float dl_to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T dl_from_float(float x);
template <>
__device__ __forceinline__ float dl_from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 dl_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half dl_from_float<__half>(float x) { return __float2half_rn(x); }

// A whole vector to and from fp32; 16-bit types go through the two-element conversions (one instruction a pair).
template <int N>
__device__ __forceinline__ void dl_unpack(const DlVec<float, N>& x, float (&f)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = x.v[e];
}
template <int N>
__device__ __forceinline__ void dl_unpack(const DlVec<__nv_bfloat16, N>& x, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = __bfloat162float(x.v[0]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 p = __bfloat1622float2(__nv_bfloat162(x.v[e], x.v[e + 1]));
            f[e] = p.x;
            f[e + 1] = p.y;
        }
    }
}
template <int N>
__device__ __forceinline__ void dl_unpack(const DlVec<__half, N>& x, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = __half2float(x.v[0]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 p = __half22float2(__half2(x.v[e], x.v[e + 1]));
            f[e] = p.x;
            f[e + 1] = p.y;
        }
    }
}
template <int N>
__device__ __forceinline__ void dl_pack(const float (&f)[N], DlVec<float, N>& x) {
#pragma unroll
    for (int e = 0; e < N; ++e) x.v[e] = f[e];
}
template <int N>
__device__ __forceinline__ void dl_pack(const float (&f)[N], DlVec<__nv_bfloat16, N>& x) {
    if constexpr (N == 1) {
        x.v[0] = __float2bfloat16_rn(f[0]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(f[e], f[e + 1]);
            x.v[e] = p.x;
            x.v[e + 1] = p.y;
        }
    }
}
template <int N>
__device__ __forceinline__ void dl_pack(const float (&f)[N], DlVec<__half, N>& x) {
    if constexpr (N == 1) {
        x.v[0] = __float2half_rn(f[0]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const __half2 p = __floats2half2_rn(f[e], f[e + 1]);
            x.v[e] = p.x;
            x.v[e + 1] = p.y;
        }
    }
}

// element `i` of an array whose type is one of DL_DTYPE_*, as fp32
__device__ __forceinline__ float dl_load_as_float(const void* p, int dtype, int64_t i) {
    if (dtype == DL_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == DL_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void dl_store_from_float(void* p, int dtype, int64_t i, float x) {
    if (dtype == DL_DTYPE_F32) static_cast<float*>(p)[i] = x;
    else if (dtype == DL_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

static inline bool dl_dtype_known(int64_t dtype) { return dtype >= DL_DTYPE_F32 && dtype <= DL_DTYPE_F16; }
static inline int64_t dl_dtype_size(int64_t dtype) { return dtype == DL_DTYPE_F32 ? 4 : 2; }

// Widest vector (elements, a power of two, at most 16 bytes) that every row of `row_elements` elements at
// every given address can be cut into.
static inline int dl_vector_width(int64_t element_size, int64_t row_elements, uintptr_t addresses_or) {
    int64_t width = 16 / element_size;
    while (width > 1 && (row_elements % width != 0 || addresses_or % (uintptr_t)(width * element_size) != 0)) width /= 2;
    return (int)width;
}

static inline uintptr_t dl_address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
