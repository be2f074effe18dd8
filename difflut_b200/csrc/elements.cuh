// Element types (fp32 / bf16 / fp16) and aligned vectors shared by the kernels that take more than one type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

// N elements of T that are loaded and stored as one access (N * sizeof(T) is 2, 4, 8 or 16 bytes)
template <typename T, int N>
struct __align__(sizeof(T) * N) DlVec {
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
