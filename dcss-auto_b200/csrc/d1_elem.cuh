// Element types of the operators that take 32- and 16-bit rows: conversion to
// and from fp32 (every sum is held in fp32), and vectors of elements for wide
// loads and stores. Rounding to 16 bits is to nearest, once, on the store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/d1.h"

namespace d1 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <class T, int N> struct alignas(sizeof(T) * N) Elems { T v[N]; };

// Sum over the warp (every lane gets it); the order is fixed.
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// Whether every pointer is a multiple of `bytes` (NULL is).
template <class... P> inline bool aligned_to(int bytes, const P *...p) {
    return ((reinterpret_cast<uintptr_t>(p) | ...) & (uintptr_t)(bytes - 1)) == 0;
}
inline bool element_aligned(const void *p, int type) { return aligned_to(type == D1_TYPE_F32 ? 4 : 2, p); }
inline bool type_ok(int type) { return type == D1_TYPE_F32 || type == D1_TYPE_BF16 || type == D1_TYPE_F16; }

}  // namespace d1
