// Element types of the layer operators: conversion to and from fp32 (rounding to nearest), and vectors of them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ringrnn {

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float up(__half x) { return __half2float(x); }
template <class E>
__device__ __forceinline__ E down(float x);
template <>
__device__ __forceinline__ float down<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half down<__half>(float x) { return __float2half_rn(x); }

// two at a time: one conversion and no packing
template <class E>
__device__ __forceinline__ void down2(float a, float b, E* to) { to[0] = a, to[1] = b; }
template <>
__device__ __forceinline__ void down2<__nv_bfloat16>(float a, float b, __nv_bfloat16* to) {
  const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
  to[0] = y.x, to[1] = y.y;
}
template <>
__device__ __forceinline__ void down2<__half>(float a, float b, __half* to) {
  const __half2 y = __floats2half2_rn(a, b);
  to[0] = y.x, to[1] = y.y;
}

template <class E, int V>
struct alignas(sizeof(E) * V) Pack {
  E v[V];
};

}  // namespace ringrnn
