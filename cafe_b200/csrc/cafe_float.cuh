// cafe_float.cuh -- the floating types that the dense operators take, to and from fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

template <typename T> __device__ __forceinline__ float cafe_to_float(T x);
template <> __device__ __forceinline__ float cafe_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float cafe_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float cafe_to_float<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T cafe_from_float(float x);
template <> __device__ __forceinline__ float cafe_from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 cafe_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half cafe_from_float<__half>(float x) { return __float2half_rn(x); }
