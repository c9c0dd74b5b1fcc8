// f32 values of elements stored in 16 or 32 bits, and back (one rounding to nearest even).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../../include/sage_cuda.h"

namespace sage {
namespace k {

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T narrowed(float x);
template <>
__device__ __forceinline__ float narrowed<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half narrowed<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrowed<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 bytes of elements
template <class T>
struct alignas(16) Pack {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// Calls f(T()) for the element type of `dtype` (f32, f16, bf16).
template <class F>
auto with_type(int dtype, F f) {
    if (dtype == SAGE_F16) return f(__half());
    if (dtype == SAGE_BF16) return f(__nv_bfloat16());
    return f(float());
}

}  // namespace k
}  // namespace sage
