// f32 values of elements stored in 16 or 32 bits, and back (one rounding to nearest even); f32 arithmetic in pairs.
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

// Two f32 operations in one instruction.  A product that only a sum takes is fused with it, whatever is written: where both roundings
// matter, the product is fma2 with a negative zero that the compiler does not see.
__device__ __forceinline__ unsigned long long bits_of(float2 x) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x.x), "f"(x.y));
    return r;
}
__device__ __forceinline__ float2 pair_of(unsigned long long r) {
    float2 x;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x.x), "=f"(x.y) : "l"(r));
    return x;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
    return pair_of(r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Calls f(T()) for the element type of `dtype` (f32, f16, bf16).
template <class F>
auto with_type(int dtype, F f) {
    if (dtype == SAGE_F16) return f(__half());
    if (dtype == SAGE_BF16) return f(__nv_bfloat16());
    return f(float());
}

}  // namespace k
}  // namespace sage
