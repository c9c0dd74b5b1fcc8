// Eight neighbouring elements in 16 or 32 bits each, as four pairs of f32 values and back.
#pragma once
#include "narrow.h"

namespace sage {
namespace k {

template <class T>
__device__ __forceinline__ float2 pair_at(const Pack<T> &p, int i) { return make_float2(widen(p.v[2 * i]), widen(p.v[2 * i + 1])); }
template <>
__device__ __forceinline__ float2 pair_at<__nv_bfloat16>(const Pack<__nv_bfloat16> &p, int i) {
    const unsigned u = ((const unsigned *)&p)[i];
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 pair_at<__half>(const Pack<__half> &p, int i) { return __half22float2(((const __half2 *)&p)[i]); }
template <class T>
__device__ __forceinline__ void put_pair(Pack<T> &p, int i, float2 x) {
    p.v[2 * i] = narrowed<T>(x.x);
    p.v[2 * i + 1] = narrowed<T>(x.y);
}
template <>
__device__ __forceinline__ void put_pair<__nv_bfloat16>(Pack<__nv_bfloat16> &p, int i, float2 x) { ((__nv_bfloat162 *)&p)[i] = __float22bfloat162_rn(x); }
template <>
__device__ __forceinline__ void put_pair<__half>(Pack<__half> &p, int i, float2 x) { ((__half2 *)&p)[i] = __float22half2_rn(x); }

template <class T>
struct Eight {  // columns, as they are stored
    static constexpr int kPacks = 8 / Pack<T>::N;
    Pack<T> p[kPacks];
    // f32: 32 bytes at once, from a 32-byte boundary (two halves of a sector asked for one after the other cost twice the requests)
    __device__ __forceinline__ void load(const char *from) {
        if constexpr (sizeof(T) == 4) {
            float *f = (float *)p;
            asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
                         : "l"(from)
                         : "memory");
        } else {
            p[0] = *(const Pack<T> *)from;
        }
    }
    // ... what nothing reads again
    __device__ __forceinline__ void load_once(const char *from) {
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            uint4 u;
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(from + i * 16));
            *(uint4 *)&p[i] = u;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPacks; ++i) *(uint4 *)&p[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void store(char *to) const {
        if constexpr (sizeof(T) == 4) {
            const float *f = (const float *)p;
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]) : "memory");
        } else {
            *(Pack<T> *)to = p[0];
        }
    }
    __device__ __forceinline__ void open(float2 (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pair_at<T>(p[i / (4 / kPacks)], i % (4 / kPacks));
    }
    __device__ __forceinline__ void close(const float2 (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) put_pair<T>(p[i / (4 / kPacks)], i % (4 / kPacks), v[i]);
    }
};
}  // namespace k
}  // namespace sage
