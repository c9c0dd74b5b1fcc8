// Random bits by position: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), keyed by
// two words of device memory, so that what a captured graph draws follows what the program wrote there before the replay.
#pragma once
#include <cuda_runtime.h>

namespace sage {
namespace k {

// Which elements dropout keeps, and the factor on them.  `bar` of 65536 are dropped.
struct Dropout {
    const unsigned *seed = nullptr;  // two words, `seed_stride` apart
    long long seed_stride = 1;
    unsigned long long site = 0;
    unsigned bar = 0;
    float factor = 1.f;
};

struct Key {
    unsigned a, b;
};
// (the shuffle tells the compiler that a warp has one key, whose sums with the rounds' constants it then keeps once for all lanes)
__device__ __forceinline__ Key key_of(const Dropout &d) {
    if (!d.bar) return Key{0u, 0u};
    return Key{__shfl_sync(0xffffffffu, __ldg(d.seed), 0), __shfl_sync(0xffffffffu, __ldg(d.seed + d.seed_stride), 0)};
}

__device__ __forceinline__ uint4 philox(Key k, unsigned long long count, unsigned long long site) {
    uint4 x = make_uint4((unsigned)count, (unsigned)(count >> 32), (unsigned)site, (unsigned)(site >> 32));
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long p = (unsigned long long)x.x * 0xD2511F53u, q = (unsigned long long)x.z * 0xCD9E8D57u;
        x = make_uint4((unsigned)(q >> 32) ^ x.y ^ k.a, (unsigned)q, (unsigned)(p >> 32) ^ x.w ^ k.b, (unsigned)p);
        k.a += 0x9E3779B9u;
        k.b += 0xBB67AE85u;
    }
    return x;
}

// ... with the rounds' keys made once (a block of threads keeps them in shared memory: five loads instead of twenty additions).
struct alignas(16) RoundKeys {  // (two rounds' are read at a time)
    uint2 k[10];
};
__device__ __forceinline__ void round_keys(RoundKeys *to, Key k, int thread) {
    if (thread < 10) to->k[thread] = make_uint2(k.a + (unsigned)thread * 0x9E3779B9u, k.b + (unsigned)thread * 0xBB67AE85u);
}
__device__ __forceinline__ uint4 philox(const RoundKeys &keys, unsigned long long count, unsigned long long site) {
    uint4 x = make_uint4((unsigned)count, (unsigned)(count >> 32), (unsigned)site, (unsigned)(site >> 32));
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const uint4 two = ((const uint4 *)keys.k)[i];
        unsigned long long p = (unsigned long long)x.x * 0xD2511F53u, q = (unsigned long long)x.z * 0xCD9E8D57u;
        x = make_uint4((unsigned)(q >> 32) ^ x.y ^ two.x, (unsigned)q, (unsigned)(p >> 32) ^ x.w ^ two.y, (unsigned)p);
        p = (unsigned long long)x.x * 0xD2511F53u, q = (unsigned long long)x.z * 0xCD9E8D57u;
        x = make_uint4((unsigned)(q >> 32) ^ x.y ^ two.z, (unsigned)q, (unsigned)(p >> 32) ^ x.w ^ two.w, (unsigned)p);
    }
    return x;
}

// Bit e: element 8 * block + e stays.  Sixteen bits an element, four words a block: a draw of ten rounds serves eight elements (one draw for
// four, with 32 bits each, is more arithmetic than the memory leaves time for), and shares are multiples of 2^-16.
__device__ __forceinline__ unsigned keep8(const Dropout &d, Key k, unsigned long long block) {
    const uint4 w = philox(k, block, d.site);
    const unsigned words[4] = {w.x, w.y, w.z, w.w};
    unsigned keep = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        keep |= ((words[i] & 0xffffu) >= d.bar ? 1u : 0u) << (2 * i);
        keep |= ((words[i] >> 16) >= d.bar ? 1u : 0u) << (2 * i + 1);
    }
    return keep;
}
// Eight elements, those that are dropped zero: of a word's halves the upper one is compared in place, the lower one shifted there.
__device__ __forceinline__ void drop8(float2 (&v)[4], const uint4 &w, unsigned bar, float zero = 0.f) {
    const unsigned words[4] = {w.x, w.y, w.z, w.w}, high = bar << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2((words[i] << 16) >= high ? v[i].x : zero, words[i] >= high ? v[i].y : zero);
}
// ... of eight elements from `first` on, wherever that lies in a block.
__device__ __forceinline__ unsigned keep_from(const Dropout &d, Key k, unsigned long long first) {
    if (!d.bar) return 0xffu;
    const unsigned at = (unsigned)first & 7u;
    const unsigned low = keep8(d, k, first >> 3);
    return at ? (low >> at | keep8(d, k, (first >> 3) + 1) << (8 - at)) & 0xffu : low;
}

}  // namespace k
}  // namespace sage
