// AdamW over many tensors: one launch updates every tensor of the call, with first and second moments in 32 or in 8 bits.
//
// 8 bits: blocks of 256 elements of a tensor share a scale, and codes follow a square law, |m| = a code^2 with a = max |m| / 127^2 and
// sqrt(v) = b code^2 with b = max sqrt(v) / 255^2: a step of 1.6 % (0.8 %) at the block's largest and 16 129 (65 025) between the
// largest and the smallest, where even steps would lose all below a 127th.  The root of v is stored because it is what divides.
// Codes and scales are those of the moments as f32 rounds them operation by operation, whatever shortcuts find them: the fast square
// root decides a code unless its result lies so near the middle of two codes that it could err, where the exact one does.
//
// A warp takes a block of 256 elements at a time, eight to a lane.  Bound by memory: 28 bytes an element with f32 states and gradients (109 M:
// 483 us, 6.3 TB/s), 16 with 8-bit states, bf16 gradients and a copy (334 M: 957 us, 5.6 TB/s, the instructions that find the codes at 64 %
// of their slots beside it).
#include <cuda_runtime.h>

#include <cmath>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

template <int SLOTS>
struct Batch {
    AdamWSlot slot[SLOTS];
    unsigned first[SLOTS + 1];  // prefix sums of the slots' blocks of 256 elements
    int count;
};
// 32 KB of kernel parameters, or 3 KB for short lists: a launch's parameters are copied with it (4, 20 and 38 tensors of 4000 elements: 3.9, 4.1 and 4.5 us
// a step with the short list, 5.3, 5.7 and 6.2 with the long one; 54 tensors 6.5, 300 13).
constexpr int kSlots = 400, kFewSlots = 40;

__device__ __forceinline__ float fast_root(float x) {  // 2^-23 off at most, of subnormal numbers 0
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float largest(float a, float b, float c) {  // NaN wins
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float one_if_positive(float x) {
    float y;
    asm("set.gt.f32.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_largest(float x) {
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// The factor of a block's codes and its stored scale, from the block's largest (not negative).  Below 2^-100 a block is zero.
template <int TOP>
__device__ __forceinline__ float block_scale(float x, float *factor) {
    *factor = 0.f;
    if (!(x < INFINITY)) return __uint_as_float(0x7fffffffu);
    if (x < 7.888609052210118e-31f) return 0.f;
    *factor = __fmul_rn(__frcp_rn(x), (float)(TOP * TOP));
    return __fmul_rn(x, 1.f / (TOP * TOP));
}
// Codes of eight elements: the nearest whole numbers to the roots of t (with `sign`'s sign), from approximate roots.  1.5 2^23 added leaves the
// whole number in the low bits.  `off` is the furthest that a root lies from its code: where that is within the approximation's error of
// one half, another code might be nearer, and the caller takes the exact root.
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ void rounded(float2 root, float *off, unsigned *n) {
    const float2 m = add2(root, both(kMagic)), d = add2(root, add2(both(kMagic), make_float2(-m.x, -m.y)));
    *off = fmaxf(*off, fmaxf(fabsf(d.x), fabsf(d.y)));
    n[0] = __float_as_uint(m.x);
    n[1] = __float_as_uint(m.y);
}
__device__ __forceinline__ unsigned low_bytes(const unsigned *n) { return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410); }

// The moments of eight elements after one more gradient, rounded operation by operation; the parameters, with approximate roots and
// quotients (2^-21).
struct Elements {
    float2 p[4], g[4], m[4], v[4], root[4];
};
__device__ __forceinline__ void update(const AdamWRule &k, Elements &e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 g = mul2(e.g[i], both(k.grad_scale));
        const float2 zero = both(k.minus_zero);  // products rounded before they are added
        e.m[i] = add2(fma2(e.m[i], both(k.beta1), zero), fma2(g, both(k.one_minus_beta1), zero));
        e.v[i] = add2(fma2(e.v[i], both(k.beta2), zero), fma2(mul2(g, g), both(k.one_minus_beta2), zero));
        e.root[i] = make_float2(fast_root(e.v[i].x), fast_root(e.v[i].y));
        const float2 below = fma2(e.root[i], both(k.root_factor), both(k.eps)), step = mul2(e.m[i], both(-k.step_size));
        e.p[i] = fma2(e.p[i], both(k.keep), mul2(step, make_float2(fast_reciprocal(below.x), fast_reciprocal(below.y))));
    }
}
__device__ __forceinline__ float &at(float2 *x, int i) { return i % 2 ? x[i / 2].y : x[i / 2].x; }

// Where the eight elements of a lane lie in the block: two times four in a row, or (blocks that end early, tensors off 16-byte
// boundaries) 32 apart.
template <bool WIDE>
__device__ __forceinline__ int place(int i) {
    const int lane = threadIdx.x % 32;
    return WIDE ? i / 4 * 128 + lane * 4 + i % 4 : i * 32 + lane;
}
// Elements of type T at `p`, the start of the block; those of [0, n) where not WIDE.
template <bool WIDE, class T, class F>
__device__ __forceinline__ void load8(const T *p, int n, F put) {
    if (WIDE) {
        struct alignas(4 * sizeof(T)) Four {
            T v[4];
        };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const Four q = *reinterpret_cast<const Four *>(p + place<true>(4 * h));
#pragma unroll
            for (int j = 0; j < 4; ++j) put(4 * h + j, q.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) put(i, place<false>(i) < n ? p[place<false>(i)] : T(0.f));
    }
}
template <bool WIDE, class T, class F>
__device__ __forceinline__ void store8(T *p, int n, F get) {
    if (WIDE) {
        struct alignas(4 * sizeof(T)) Four {
            T v[4];
        };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Four q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q.v[j] = get(4 * h + j);
            *reinterpret_cast<Four *>(p + place<true>(4 * h)) = q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (place<false>(i) < n) p[place<false>(i)] = get(i);
    }
}

// What a lane reads of a whole block, as it lies in memory: asked for a block ahead where states have 8 bits, whose arithmetic would
// otherwise wait for memory and memory for it.
struct Raw {
    uint4 p[2], g[2];
    unsigned m[2], v[2];
    float ms, vs;
};
__device__ __forceinline__ void load_raw(const AdamWSlot &s, long long block, Raw &r) {
    const long long from = block * kAdamWBlock;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long j = from + place<true>(4 * h);
        r.p[h] = *reinterpret_cast<const uint4 *>(s.p + j);
        r.m[h] = *reinterpret_cast<const unsigned *>((const char *)s.m + j);
        r.v[h] = *reinterpret_cast<const unsigned *>((const char *)s.v + j);
        if (s.g_dtype == SAGE_F32) r.g[h] = *reinterpret_cast<const uint4 *>((const float *)s.g + j);
        else *reinterpret_cast<uint2 *>(&r.g[h]) = *reinterpret_cast<const uint2 *>((const char *)s.g + 2 * j);
    }
    r.ms = s.m_scale[block];
    r.vs = s.v_scale[block];
}
__device__ __forceinline__ float2 two(unsigned a, unsigned b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
// Bytes 2 j and 2 j + 1 of a word: behind the exponent of 2^23 they count from there.
__device__ __forceinline__ float2 codes_of(unsigned word, int j, float zero) {
    return add2(two(__byte_perm(word, 0x4b000000u, 0x7440 + 2 * j), __byte_perm(word, 0x4b000000u, 0x7441 + 2 * j)), both(-zero));
}
__device__ __forceinline__ void elements_of(const Raw &r, int g_dtype, Elements &e) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        e.p[2 * h] = two(r.p[h].x, r.p[h].y);
        e.p[2 * h + 1] = two(r.p[h].z, r.p[h].w);
        e.g[2 * h] = two(r.g[h].x, r.g[h].y);
        e.g[2 * h + 1] = two(r.g[h].z, r.g[h].w);
        if (g_dtype == SAGE_BF16) {
            e.g[2 * h] = two(r.g[h].x << 16, r.g[h].x & 0xffff0000u);
            e.g[2 * h + 1] = two(r.g[h].y << 16, r.g[h].y & 0xffff0000u);
        } else if (g_dtype == SAGE_F16) {
            e.g[2 * h] = __half22float2(*reinterpret_cast<const __half2 *>(&r.g[h].x));
            e.g[2 * h + 1] = __half22float2(*reinterpret_cast<const __half2 *>(&r.g[h].y));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 c = codes_of(r.m[h] ^ 0x80808080u, j, 8388608.f + 128.f);
            e.m[2 * h + j] = mul2(make_float2(c.x * fabsf(c.x), c.y * fabsf(c.y)), both(r.ms));
            e.v[2 * h + j] = codes_of(r.v[h], j, 8388608.f);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 q = mul2(mul2(e.v[i], e.v[i]), both(r.vs));
        e.v[i] = mul2(q, q);
    }
}

template <bool STATES8, bool WIDE>
__device__ __forceinline__ void load_elements(const AdamWSlot &s, long long block, int n, Elements &e) {
    const long long from = block * kAdamWBlock;
    if (s.g_dtype == SAGE_F32) load8<WIDE>((const float *)s.g + from, n, [&](int i, float x) { at(e.g, i) = x; });
    else if (s.g_dtype == SAGE_BF16) load8<WIDE>((const __nv_bfloat16 *)s.g + from, n, [&](int i, __nv_bfloat16 x) { at(e.g, i) = widen(x); });
    else load8<WIDE>((const __half *)s.g + from, n, [&](int i, __half x) { at(e.g, i) = widen(x); });
    load8<WIDE>(s.p + from, n, [&](int i, float x) { at(e.p, i) = x; });
    if (STATES8) {
        const float ms = s.m_scale[block], vs = s.v_scale[block];
        load8<WIDE>((const signed char *)s.m + from, n, [&](int i, signed char c) {
            const float f = (float)c;
            at(e.m, i) = __fmul_rn(ms, f * fabsf(f));
        });
        load8<WIDE>((const unsigned char *)s.v + from, n, [&](int i, unsigned char c) { at(e.v, i) = (float)c; });
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 q = mul2(mul2(e.v[i], e.v[i]), both(vs));
            e.v[i] = mul2(q, q);
        }
        if (!WIDE) {  // a scale that is NaN makes zeros behind the end NaN too
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (place<false>(i) >= n) at(e.m, i) = at(e.v, i) = 0.f;
        }
    } else {
        load8<WIDE>((const float *)s.m + from, n, [&](int i, float x) { at(e.m, i) = x; });
        load8<WIDE>((const float *)s.v + from, n, [&](int i, float x) { at(e.v, i) = x; });
    }
}

template <bool STATES8, bool WIDE>
__device__ __forceinline__ void block_update(const AdamWSlot &s, const AdamWRule &k, long long block, int n, Elements &e) {
    const long long from = block * kAdamWBlock;
    update(k, e);
    store8<WIDE>(s.p + from, n, [&](int i) { return at(e.p, i); });
    if (s.copy) {
        if (s.copy_dtype == SAGE_BF16) store8<WIDE>((__nv_bfloat16 *)s.copy + from, n, [&](int i) { return narrowed<__nv_bfloat16>(at(e.p, i)); });
        else store8<WIDE>((__half *)s.copy + from, n, [&](int i) { return narrowed<__half>(at(e.p, i)); });
    }
    if (!STATES8) {
        store8<WIDE>((float *)s.m + from, n, [&](int i) { return at(e.m, i); });
        store8<WIDE>((float *)s.v + from, n, [&](int i) { return at(e.v, i); });
        return;
    }
    float m_top = 0.f, v_top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m_top = largest(m_top, fabsf(e.m[i].x), fabsf(e.m[i].y));
        v_top = largest(v_top, e.v[i].x, e.v[i].y);
    }
    m_top = warp_largest(m_top);
    v_top = __fsqrt_rn(warp_largest(v_top));
    float mf, vf;
    const float ms = block_scale<127>(m_top, &mf), vs = block_scale<255>(v_top, &vf);
    if (threadIdx.x % 32 == 0) {
        s.m_scale[block] = ms;
        s.v_scale[block] = vs;
    }
    unsigned m[8], v[8];
    float m_off = 0.f, v_off = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = mul2(make_float2(fabsf(e.m[i].x), fabsf(e.m[i].y)), both(mf)), u = mul2(e.root[i], both(vf));
        rounded(make_float2(copysignf(fast_root(t.x), e.m[i].x), copysignf(fast_root(t.y), e.m[i].y)), &m_off, m + 2 * i);
        // one at least for what is not zero
        rounded(make_float2(fmaxf(fast_root(u.x), one_if_positive(e.v[i].x)), fmaxf(fast_root(u.y), one_if_positive(e.v[i].y))), &v_off, v + 2 * i);
    }
    // How far a fast root can lie from the exact one's rounded result.  u = 2^-24 is one rounding, a fast root is 2 u off at most, and errors in
    // front of a root halve.  Of m: 2 u of up to 127, and half an f32 step there, 1.9e-5.  Of v: the fast way has 2 u (outer root), u / 2 (product)
    // and u (inner root), the exact way u, u / 2 and u / 2, in all 5.5 u of up to 255, 8.4e-5.  Where all of a block's v lie below 2^-80,
    // subnormal ones count, which the fast root takes for zero.
    constexpr float kMOff = 2.2e-5f, kVOff = 0x1.8p-14f;
    if (m_off > 0.5f - kMOff || v_off > 0.5f - kVOff || v_top < 0x1p-40f) {
        float none = 0.f;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            float2 x = e.m[0], y = e.v[0];
#pragma unroll
            for (int j = 1; j < 4; ++j)
                if (j == i) {
                    x = e.m[j];
                    y = e.v[j];
                }
            unsigned c[2], d[2];
            rounded(make_float2(copysignf(__fsqrt_rn(__fmul_rn(fabsf(x.x), mf)), x.x), copysignf(__fsqrt_rn(__fmul_rn(fabsf(x.y), mf)), x.y)), &none, c);
            rounded(make_float2(fmaxf(__fsqrt_rn(__fmul_rn(__fsqrt_rn(y.x), vf)), one_if_positive(y.x)), fmaxf(__fsqrt_rn(__fmul_rn(__fsqrt_rn(y.y), vf)), one_if_positive(y.y))), &none, d);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j == i) {
                    m[2 * j] = c[0];
                    m[2 * j + 1] = c[1];
                    v[2 * j] = d[0];
                    v[2 * j + 1] = d[1];
                }
        }
    }
    unsigned mw[2], vw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // no codes in blocks that are zero or not finite
        mw[h] = mf > 0.f ? low_bytes(m + 4 * h) : 0;
        vw[h] = vf > 0.f ? low_bytes(v + 4 * h) : 0;
    }
    if (WIDE) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<unsigned *>((unsigned char *)s.m + from + place<true>(4 * h)) = mw[h];
            *reinterpret_cast<unsigned *>((unsigned char *)s.v + from + place<true>(4 * h)) = vw[h];
        }
    } else {
        store8<false>((unsigned char *)s.m + from, n, [&](int i) { return (unsigned char)(mw[i / 4] >> (8 * (i % 4))); });
        store8<false>((unsigned char *)s.v + from, n, [&](int i) { return (unsigned char)(vw[i / 4] >> (8 * (i % 4))); });
    }
}

// The slots' blocks in the order that a warp takes them.
template <int SLOTS>
struct Walk {
    const Batch<SLOTS> &b;
    unsigned block;
    int slot = 0;
    __device__ __forceinline__ bool valid() const { return block < b.first[b.count]; }
    __device__ __forceinline__ void find() {  // from the last slot on
        if (!valid() || b.first[slot + 1] > block) return;
        int lo = slot + 1, hi = b.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (b.first[mid] <= block) lo = mid;
            else hi = mid - 1;
        }
        slot = lo;
    }
    __device__ __forceinline__ void next() {
        block += gridDim.x * 8;
        find();
    }
    __device__ __forceinline__ long long mine() const { return block - b.first[slot]; }
    __device__ __forceinline__ bool whole() const { return b.slot[slot].wide && (mine() + 1) * kAdamWBlock <= b.slot[slot].n; }
};

template <bool STATES8, int SLOTS>
__global__ void __launch_bounds__(256, STATES8 ? 3 : 4) adamw_kernel(const __grid_constant__ Batch<SLOTS> b, const AdamWRule k) {
    grid_dependency_sync();
    Walk<SLOTS> at{b, blockIdx.x * 8 + threadIdx.x / 32};
    at.find();
    if constexpr (STATES8) {
        Raw raw;
        if (at.valid() && at.whole()) load_raw(b.slot[at.slot], at.mine(), raw);
        while (at.valid()) {
            const AdamWSlot &s = b.slot[at.slot];
            const long long mine = at.mine();
            Elements e;
            if (at.whole()) {
                elements_of(raw, s.g_dtype, e);
                at.next();
                if (at.valid() && at.whole()) load_raw(b.slot[at.slot], at.mine(), raw);
                block_update<STATES8, true>(s, k, mine, kAdamWBlock, e);
            } else {
                const int n = (int)min(s.n - mine * kAdamWBlock, (long long)kAdamWBlock);
                at.next();
                if (at.valid() && at.whole()) load_raw(b.slot[at.slot], at.mine(), raw);
                load_elements<STATES8, false>(s, mine, n, e);
                block_update<STATES8, false>(s, k, mine, n, e);
            }
        }
    } else {
        for (; at.valid(); at.next()) {
            const AdamWSlot &s = b.slot[at.slot];
            Elements e;
            if (at.whole()) {
                load_elements<STATES8, true>(s, at.mine(), kAdamWBlock, e);
                block_update<STATES8, true>(s, k, at.mine(), kAdamWBlock, e);
            } else {
                const int n = (int)min(s.n - at.mine() * kAdamWBlock, (long long)kAdamWBlock);
                load_elements<STATES8, false>(s, at.mine(), n, e);
                block_update<STATES8, false>(s, k, at.mine(), n, e);
            }
        }
    }
}

// Values of codes: four to a thread where `wide`, else one.  Bound by memory: 2 bytes read, 8 written (334 M: 580 us, 5.8 TB/s).
template <bool WIDE>
__global__ void __launch_bounds__(256) adamw_states_kernel(const signed char *m, const float *m_scale, const unsigned char *v, const float *v_scale, long long n, float *m_out, float *v_out) {
    grid_dependency_sync();
    constexpr int N = WIDE ? 4 : 1;
    struct alignas(N) Codes {
        signed char c[N];
    };
    struct alignas(4 * N) Values {
        float x[N];
    };
    const long long step = (long long)gridDim.x * 256 * N;
    for (long long j = ((long long)blockIdx.x * 256 + threadIdx.x) * N; j + N <= n; j += step) {
        const Codes c = *reinterpret_cast<const Codes *>(m + j), d = *reinterpret_cast<const Codes *>(v + j);
        const float ms = m_scale[j / kAdamWBlock], vs = v_scale[j / kAdamWBlock];
        Values a, b;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = (float)c.c[i], h = (float)(unsigned char)d.c[i], q = __fmul_rn(vs, h * h);
            a.x[i] = __fmul_rn(ms, f * fabsf(f));
            b.x[i] = __fmul_rn(q, q);
        }
        *reinterpret_cast<Values *>(m_out + j) = a;
        *reinterpret_cast<Values *>(v_out + j) = b;
    }
}

}  // namespace

// The constants of a step, from 64 bits.
AdamWRule adamw_rule(double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale, long long step) {
    AdamWRule r;
    r.beta1 = (float)beta1;
    r.one_minus_beta1 = (float)(1.0 - beta1);
    r.beta2 = (float)beta2;
    r.one_minus_beta2 = (float)(1.0 - beta2);
    r.keep = (float)(1.0 - lr * weight_decay);
    r.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    r.root_factor = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    r.eps = (float)eps;
    r.grad_scale = (float)grad_scale;
    return r;
}

template <int SLOTS>
static sage_status step_batches(Context &ctx, const AdamWSlot *slots, int count, bool states8, const AdamWRule &rule) {
    for (int at = 0; at < count; at += SLOTS) {
        static thread_local Batch<SLOTS> b;
        b.count = count - at < SLOTS ? count - at : SLOTS;
        unsigned blocks = 0;
        for (int i = 0; i < b.count; ++i) {
            AdamWSlot &s = b.slot[i] = slots[at + i];
            const auto on = [](const void *p, size_t boundary) { return reinterpret_cast<uintptr_t>(p) % boundary == 0; };
            s.wide = on(s.p, 16) && on(s.g, s.g_dtype == SAGE_F32 ? 16 : 8) && on(s.m, states8 ? 4 : 16) && on(s.v, states8 ? 4 : 16) && on(s.copy, 8);
            b.first[i] = blocks;
            const long long c = (s.n + kAdamWBlock - 1) / kAdamWBlock;
            if (c + blocks > 0x7fff0000ll) return ctx.fail(SAGE_ERR_INVALID, "adamw_step: too many elements in one call");
            blocks += (unsigned)c;
        }
        b.first[b.count] = blocks;
        if (!blocks) continue;
        ctx.note_launch("adamw_step");
        if (ctx.dry()) continue;
        // As many blocks as are resident with a block of elements asked for ahead (334 M parameters: 985 us, with 4 and 8 an SM 1195 and 1049); else
        // twice as many, which evens the ends out (109 M in 32 bits: 488 us, with 4 an SM 500).
        const unsigned most = (unsigned)ctx.sm_count * (states8 ? 3 : 8), grid = (blocks + 7) / 8 < most ? (blocks + 7) / 8 : most;
        sage_status st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), states8 ? adamw_kernel<true, SLOTS> : adamw_kernel<false, SLOTS>, dim3(grid), dim3(256), 0, b, rule), "adamw_step");
        if (st) return st;
    }
    return SAGE_OK;
}

sage_status adamw_step(Context &ctx, const AdamWSlot *slots, int count, bool states8, const AdamWRule &rule) {
    return count <= kFewSlots ? step_batches<kFewSlots>(ctx, slots, count, states8, rule) : step_batches<kSlots>(ctx, slots, count, states8, rule);
}

sage_status adamw_states(Context &ctx, const void *m, const float *m_scale, const void *v, const float *v_scale, long long n, float *m_out, float *v_out) {
    if (!n) return SAGE_OK;
    const uintptr_t codes = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v), values = reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out);
    const bool wide = n % 4 == 0 && codes % 4 == 0 && values % 16 == 0;
    ctx.note_launch("adamw_states");
    if (ctx.dry()) return SAGE_OK;
    const long long each = wide ? 1024 : 256, blocks = (n + each - 1) / each, most = ctx.sm_count * 32ll;
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? adamw_states_kernel<true> : adamw_states_kernel<false>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0,
                                           (const signed char *)m, m_scale, (const unsigned char *)v, v_scale, n, m_out, v_out),
                          "adamw_states");
}

}  // namespace k
}  // namespace sage
