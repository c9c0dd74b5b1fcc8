// AdamW over many tensors: one launch updates every tensor of the call, with first and second moments in 32 or in 8 bits.
//
// 8 bits: blocks of 256 elements of a tensor share a scale, and codes follow a square law, |m| = a code^2 with a = max |m| / 127^2 and
// sqrt(v) = b code^2 with b = max sqrt(v) / 255^2: a step of 1.6 % (0.8 %) at the block's largest and 16 129 (65 025) between the
// largest and the smallest, where even steps would lose all below a 127th.  The root of v is stored because it is what divides.
// Every operation on the moments is rounded by itself, so that codes do not depend on how a compiler contracts them.
#include <cuda_runtime.h>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

constexpr int kSlots = 400;  // 30 KB of kernel parameters
struct Batch {
    AdamWSlot slot[kSlots];
    unsigned first[kSlots + 1];  // prefix sums of the slots' blocks of 256 elements
    int count;
};

__device__ __forceinline__ float load_as_float(const void *p, int dtype, long long i) {
    if (dtype == SAGE_F16) return widen(((const __half *)p)[i]);
    if (dtype == SAGE_BF16) return widen(((const __nv_bfloat16 *)p)[i]);
    return ((const float *)p)[i];
}

// A value's moments after one more gradient; `root` is sqrt(v).
__device__ __forceinline__ void moments(const AdamWRule &k, float g, float *m, float *v, float *root) {
    g = __fmul_rn(g, k.grad_scale);
    *m = __fadd_rn(__fmul_rn(*m, k.beta1), __fmul_rn(g, k.one_minus_beta1));
    *v = __fadd_rn(__fmul_rn(*v, k.beta2), __fmul_rn(__fmul_rn(g, g), k.one_minus_beta2));
    *root = __fsqrt_rn(*v);
}
__device__ __forceinline__ float updated(const AdamWRule &k, float p, float m, float root) {
    return p * k.keep - m * k.step_size / (root * k.root_factor + k.eps);
}

// Largest of non-negative values by their bits: NaN is above infinity, and both above every number.
__device__ __forceinline__ unsigned warp_largest(unsigned v) {
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// The factor of a block's codes and its stored scale, from the block's largest.  Below 2^-100 a block is zero.
template <int TOP>
__device__ __forceinline__ float block_scale(unsigned largest, float *factor) {
    const float x = __uint_as_float(largest);
    *factor = 0.f;
    if (largest >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
    if (x < 7.888609052210118e-31f) return 0.f;
    *factor = __fmul_rn(__frcp_rn(x), (float)(TOP * TOP));
    return __fmul_rn(x, 1.f / (TOP * TOP));
}

template <bool STATES8>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ Batch b, const AdamWRule k) {
    grid_dependency_sync();
    const unsigned total = b.first[b.count], lane = threadIdx.x % 32;
    for (unsigned block = blockIdx.x * 8 + threadIdx.x / 32; block < total; block += gridDim.x * 8) {
        int lo = 0, hi = b.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (b.first[mid] <= block) lo = mid;
            else hi = mid - 1;
        }
        const AdamWSlot &s = b.slot[lo];
        const long long at = (long long)(block - b.first[lo]) * kAdamWBlock;
        float m[8], v[8], root[8], g[8];
        unsigned m_top = 0, v_top = 0;
        const float ms = STATES8 ? s.m_scale[at / kAdamWBlock] : 0.f, vs = STATES8 ? s.v_scale[at / kAdamWBlock] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long j = at + i * 32 + lane;
            m[i] = v[i] = root[i] = g[i] = 0.f;
            if (j >= s.n) continue;
            if (STATES8) {
                const int c = ((const signed char *)s.m)[j], d = ((const unsigned char *)s.v)[j];
                m[i] = __fmul_rn(ms, (float)(c * abs(c)));
                const float q = __fmul_rn(vs, (float)(d * d));
                v[i] = __fmul_rn(q, q);
            } else {
                m[i] = ((const float *)s.m)[j];
                v[i] = ((const float *)s.v)[j];
            }
            moments(k, load_as_float(s.g, s.g_dtype, j), &m[i], &v[i], &root[i]);
            const float p = updated(k, s.p[j], m[i], root[i]);
            s.p[j] = p;
            if (s.copy) {
                if (s.copy_dtype == SAGE_F16) ((__half *)s.copy)[j] = narrowed<__half>(p);
                else ((__nv_bfloat16 *)s.copy)[j] = narrowed<__nv_bfloat16>(p);
            }
            if (!STATES8) {
                ((float *)s.m)[j] = m[i];
                ((float *)s.v)[j] = v[i];
            }
            m_top = max(m_top, __float_as_uint(fabsf(m[i])));
            v_top = max(v_top, __float_as_uint(fabsf(root[i])));
        }
        if (!STATES8) continue;
        float mf, vf;
        const float new_ms = block_scale<127>(warp_largest(m_top), &mf), new_vs = block_scale<255>(warp_largest(v_top), &vf);
        if (lane == 0) {
            s.m_scale[at / kAdamWBlock] = new_ms;
            s.v_scale[at / kAdamWBlock] = new_vs;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long j = at + i * 32 + lane;
            if (j >= s.n) continue;
            int c = mf > 0.f ? min(127, __float2int_rn(__fsqrt_rn(__fmul_rn(fabsf(m[i]), mf)))) : 0;
            int d = vf > 0.f ? min(255, __float2int_rn(__fsqrt_rn(__fmul_rn(root[i], vf)))) : 0;
            if (vf > 0.f && root[i] > 0.f) d = max(d, 1);
            ((signed char *)s.m)[j] = (signed char)(m[i] < 0.f ? -c : c);
            ((unsigned char *)s.v)[j] = (unsigned char)d;
        }
    }
}

__global__ void __launch_bounds__(256) adamw_states_kernel(const signed char *m, const float *m_scale, const unsigned char *v, const float *v_scale, long long n, float *m_out, float *v_out) {
    grid_dependency_sync();
    for (long long j = (long long)blockIdx.x * 256 + threadIdx.x; j < n; j += (long long)gridDim.x * 256) {
        const int c = m[j], d = v[j];
        m_out[j] = __fmul_rn(m_scale[j / kAdamWBlock], (float)(c * abs(c)));
        const float q = __fmul_rn(v_scale[j / kAdamWBlock], (float)(d * d));
        v_out[j] = __fmul_rn(q, q);
    }
}

}  // namespace

sage_status adamw_step(Context &ctx, const AdamWSlot *slots, int count, bool states8, const AdamWRule &rule) {
    for (int at = 0; at < count; at += kSlots) {
        static thread_local Batch b;
        b.count = count - at < kSlots ? count - at : kSlots;
        unsigned blocks = 0;
        for (int i = 0; i < b.count; ++i) {
            b.slot[i] = slots[at + i];
            b.first[i] = blocks;
            const long long c = (b.slot[i].n + kAdamWBlock - 1) / kAdamWBlock;
            if (c + blocks > 0x7fffffffll) return ctx.fail(SAGE_ERR_INVALID, "adamw_step: too many elements in one call");
            blocks += (unsigned)c;
        }
        b.first[b.count] = blocks;
        if (!blocks) continue;
        ctx.note_launch("adamw_step");
        if (ctx.dry()) continue;
        const unsigned most = (unsigned)ctx.sm_count * 8, grid = (blocks + 7) / 8 < most ? (blocks + 7) / 8 : most;
        sage_status st = ctx.check_cuda(states8 ? launch_dependent(ctx.pdl, ctx.stream(), adamw_kernel<true>, dim3(grid), dim3(256), 0, b, rule)
                                                : launch_dependent(ctx.pdl, ctx.stream(), adamw_kernel<false>, dim3(grid), dim3(256), 0, b, rule),
                                        "adamw_step");
        if (st) return st;
    }
    return SAGE_OK;
}

sage_status adamw_states(Context &ctx, const void *m, const float *m_scale, const void *v, const float *v_scale, long long n, float *m_out, float *v_out) {
    if (!n) return SAGE_OK;
    ctx.note_launch("adamw_states");
    if (ctx.dry()) return SAGE_OK;
    const long long blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < ctx.sm_count * 32ll ? blocks : ctx.sm_count * 32ll));
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), adamw_states_kernel, grid, dim3(256), 0, (const signed char *)m, m_scale, (const unsigned char *)v, v_scale, n, m_out, v_out), "adamw_states");
}

}  // namespace k
}  // namespace sage
