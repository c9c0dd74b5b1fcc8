// Log probabilities of given tokens, with entropy, alternatives and gradient.
//
// With x the row's logits, c the scale, m = max x, S = sum exp(c (x - m)):
//   log p_j = c (x_j - m) - ln S,   H = ln S - sum c (x_j - m) exp(c (x_j - m)) / S.
#include <cuda_runtime.h>

#include <cfloat>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

constexpr int kThreads = 256;

// Larger for larger logits and, among equals, for lower tokens; no two tokens of a row have the same.  NaN counts as -inf.
__device__ __forceinline__ unsigned long long rank_key(float x, unsigned token) {
    x = x != x ? -INFINITY : x + 0.f;  // -0 and 0 are equal
    const unsigned b = __float_as_uint(x);
    return (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - token);
}
__device__ __forceinline__ float rank_logit(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

template <class V, class F>
__device__ V block_combine(V v, F f, V *shared) {
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
    __syncthreads();
    v = shared[0];
    for (int i = 1; i < kThreads / 32; ++i) v = f(v, shared[i]);
    __syncthreads();
    return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(const LogProbs a) {
    grid_dependency_sync();
    __shared__ float fs[kThreads / 32];
    __shared__ unsigned long long ks[kThreads / 32];
    const long long r = blockIdx.x, vocab = a.logits.cols;
    const T *x = (const T *)a.logits.ptr + r * a.logits.pitch;
    float m = -INFINITY;
    for (long long j = threadIdx.x; j < vocab; j += kThreads) m = fmaxf(m, widen(x[j]));
    m = block_combine(m, [](float p, float q) { return fmaxf(p, q); }, fs);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, sd = 0.f;
    for (long long j = threadIdx.x; j < vocab; j += kThreads) {
        const float d = (widen(x[j]) - base) * a.scale, e = expf(d);
        s += e;
        sd += e * fmaxf(d, -FLT_MAX);
    }
    s = block_combine(s, [](float p, float q) { return p + q; }, fs);
    sd = block_combine(sd, [](float p, float q) { return p + q; }, fs);
    const bool none = s == 0.f;
    const float ln_s = logf(s);
    if (threadIdx.x == 0) {
        const int id = ((const int *)a.ids.ptr)[r * a.ids.stride];
        float lp = 0.f;
        if (id >= 0 && id < vocab) lp = none ? -INFINITY : (widen(x[id]) - base) * a.scale - ln_s;
        ((float *)a.log_probs.ptr)[r * a.log_probs.stride] = lp;
        if (a.entropy.ptr) ((float *)a.entropy.ptr)[r * a.entropy.stride] = none ? 0.f : ln_s - sd / s;
        if (a.stats.ptr) {
            ((float *)a.stats.ptr)[r * a.stats.pitch] = m;
            ((float *)a.stats.ptr)[r * a.stats.pitch + 1] = s;
        }
    }
    unsigned long long below = ~0ull;
    for (int i = 0; i < a.top; ++i) {
        unsigned long long best = 0;
        for (long long j = threadIdx.x; j < vocab; j += kThreads) {
            const unsigned long long key = rank_key(widen(x[j]), (unsigned)j);
            if (key < below && key > best) best = key;
        }
        below = block_combine(best, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; }, ks);
        if (threadIdx.x == 0) {
            ((int *)a.top_ids.ptr)[r * a.top_ids.pitch + i] = (int)(0xffffffffu - (unsigned)below);
            ((float *)a.top_log_probs.ptr)[r * a.top_log_probs.pitch + i] = none ? -INFINITY : (rank_logit(below) - base) * a.scale - ln_s;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) log_probs_grad_kernel(const LogProbsGrad a) {
    grid_dependency_sync();
    const long long r = blockIdx.x, vocab = a.logits.cols;
    const T *x = (const T *)a.logits.ptr + r * a.logits.pitch;
    T *dx = (T *)a.dlogits.ptr + r * a.dlogits.pitch;
    const float m = ((const float *)a.stats.ptr)[r * a.stats.pitch], s = ((const float *)a.stats.ptr)[r * a.stats.pitch + 1];
    const int id = ((const int *)a.ids.ptr)[r * a.ids.stride];
    const float gl = a.g_log_probs.ptr && id >= 0 && id < vocab ? ((const float *)a.g_log_probs.ptr)[r * a.g_log_probs.stride] : 0.f;
    const float ge = a.g_entropy.ptr ? ((const float *)a.g_entropy.ptr)[r * a.g_entropy.stride] : 0.f;
    const float h = a.g_entropy.ptr ? ((const float *)a.entropy.ptr)[r * a.entropy.stride] : 0.f;
    const float ln_s = logf(s);
    for (long long j = threadIdx.x; j < vocab; j += kThreads) {
        float v = 0.f;
        if (s != 0.f) {
            const float d = (widen(x[j]) - m) * a.scale, p = expf(d) / s;
            v = (j == id ? gl : 0.f) - gl * p - ge * p * (fmaxf(d, -FLT_MAX) - ln_s + h);
        }
        dx[j] = narrowed<T>(v * a.scale);
    }
}

}  // namespace

sage_status token_log_probs(Context &ctx, const LogProbs &a) {
    if (!a.logits.rows) return SAGE_OK;
    ctx.note_launch("token_log_probs");
    if (ctx.dry()) return SAGE_OK;
    return with_type(a.logits.dtype, [&](auto t) {
        return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), log_probs_kernel<decltype(t)>, dim3((unsigned)a.logits.rows), dim3(kThreads), 0, a), "token_log_probs");
    });
}

sage_status token_log_probs_grad(Context &ctx, const LogProbsGrad &a) {
    if (!a.logits.rows) return SAGE_OK;
    ctx.note_launch("token_log_probs_grad");
    if (ctx.dry()) return SAGE_OK;
    return with_type(a.logits.dtype, [&](auto t) {
        return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), log_probs_grad_kernel<decltype(t)>, dim3((unsigned)a.logits.rows), dim3(kThreads), 0, a), "token_log_probs_grad");
    });
}

sage_status token_log_probs_and_grad(Context &ctx, const LogProbsGrad &a, const VectorArg &log_probs, const VectorArg &entropy) {
    if (!a.logits.rows) return SAGE_OK;
    Block *scratch = ctx.allocator().alloc((size_t)a.logits.rows * 12);
    if (!scratch) return ctx.fail(SAGE_ERR_OOM, "token_log_probs_and_grad: out of memory");
    LogProbs f;
    f.logits = a.logits;
    f.ids = a.ids;
    f.scale = a.scale;
    f.log_probs = log_probs;
    f.stats = RowsArg{scratch->ptr, SAGE_F32, a.logits.rows, 2, 2};
    f.entropy = entropy.ptr ? entropy : VectorArg{(float *)scratch->ptr + 2 * a.logits.rows, 1};
    LogProbsGrad b = a;
    b.stats = f.stats;
    b.entropy = f.entropy;
    sage_status st = token_log_probs(ctx, f);
    if (!st) st = token_log_probs_grad(ctx, b);
    ctx.allocator().free(scratch);
    return st;
}

}  // namespace k
}  // namespace sage
