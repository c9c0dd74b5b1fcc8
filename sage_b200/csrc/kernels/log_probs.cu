// Log probabilities of given tokens, with entropy, alternatives and gradient.
//
// With x the row's logits, c the scale, m = max x, S = sum exp(c (x - m)):
//   log p_j = c (x_j - m) - ln S,   H = ln S - sum c (x_j - m) exp(c (x_j - m)) / S.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

// ------------------------------------------------------------------------------------------ elements
constexpr float kLeast = -200.f, kLn2 = 0.69314718055994531f;
// 16 bytes of a row as they lie in memory.  `kFill` stands for elements outside the row: -inf, which adds nothing.
template <class T>
struct Bits;
template <>
struct Bits<float> {
    static constexpr int N = 4;
    static constexpr unsigned kFill = 0xff800000u;
    __device__ static unsigned element(const void *p) { return *(const unsigned *)p; }
    __device__ static void put(uint4 &v, int j, unsigned e) { (&v.x)[j] = e; }
    __device__ static float largest(const uint4 &v) { return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))); }
    __device__ static unsigned bound(float) { return 0; }
    __device__ static uint4 bounded(const uint4 &v, unsigned) { return v; }
    __device__ static float2 exponents(float2 t) { return make_float2(fmaxf(t.x, kLeast), fmaxf(t.y, kLeast)); }
    __device__ static void unpack(const uint4 &v, float2 *x) {
        x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ static uint4 packed(const float2 *x) { return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y)); }
};
__device__ __forceinline__ __half2 narrowed_pair(__half2 *, float2 x) { return __float22half2_rn(x); }
__device__ __forceinline__ __nv_bfloat162 narrowed_pair(__nv_bfloat162 *, float2 x) { return __float22bfloat162_rn(x); }
__device__ __forceinline__ __half2 rounded_down(__half2 *, float x) { return __half2half2(__float2half_rd(x)); }
__device__ __forceinline__ __nv_bfloat162 rounded_down(__nv_bfloat162 *, float x) { return __bfloat162bfloat162(__float2bfloat16_rd(x)); }
__device__ __forceinline__ float2 widened_pair(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 widened_pair(__nv_bfloat162 x) {  // an f32's upper half
    const unsigned w = *reinterpret_cast<const unsigned *>(&x);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T, class T2>
struct Bits16 {
    static constexpr int N = 8;
    __device__ static unsigned element(const void *p) { return *(const unsigned short *)p; }
    __device__ static void put(uint4 &v, int j, unsigned e) {
        unsigned &w = (&v.x)[j / 2];
        w = j % 2 ? (w & 0xffffu) | e << 16 : (w & 0xffff0000u) | e;
    }
    __device__ static T2 pair(unsigned w) { return *reinterpret_cast<T2 *>(&w); }
    __device__ static float largest(const uint4 &v) {  // two at a time; NaN loses
        const T2 h = __hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w)));
        return fmaxf(widen(h.x), widen(h.y));
    }
    // `least` rounded down, twice; and the elements, none below it.  NaN stays.
    __device__ static unsigned bound(float least) {
        const T2 h = rounded_down((T2 *)nullptr, least);
        return *reinterpret_cast<const unsigned *>(&h);
    }
    __device__ static uint4 bounded(const uint4 &v, unsigned least) {
        uint4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T2 h = __hmax2_nan(pair((&v.x)[i]), pair(least));
            (&y.x)[i] = *reinterpret_cast<const unsigned *>(&h);
        }
        return y;
    }
    __device__ static float2 exponents(float2 t) { return t; }
    __device__ static void unpack(const uint4 &v, float2 *x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = widened_pair(pair((&v.x)[i]));
    }
    __device__ static uint4 packed(const float2 *x) {
        uint4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T2 h = narrowed_pair((T2 *)nullptr, x[i]);
            (&v.x)[i] = *reinterpret_cast<const unsigned *>(&h);
        }
        return v;
    }
};
template <>
struct Bits<__half> : Bits16<__half, __half2> {
    static constexpr unsigned kFill = 0xfc00fc00u;
};
template <>
struct Bits<__nv_bfloat16> : Bits16<__nv_bfloat16, __nv_bfloat162> {
    static constexpr unsigned kFill = 0xff80ff80u;
};

// A row cut into 16-byte vectors at addresses that are multiples of 16: vector i holds elements i * N - head onwards, and those of
// [first, full) lie wholly in the row.  The others are read element by element, so nothing outside the row is touched.
template <class T>
struct RowVectors {
    static constexpr int N = Bits<T>::N;
    const char *origin;  // of vector 0; in front of the row when head > 0
    int head, first, full, count, cols;
    __device__ RowVectors(const void *row, long long cols_) {
        head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        origin = (const char *)row - head * sizeof(T);
        cols = (int)cols_;
        first = head ? 1 : 0;
        full = (int)((head + cols_) / N);
        count = (int)((head + cols_ + N - 1) / N);
    }
    __device__ __forceinline__ bool whole(int i) const { return i >= first && i < full; }
    __device__ __forceinline__ bool ragged() const { return first != 0 || full != count; }
    __device__ __forceinline__ int element(int i) const { return i * N - head; }
    __device__ __forceinline__ uint4 load(int i) const { return whole(i) ? __ldcg(reinterpret_cast<const uint4 *>(origin) + i) : load_edge(i); }
    // Vectors i, i + STEP ...: those in front of `end`.
    template <int U, int STEP>
    __device__ __forceinline__ void load_all(uint4 (&v)[U], int i, int end) const {
        const uint4 *p = reinterpret_cast<const uint4 *>(origin) + i;
        const int stop = min(end, full);
        if (i >= first && i + (U - 1) * STEP < stop) {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = __ldcg(p + u * STEP);
            return;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = nothing();
            if (i + u * STEP < stop && (u > 0 || i >= first)) v[u] = __ldcg(p + u * STEP);
        }
        if (!ragged()) return;
#pragma unroll 1
        for (int at = 0; at < count; at += max(count - 1, 1)) {  // the row's first and last vector, where they reach beyond it
            if (whole(at) || at < i || at >= end || at > i + (U - 1) * STEP || (at - i) % STEP) continue;
            const uint4 e = load_edge(at);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * STEP == at) v[u] = e;
        }
    }
    __device__ __noinline__ uint4 load_edge(int i) const {
        uint4 v = nothing();
        const int e = element(i);
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (e + j >= 0 && (unsigned)(e + j) < (unsigned)cols) Bits<T>::put(v, j, Bits<T>::element(origin + 16ll * i + j * (int)sizeof(T)));
        return v;
    }
    __device__ __forceinline__ static uint4 nothing() { return make_uint4(Bits<T>::kFill, Bits<T>::kFill, Bits<T>::kFill, Bits<T>::kFill); }
};

__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; below 2^-126 zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------ sums of a part of a row
// The part's largest logit m, s = sum of 2^t and w = sum of t 2^t with t = c2 (x - m), c2 = c log2(e); with m = -inf both are relative
// to 0.  Differences are taken before they are scaled, so that a large m costs nothing.  Below 2^-200 a term is zero, and t is held at
// kLeast in w: a masked logit adds 0 times a number.
struct Sums {
    float m = -INFINITY, s = 0.f, w = 0.f;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
// Makes the sums relative to `m`.  A factor of zero takes all with it (a part of masks of the type's lowest value), NaN stays in s.
__device__ __forceinline__ void move_to(Sums &a, float m, float c2) {
    const float t = (a.m - base_of(m)) * c2, f = exp2_fast(t);
    a.w = f > 0.f ? f * (a.w + t * a.s) : 0.f;
    a.s *= f;
    a.m = m;
}
// `used`: how many of the vectors the block's threads have; the others are empty in all of them.
template <class T, int U>
__device__ __forceinline__ void add_vectors(Sums &a, const uint4 (&v)[U], float c2, int used = U) {
    float m = Bits<T>::largest(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) m = fmaxf(m, Bits<T>::largest(v[u]));
    if (m > a.m) move_to(a, m, c2);
    const float2 base = both(-base_of(a.m)), factor = both(c2);
    float2 s = make_float2(a.s, 0.f), w = make_float2(a.w, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u >= used) break;
        float2 x[Bits<T>::N / 2];
        Bits<T>::unpack(v[u], x);
#pragma unroll
        for (int j = 0; j < Bits<T>::N / 2; ++j) {
            const float2 t = mul2(add2(x[j], base), factor), e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
            s = add2(s, e);
            w = fma2(e, make_float2(fmaxf(t.x, kLeast), fmaxf(t.y, kLeast)), w);
        }
    }
    a.s = s.x + s.y;
    a.w = w.x + w.y;
}
// Where the largest logit is of ordinary size, differences may be scaled first: t = fma(c2, x, -b) with b = c2 m, rounded once and the same for all,
// is as exact, and one instruction less for two elements; and 16-bit logits can be held at m + kLeast / c2, two to an instruction, in place of t.
// `least`: that bound, or Bits<T>::kFill where this form is not open (b large, its rounding then reaching kLeast; the bound not finite).  Values and
// gradient without it and with it, on one GPU: 4096 x 131072 f32 811 and 796 us, 8192 x 32000 bf16 211 and 208; for a second on end, with the clock down
// to 1.8 GHz at the power limit, 4096 x 131072 f32 817 and 801.  8192 x 131072 bf16 is the same with both.
template <class T>
struct Ordinary {
    float b, rest;  // t relative to b is t relative to m, plus `rest`
    unsigned least;
    __device__ Ordinary(float base, float c2) {
        b = base * c2;
        rest = fmaf(base, c2, -b);
        least = fabsf(b) < 1e6f && c2 < 1e6f ? Bits<T>::bound(base + __fdividef(kLeast, c2)) : Bits<T>::kFill;
    }
    __device__ bool open() const { return least != Bits<T>::kFill; }
};
// The sums of all the vectors that the thread has.
template <class T, int U>
__device__ __forceinline__ void sum_vectors(Sums &a, const uint4 (&v)[U], float c2, int used) {
    float m = Bits<T>::largest(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) m = fmaxf(m, Bits<T>::largest(v[u]));
    const Ordinary<T> o(base_of(m), c2);
    if (!o.open()) {
        add_vectors<T, U>(a, v, c2, used);
        return;
    }
    const float2 base = both(-o.b), factor = both(c2);
    float2 s = make_float2(0.f, 0.f), w = s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u >= used) break;
        float2 x[Bits<T>::N / 2];
        Bits<T>::unpack(Bits<T>::bounded(v[u], o.least), x);
#pragma unroll
        for (int j = 0; j < Bits<T>::N / 2; ++j) {
            const float2 t = fma2(x[j], factor, base), e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
            s = add2(s, e);
            w = fma2(e, Bits<T>::exponents(t), w);
        }
    }
    const float f = exp2_fast(-o.rest), all = s.x + s.y;
    a.m = m;
    a.s = f * all;
    a.w = f * (w.x + w.y - o.rest * all);
}
// Of the warp's lanes: the largest m first, then sums relative to it.  In all lanes; or, where those behind the first LANES have nothing, in
// these (8192 x 131072 bf16 with its gradient: 1.7 % less with as many lanes as there are warps and CTAs than with 32 everywhere).
template <int LANES = 32>
__device__ __forceinline__ Sums warp_join(Sums a, float c2) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(a.m));
    move_to(a, m, c2);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    }
    return a;
}
// Of all threads, in warp 0 (its first LANES lanes).  `shared`: one for each warp.
constexpr int kMaxCluster = 8;  // CTAs that share a row
template <int THREADS>
constexpr int kJoinLanes = THREADS / 32 < kMaxCluster ? kMaxCluster : THREADS / 32;  // for each warp, and one to send to each CTA
template <int THREADS, int LANES>
__device__ __forceinline__ Sums block_join(Sums a, float c2, Sums *shared) {
    a = warp_join(a, c2);
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = a;
    __syncthreads();
    return threadIdx.x < 32 ? warp_join<LANES>((int)threadIdx.x < THREADS / 32 ? shared[threadIdx.x] : Sums(), c2) : a;
}

// ------------------------------------------------------------------------------------------ clusters: CTAs that share a row
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_number() {
    unsigned r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }  // of a thread with nothing to show
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// The address in CTA `rank`'s shared memory of what lies at `p` in this one's.
__device__ __forceinline__ unsigned peer_shared(const void *p, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void peer_store(unsigned a, float x) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory"); }
__device__ __forceinline__ void peer_store(unsigned a, unsigned long long x) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(x) : "memory"); }

// ------------------------------------------------------------------------------------------ alternatives
// Larger for larger logits and, among equals, for lower tokens; no two tokens of a row have the same, and none has 0.  NaN counts as -inf.
__device__ __forceinline__ unsigned rank_bits(float x) {
    x = x != x ? -INFINITY : x + 0.f;  // -0 and 0 are equal
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long rank_key(float x, unsigned token) { return (unsigned long long)rank_bits(x) << 32 | (0xffffffffu - token); }
__device__ __forceinline__ float rank_logit(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// The warp's largest keys, sorted over its lanes; `least` is the k-th, what a key has to pass.
struct TopList {
    unsigned long long key = 0, least = 0;
    __device__ __forceinline__ void offer(unsigned long long x, bool want, int k) {
        unsigned todo = __ballot_sync(0xffffffffu, want && x > least);
        while (todo) {
            const unsigned long long y = __shfl_sync(0xffffffffu, x, __ffs(todo) - 1);
            todo &= todo - 1;
            if (y <= least) continue;
            const unsigned lane = threadIdx.x % 32, at = __popc(__ballot_sync(0xffffffffu, key > y));
            const unsigned long long before = __shfl_up_sync(0xffffffffu, key, 1);
            key = lane < at ? key : lane == at ? y : before;
            least = __shfl_sync(0xffffffffu, key, k - 1);
        }
    }
};

constexpr int kCandidates = 256;
template <int THREADS>
struct TopShared {
    unsigned short chosen[THREADS];
    int sets, found;
    unsigned long long candidates[kCandidates], best[kMaxTop], lists[THREADS / 32][kMaxTop];
};

// best[0 .. k) = the k largest of `keys` (0 = none), sorted: a key's place is how many are above it.  best is 0 before; the block calls this
// together and waits before it reads.
__device__ __forceinline__ void sort_by_rank(const unsigned long long *keys, int n, int k, unsigned long long *best) {
    for (int t = threadIdx.x; t < n; t += blockDim.x) {
        const unsigned long long key = keys[t];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) above += keys[j] > key;
        if (key && above < k) best[above] = key;
    }
}

// The k largest of the block's vectors [begin, end), sorted, in sh.best.  Each thread knows the largest of the vectors it has summed
// (begin + its number + multiples of THREADS).  The k-th largest of those maxima bounds the k-th largest element from below, and only
// threads whose maximum reaches it hold candidates: about k of them, whose vectors are read again (from L2) and whose candidates are
// ranked.  The bound is taken to 16 bits of the order, which ties and nearness make a little lower; where that lets many threads in (masks
// that leave less than k tokens, equal logits), to all bits, the token's among them.  Where there are more candidates than the list holds
// all the same (thousands of open tokens in a few threads, the others masked), everything is read again in order, into sorted lists.
template <class T, int THREADS>
__device__ void block_top(const RowVectors<T> &row, int begin, int end, float thread_max, int k, TopShared<THREADS> &sh) {
    constexpr int N = Bits<T>::N, W = THREADS / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, own = begin + (int)threadIdx.x;
    unsigned long long mine = own < end ? (unsigned long long)rank_bits(thread_max) << 32 : 0, bound = 0;
    for (int bit = 63; bit >= 48; --bit) {
        const unsigned long long t = bound | 1ull << bit;
        if (__syncthreads_count(mine >= t) >= k) bound = t;
    }
    if (__syncthreads_count(mine >= bound) > THREADS / 4) {
        const unsigned top = rank_bits(thread_max);
        int token = -1;  // the first of the thread's largest
        for (int i = own; i < end && token < 0; i += THREADS) {
            float2 x[N / 2];
            Bits<T>::unpack(row.load(i), x);
#pragma unroll
            for (int j = N - 1; j >= 0; --j)
                if (rank_bits(j % 2 ? x[j / 2].y : x[j / 2].x) == top && (unsigned)(row.element(i) + j) < (unsigned)row.cols) token = row.element(i) + j;
        }
        mine = token >= 0 ? (unsigned long long)top << 32 | (0xffffffffu - (unsigned)token) : 0;
        const int token_bits = 32 - __clz(row.cols);  // the bits above them are set in every key
        for (int bit = 47; bit >= 0; --bit) {
            const unsigned long long t = bound | 1ull << bit;
            if ((bit < 32 && bit >= token_bits) || __syncthreads_count(mine >= t) >= k) bound = t;
        }
        if (__syncthreads_count(mine >= bound) < k) bound = 0;  // fewer than k threads have anything
    }
    if (threadIdx.x == 0) sh.sets = sh.found = 0;
    if (threadIdx.x < kMaxTop) sh.best[threadIdx.x] = 0;
    __syncthreads();
    if (mine >= bound) sh.chosen[atomicAdd(&sh.sets, 1)] = (unsigned short)threadIdx.x;  // in any order: keys decide
    __syncthreads();
    const int sets = sh.sets;
    // The warp's vectors i, i + step ... in front of `end`, each lane its own: f(key, is it one)
    auto each = [&](int i, int step, auto f) {
        for (; __any_sync(0xffffffffu, i < end); i += step) {
            const bool some = i < end;
            const uint4 v = some ? row.load(i) : RowVectors<T>::nothing();
            float2 x[N / 2];
            Bits<T>::unpack(v, x);
            const int e = row.element(i);
            bool any = false;
#pragma unroll
            for (int j = 0; j < N; ++j) any |= rank_bits(j % 2 ? x[j / 2].y : x[j / 2].x) >= (unsigned)(bound >> 32);
            if (!__any_sync(0xffffffffu, any && some)) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned long long key = rank_key(j % 2 ? x[j / 2].y : x[j / 2].x, (unsigned)(e + j));
                f(key, some && (unsigned)(e + j) < (unsigned)row.cols && key >= bound);
            }
        }
    };
    const bool few = sets <= THREADS / 4;
    if (few) {
        int lanes = 32;  // to a thread's vectors: as many as it has, and the other lanes to other threads'
        while (lanes > 1 && lanes / 2 * THREADS >= end - begin) lanes /= 2;
        for (int q0 = 0; q0 < sets; q0 += W * (32 / lanes)) {
            const int q = q0 + lane / lanes * W + warp;
            each(q < sets ? begin + sh.chosen[q] + lane % lanes * THREADS : end, lanes * THREADS, [&](unsigned long long key, bool in) {
                if (!in) return;
                const int at = atomicAdd(&sh.found, 1);
                if (at < kCandidates) sh.candidates[at] = key;
            });
        }
    }
    __syncthreads();
    if (few && sh.found <= kCandidates) {
        sort_by_rank(sh.candidates, sh.found, k, sh.best);
    } else {
        TopList list;
        each(own, THREADS, [&](unsigned long long key, bool in) { list.offer(key, in, k); });
        sh.lists[warp][lane] = lane < k ? list.key : 0;
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < W; ++w) list.offer(sh.lists[w][lane], true, k);
            sh.best[lane] = lane < k ? list.key : 0;
        }
    }
    __syncthreads();
}

// scale (x - m) - ln S, where x - m is beyond f32 too.
__device__ __forceinline__ float log_prob(float x, float base, float scale, float ln_s) {
    const float d = x - base;
    return (fabsf(d) <= FLT_MAX ? d * scale : x * scale - base * scale) - ln_s;
}

// ------------------------------------------------------------------------------------------ values
// A cluster of 2^shift CTAs for each row; each reads a part of it once, and the running maximum and sums are joined over lanes, warps and CTAs.
// Bound by memory in many rows (8192 x 50021 f32: 268 us, 6.1 TB/s), by the chain of joins in few (1 x 30522: 6 us with 5 alternatives).
template <class T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) log_probs_kernel(const LogProbs a, const int shift) {
    constexpr int U = 4;
    __shared__ Sums sums[THREADS / 32], part_sums[kMaxCluster];
    __shared__ unsigned long long part_lists[TOP ? kMaxCluster * kMaxTop : 1];
    __shared__ TopShared<TOP ? THREADS : 32> top;
    grid_dependency_sync();
    const int parts = 1 << shift;
    if (parts > 1) cluster_arrive_relaxed();
    const long long r = blockIdx.x >> shift;
    const unsigned rank = parts > 1 ? cluster_rank() : 0;
    const T *x = (const T *)a.logits.ptr + r * a.logits.pitch;
    const RowVectors<T> row(x, a.logits.cols);
    const int each = (row.count + parts - 1) >> shift, begin = (int)rank * each, end = min(begin + each, row.count);
    const float c2 = a.scale * kLog2E;
    float own = 0.f;
    bool scored = false;
    if (rank == 0 && threadIdx.x == 0 && a.ids.ptr) {
        const int id = ((const int *)a.ids.ptr)[r * a.ids.stride];
        scored = id >= 0 && id < a.logits.cols;
        if (scored) own = widen(x[id]);
    }
    Sums mine;
    for (int i = begin + (int)threadIdx.x; i < end; i += THREADS * U) {
        uint4 v[U];
        row.template load_all<U, THREADS>(v, i, end);
        add_vectors<T, U>(mine, v, c2);
    }
    const float thread_max = mine.m;
    Sums all = block_join<THREADS, TOP ? 32 : kJoinLanes<THREADS>>(mine, c2, sums);
    if constexpr (TOP) block_top<T, THREADS>(row, begin, end, thread_max, a.top, top);
    const int lane = threadIdx.x % 32;
    if (parts > 1) {  // everything to the first CTA, which has started when the wait ends
        cluster_wait();
        if (threadIdx.x == 0) {
            const unsigned to = peer_shared(&part_sums[rank], 0);
            peer_store(to, all.m);
            peer_store(to + 4, all.s);
            peer_store(to + 8, all.w);
        }
        if (TOP && (int)threadIdx.x < a.top) peer_store(peer_shared(&part_lists[rank * a.top + threadIdx.x], 0), top.best[threadIdx.x]);
        if (threadIdx.x < 32) cluster_arrive();
        else cluster_arrive_relaxed();
        cluster_wait();
        if (rank) return;
        if constexpr (TOP) {
            if (threadIdx.x < kMaxTop) top.best[threadIdx.x] = 0;
            __syncthreads();
            sort_by_rank(part_lists, parts * a.top, a.top, top.best);
            __syncthreads();
        }
        if (threadIdx.x < 32) all = warp_join<TOP ? 32 : kMaxCluster>(lane < parts ? part_sums[lane < parts ? lane : 0] : Sums(), c2);
    }
    if (threadIdx.x >= 32) return;
    const float base = base_of(all.m), ln_s = logf(all.s);
    const bool none = all.s == 0.f;
    if (threadIdx.x == 0) {
        if (a.log_probs.ptr) ((float *)a.log_probs.ptr)[r * a.log_probs.stride] = !scored ? 0.f : none ? -INFINITY : log_prob(own, base, a.scale, ln_s);
        if (a.entropy.ptr) ((float *)a.entropy.ptr)[r * a.entropy.stride] = none ? 0.f : ln_s - kLn2 * (all.w / all.s);
        if (a.stats.ptr) {
            ((float *)a.stats.ptr)[r * a.stats.pitch] = all.m;
            ((float *)a.stats.ptr)[r * a.stats.pitch + 1] = all.s;
        }
    }
    if (TOP && (int)threadIdx.x < a.top) {
        const unsigned long long key = top.best[lane];
        ((int *)a.top_ids.ptr)[r * a.top_ids.pitch + lane] = (int)(0xffffffffu - (unsigned)key);
        if (a.top_log_probs.ptr) ((float *)a.top_log_probs.ptr)[r * a.top_log_probs.pitch + lane] = none ? -INFINITY : log_prob(rank_logit(key), base, a.scale, ln_s);
    }
}

// ------------------------------------------------------------------------------------------ gradient
// With t = c2 (x - m), e = 2^t, p = e / S and K = H - ln S:
//   dx_j = c gl (delta - p_j) - c ge p_j (ln2 t_j + K) = e (slope t_j + level) + c gl delta.
struct GradRow {
    float base, c2, slope, level, at_id;
    int id;
    unsigned least;
    __device__ void set(float m, float s, float ln_s, float scale, float gl, float ge, float entropy, int id_) {
        base = base_of(m);
        c2 = scale * kLog2E;
        id = id_;
        if (s == 0.f) gl = ge = 0.f;  // masked throughout
        const float share = s == 0.f ? 0.f : scale / s;
        slope = -share * (ge * kLn2);
        level = -share * (ge != 0.f ? gl + ge * (entropy - ln_s) : gl);  // NaN where s is: so is every gradient
        at_id = scale * gl;
    }
    // Behind set(): into the form with scaled differences, where it is open.
    template <class T>
    __device__ void scale_first() {
        const Ordinary<T> o(base, c2);
        least = o.least;
        if (o.open()) {  // relative to b
            const float f = exp2_fast(-o.rest);
            base = o.b;
            level = f * (level - slope * o.rest);
            slope *= f;
        }
    }
    // The gradients at one vector's logits, in the logits' type; `own`: the token's place in the vector, if it is there.
    template <class T, bool ORDINARY>
    __device__ __forceinline__ uint4 gradient(const uint4 &v, bool has_own, int own) const {
        constexpr int N = Bits<T>::N;
        const float2 b = both(-base), f = both(c2), k = both(slope), l = both(level);
        float2 x[N / 2];
        Bits<T>::unpack(ORDINARY ? Bits<T>::bounded(v, least) : v, x);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            float2 t = ORDINARY ? Bits<T>::exponents(fma2(x[j], f, b)) : mul2(add2(x[j], b), f);
            if (!ORDINARY) t = make_float2(fmaxf(t.x, kLeast), fmaxf(t.y, kLeast));  // masked: 0 times a number
            x[j] = mul2(make_float2(exp2_fast(t.x), exp2_fast(t.y)), fma2(k, t, l));
        }
        if (has_own) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j == own) (j % 2 ? x[j / 2].y : x[j / 2].x) += at_id;
        }
        return Bits<T>::packed(x);
    }
};

template <class T>
__device__ __noinline__ void store_elements(T *dx, int e, int cols, uint4 g) {
    Pack<T> out;
    *reinterpret_cast<uint4 *>(out.v) = g;
#pragma unroll
    for (int j = 0; j < Pack<T>::N; ++j)
        if ((unsigned)(e + j) < (unsigned)cols) dx[e + j] = out.v[j];
}
// Gradients at the vectors that load_all loaded.  `same` says that the results lie on the same 16-byte grid as the logits, where one
// store writes a vector.
template <class T, int U, int STEP, bool ORDINARY>
__device__ __forceinline__ void store_some(const RowVectors<T> &row, const GradRow &g, T *dx, bool same, const uint4 (&v)[U], int i, int end) {
    uint4 *p = reinterpret_cast<uint4 *>(dx + row.element(0)) + i;
    constexpr int N = Bits<T>::N;
    const int from_own = g.id >= 0 ? (g.id + row.head) / N - i : -1, own = (g.id + row.head) % N;  // in vectors
    if (same && i >= row.first && i + (U - 1) * STEP < min(end, row.full)) {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u * STEP] = g.gradient<T, ORDINARY>(v[u], from_own == u * STEP, own);
        return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (i + u * STEP >= end) return;
        const uint4 out = g.gradient<T, ORDINARY>(v[u], from_own == u * STEP, own);
        if (same && row.whole(i + u * STEP)) p[u * STEP] = out;
        else store_elements(dx, row.element(i + u * STEP), row.cols, out);
    }
}
template <class T, int U, int STEP>
__device__ __forceinline__ void store_all(const RowVectors<T> &row, const GradRow &g, T *dx, bool same, const uint4 (&v)[U], int i, int end) {
    if (g.least != Bits<T>::kFill) store_some<T, U, STEP, true>(row, g, dx, same, v, i, end);
    else store_some<T, U, STEP, false>(row, g, dx, same, v, i, end);
}
template <class T>
__device__ __forceinline__ bool same_grid(const T *x, const T *dx) { return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0; }

__device__ __forceinline__ float at_row(const VectorArg &v, long long r) { return v.ptr ? ((const float *)v.ptr)[r * v.stride] : 0.f; }
__device__ __forceinline__ int token_of(const LogProbsGrad &a, long long r) {
    const int id = ((const int *)a.ids.ptr)[r * a.ids.stride];
    return id >= 0 && id < a.logits.cols ? id : -1;
}

// From the forward pass's sums: `pieces` blocks for a row, kGradVectors vectors each.  Bound by memory: a read and a write (4096 x
// 30522 f32: 151 us, 6.6 TB/s; with scaled differences, worked out by each thread, 157).
constexpr int kGradVectors = 1024;
template <class T>
__global__ void __launch_bounds__(256) log_probs_grad_kernel(const LogProbsGrad a, const unsigned pieces) {
    constexpr int U = kGradVectors / 256;
    grid_dependency_sync();
    const long long r = blockIdx.x / pieces;
    const int piece = blockIdx.x - (unsigned)r * pieces;
    const T *x = (const T *)a.logits.ptr + r * a.logits.pitch;
    T *dx = (T *)a.dlogits.ptr + r * a.dlogits.pitch;
    const RowVectors<T> row(x, a.logits.cols);
    const int i = piece * kGradVectors + threadIdx.x;
    uint4 v[U];
    row.template load_all<U, 256>(v, i, row.count);
    const float *stats = (const float *)a.stats.ptr + r * a.stats.pitch;
    const int id = token_of(a, r);
    GradRow g;
    g.set(stats[0], stats[1], logf(stats[1]), a.scale, id >= 0 ? at_row(a.g_log_probs, r) : 0.f, at_row(a.g_entropy, r), at_row(a.entropy, r), id);
    const bool same = same_grid(x, dx);
    store_some<T, U, 256, false>(row, g, dx, same, v, i, row.count);
}

// Values and gradient together: a cluster holds its row in registers (NV vectors for each thread) between the sums and the
// gradient, so the logits are read once.  All CTAs of the cluster give their sums to all.  Bound by memory and by the joins
// that each row waits for between its loads and its stores (8192 x 131072 bf16: 915 us, 4.7 TB/s; without the joins it would be
// 657), so nothing else is left to be waited for there: what the row is asked about is fetched beside its logits (8192 x 50021
// bf16: 384 us with those loads behind the join, 369 beside; 4096 x 131072 f32: 865 and 818).
template <class T, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) log_probs_and_grad_kernel(const LogProbsGrad a, const VectorArg log_probs, const VectorArg entropy, const int parts, const int each) {
    __shared__ Sums sums[THREADS / 32], part_sums[kMaxCluster];
    __shared__ GradRow constants;
    __shared__ struct {
        int id;
        float g_log_prob, g_entropy, own;
    } asked;
    grid_dependency_sync();
    if (parts > 1) cluster_arrive_relaxed();
    const long long r = cluster_number();
    const unsigned rank = parts > 1 ? cluster_rank() : 0;
    const T *x = (const T *)a.logits.ptr + r * a.logits.pitch;
    T *dx = (T *)a.dlogits.ptr + r * a.dlogits.pitch;
    const RowVectors<T> row(x, a.logits.cols);
    const int begin = min((int)rank * each, row.count), end = min(begin + each, row.count), i = begin + (int)threadIdx.x;
    const float c2 = a.scale * kLog2E;
    // What the row is asked about, fetched by the last thread while the logits are under way.
    const bool asks = threadIdx.x == THREADS - 1;
    int id = -1;
    float g_log_prob = 0.f, g_entropy = 0.f, own = 0.f;
    if (asks) {
        id = ((const int *)a.ids.ptr)[r * a.ids.stride];
        g_log_prob = at_row(a.g_log_probs, r);
        g_entropy = at_row(a.g_entropy, r);
    }
    uint4 v[NV];
    row.template load_all<NV, THREADS>(v, i, end);
    if (asks && id >= 0 && id < a.logits.cols) own = widen(x[id]);
    Sums all;
    sum_vectors<T, NV>(all, v, c2, (end - begin + THREADS - 1) / THREADS);
    if (asks) {
        const bool scored = id >= 0 && id < a.logits.cols;
        asked.id = scored ? id : -1;
        asked.g_log_prob = scored ? g_log_prob : 0.f;
        asked.g_entropy = g_entropy;
        asked.own = own;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) asm volatile("" : "+r"(v[u].x), "+r"(v[u].y), "+r"(v[u].z), "+r"(v[u].w));  // as loaded: unpacked twice rather than kept unpacked
    all = block_join<THREADS, kJoinLanes<THREADS>>(all, c2, sums);
    if (parts > 1) {
        cluster_wait();
        if ((int)threadIdx.x < parts) {
            const unsigned to = peer_shared(&part_sums[rank], threadIdx.x);
            peer_store(to, all.m);
            peer_store(to + 4, all.s);
            peer_store(to + 8, all.w);
        }
        // Behind the token's own logit too, which was read in front of the block's join: from here on results may take the logits' place.
        if (threadIdx.x < 32) cluster_arrive();
        else cluster_arrive_relaxed();
        cluster_wait();
    }
    if (threadIdx.x < 32) {  // the row's constants once; a thread's other work is 64 elements
        const int lane = threadIdx.x;
        if (parts > 1) all = warp_join<kMaxCluster>(lane < parts ? part_sums[lane < parts ? lane : 0] : Sums(), c2);
        const float ln_s = logf(all.s);
        const bool none = all.s == 0.f;
        const float h = none ? 0.f : ln_s - kLn2 * (all.w / all.s);
        if (lane == 0) {
            constants.set(all.m, all.s, ln_s, a.scale, asked.g_log_prob, asked.g_entropy, h, asked.id);
            constants.scale_first<T>();
        } else if (lane == 1 && rank == 0) {
            ((float *)log_probs.ptr)[r * log_probs.stride] = asked.id < 0 ? 0.f : none ? -INFINITY : log_prob(asked.own, base_of(all.m), a.scale, ln_s);
            if (entropy.ptr) ((float *)entropy.ptr)[r * entropy.stride] = h;
        }
    }
    __syncthreads();
    const GradRow g = constants;
    const bool same = same_grid(x, dx);
    store_all<T, NV, THREADS>(row, g, dx, same, v, i, end);
}

// The most 16-byte vectors that a row touches.
long long most_vectors(const RowsArg &x) {
    const long long size = x.dtype == SAGE_F32 ? 4 : 2, n = 16 / size;
    const bool fixed = x.rows <= 1 || x.pitch * size % 16 == 0;  // every row starts at the same place of a vector
    const long long head = fixed ? (long long)(reinterpret_cast<uintptr_t>(x.ptr) % 16) / size : n - 1;
    return (head + x.cols + n - 1) / n;
}

int log2_of(int power) { return __builtin_ctz((unsigned)power); }

// The block's size: small blocks, of which more run on an SM, interleave reading and joining better, as long as there are rows for them (8192 x
// 50021 f32: 259, 269 and 283 us with 128, 256 and 512 threads; 16384 x 8000: 85, 103 and 148); with few rows the largest, a cluster of eight of
// which reads a row fastest (64 x 131072 bf16 with 20 alternatives: 14.4 us with 256 threads, 10.8 with 512; 19.2 and 16.7 where masks leave parts of
// rows empty; 73 rows 14.8 and 17.5).  Alternatives are found by few threads, which have more to read again in long rows of small
// blocks (3000 x 131072 bf16 with 20: 234 us with 128 threads, 191 with 256).
int threads_of_rows(long long rows, long long bytes, bool top, int sms) {
    if (bytes <= 16384 || (rows >= 16ll * sms && (!top || bytes <= 65536))) return 128;
    return rows * kMaxCluster < 4ll * sms ? 512 : 256;
}

// How many CTAs share a row: the fewest steps of the resident CTAs, each step the part's bytes and a fixed cost that measures like 24 KB of them
// (joining), 128 KB with alternatives (candidates found and ranked); twice that where the cluster's barriers come in (32 x 30522 f32 with 20
// alternatives: 13.8 us with eight CTAs a row, 8.2 with one; 1000 x 131072 bf16 without: 60 us with four, 53 with one).  Clusters of eight do not
// fill all SMs: their number differs from one part of the GPU to the other.  So few rows that they are one step however they are cut have the same
// parts, and the same bits, whether alternatives are asked for or not; there a CTA more costs what reading 7 KB does (one row of 8191 f32 with 20
// alternatives: 6.2, 7.7 and 8.3 us with one, four and eight CTAs; of 30522 7.8, 7.8, 8.4; of 131072 14.4, 9.2, 8.8).
constexpr double kFixed = 24576, kFixedTop = 131072;  // of a block of 512 threads
int parts_of_rows(long long rows, long long bytes, int threads, bool top, int sms) {
    const long long slots = sms * 1024ll / threads, slots8 = slots * 27 / 32;
    const bool few = rows * kMaxCluster <= slots8;
    const double fixed = (top ? kFixedTop : kFixed) * threads / 512;
    int best = 1;
    double least = 0;
    for (int c = 1; c <= kMaxCluster; c *= 2) {
        const long long resident = c == 1 ? slots : c < kMaxCluster ? slots * 15 / 16 : slots8;
        const double one = (double)bytes / c, cost = few ? one + (c == 1 ? 0 : 6144 + 7168 * c) : (double)((rows * c + resident - 1) / resident) * (one + (c == 1 ? fixed : 2 * fixed));
        if (c == 1 || cost < least) {
            best = c;
            least = cost;
        }
    }
    return rows * best > 0x7fffffffll ? 1 : best;
}

}  // namespace

sage_status token_log_probs(Context &ctx, const LogProbs &a) {
    if (!a.logits.rows) return SAGE_OK;
    ctx.note_launch("token_log_probs");
    if (ctx.dry()) return SAGE_OK;
    return with_type(a.logits.dtype, [&](auto t) {
        typedef decltype(t) T;
        const long long bytes = a.logits.cols * (long long)sizeof(T);
        const int threads = threads_of_rows(a.logits.rows, bytes, a.top > 0, ctx.sm_count);
        const int parts = threads == 128 ? 1 : parts_of_rows(a.logits.rows, bytes, threads, a.top > 0, ctx.sm_count);
        auto launch = [&](auto kernel) {
            return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), parts, kernel, dim3((unsigned)(a.logits.rows * parts)), dim3(threads), 0, a, log2_of(parts)), "token_log_probs");
        };
        if (threads == 128) return a.top ? launch(log_probs_kernel<T, 128, true>) : launch(log_probs_kernel<T, 128, false>);
        if (threads == 256) return a.top ? launch(log_probs_kernel<T, 256, true>) : launch(log_probs_kernel<T, 256, false>);
        return a.top ? launch(log_probs_kernel<T, 512, true>) : launch(log_probs_kernel<T, 512, false>);
    });
}

sage_status token_log_probs_grad(Context &ctx, const LogProbsGrad &a) {
    if (!a.logits.rows) return SAGE_OK;
    ctx.note_launch("token_log_probs_grad");
    if (ctx.dry()) return SAGE_OK;
    return with_type(a.logits.dtype, [&](auto t) {
        typedef decltype(t) T;
        const long long pieces = (most_vectors(a.logits) + kGradVectors - 1) / kGradVectors;
        const long long most = 0x7fffffffll / pieces;  // rows of one launch
        for (long long at = 0; at < a.logits.rows; at += most) {
            LogProbsGrad b = a;
            b.logits.rows = a.logits.rows - at < most ? a.logits.rows - at : most;
            b.logits.ptr = (T *)a.logits.ptr + at * a.logits.pitch;
            b.dlogits.ptr = (T *)a.dlogits.ptr + at * a.dlogits.pitch;
            b.stats.ptr = (float *)a.stats.ptr + at * a.stats.pitch;
            for (auto *v : {&b.ids, &b.entropy, &b.g_log_probs, &b.g_entropy})
                if (v->ptr) v->ptr = (float *)v->ptr + at * v->stride;
            sage_status st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), log_probs_grad_kernel<T>, dim3((unsigned)(b.logits.rows * pieces)), dim3(256), 0, b, (unsigned)pieces),
                                            "token_log_probs_grad");
            if (st) return st;
        }
        return (sage_status)SAGE_OK;
    });
}

sage_status token_log_probs_and_grad(Context &ctx, const LogProbsGrad &a, const VectorArg &log_probs, const VectorArg &entropy) {
    if (!a.logits.rows) return SAGE_OK;
    constexpr int NV = 8;
    const long long vectors = most_vectors(a.logits);
    // The smallest blocks eight of which hold a row: more of them run on an SM, and loads, sums and stores of different ones interleave (8192
    // x 131072 bf16: 16 % more time with 512 threads than with 256; 8192 x 50021: 25 % more with 256 than with 128, 40 % with 512).
    const int threads = vectors <= kMaxCluster * 128 * NV ? 128 : vectors <= kMaxCluster * 256 * NV ? 256 : 512;
    int parts = (int)std::min((vectors + threads * NV - 1) / (threads * NV), kMaxCluster + 1ll);
    // Rows that fit the registers of a cluster.
    if (parts <= kMaxCluster && a.logits.rows * kMaxCluster <= 0x7fffffffll) {
        ctx.note_launch("token_log_probs_and_grad");
        if (ctx.dry()) return SAGE_OK;
        // Parts as large as registers hold, whose threads need not look where their vectors end; smaller ones where SMs would be idle.
        int each = threads * NV;
        if (a.logits.rows * parts * threads < ctx.sm_count * 1024ll) {
            parts = (int)std::min<long long>(kMaxCluster, std::max<long long>(parts, ctx.sm_count * 1024ll / (a.logits.rows * threads)));
            parts = (int)std::min<long long>(parts, (vectors + threads - 1) / threads);
            each = (int)((vectors + parts - 1) / parts);
        }
        return with_type(a.logits.dtype, [&](auto t) {
            typedef decltype(t) T;
            auto launch = [&](auto kernel) {
                return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), parts, kernel, dim3((unsigned)(a.logits.rows * parts)), dim3(threads), 0, a, log_probs, entropy, parts, each),
                                      "token_log_probs_and_grad");
            };
            return threads == 128 ? launch(log_probs_and_grad_kernel<T, 128, NV>) : threads == 256 ? launch(log_probs_and_grad_kernel<T, 256, NV>) : launch(log_probs_and_grad_kernel<T, 512, NV>);
        });
    }
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
