// The norms before and after a block of a model, with what joins the block to the residual stream, row by row:
//   n = A(y)              A, B: none, x / sqrt(mean(x^2) + eps) or (x - mean x) / sqrt(mean((x - mean x)^2) + eps), then a weight and a bias
//   out = c x + gate * dropout(n)
//   h = B(out)            (of `out` as it is stored)
// and the gradient for arrivals go (of out) and gh (of h), with u = the unit rows of B's operand, v of A's, keep the mask times its factor:
//   G = go + B'(gh): with q = gh wb, rstd (q - mean(q u) u [- mean q]);   dx = c G;   d gate = sum over rows of G dropout(n)
//   t = G gate keep;   dy = A'(t) likewise;   the weights' and biases' gradients: sums over rows of gh u, gh, t v, t
//
// A thread owns eight neighbouring columns (NV runs of them, where rows are long) and a team of threads a row, so that the sums over
// rows stay in registers, the team's sums over columns are one shuffle tree and one exchange in shared memory, and a block of dropout's mask is
// one draw.  Teams go through rows in steps of their number; what a thread reads of its team's next rows is copied into places of its own in shared
// memory while the present row is worked on (no barrier: only the thread that asked reads them).
// Sums over rows are joined in a fixed order: team by team within a CTA, then CTA by CTA in a second launch.
#include <algorithm>

#include "counter_random.h"
#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {
namespace {

constexpr int kMaxThreads = 512, kMaxTeams = 15;  // named barriers 1 to 15

struct Rows {
    void *p;
    long long pitch;
};

struct NormsArgs {
    Rows x, y, out, h;     // forward: x, y in, out, h out; backward: out, y in
    Rows go, gh, dx, dy;   // backward
    float *stats;          // [rows, 4]: mean and 1 / deviation of A's operand, of B's
    long long stats_pitch;
    const float *wa, *ba, *wb, *bb, *gate;
    long long gate_pitch;
    int after, before;     // sage_norm
    float eps, scale;
    Dropout d;
    int rows, dim;
    int group_rows;        // rows that share a row of the gate
    int team, teams;       // threads that share a row, teams of a CTA
    int stages;            // rows on their way
    int splits;            // of a group's rows
    float *partial;        // backward: [CTA][sum][dim]
    float *gate_partial;   // ... and for gates of several groups [group * splits + split][dim]
    int sums;              // bits: which of kSums are wanted
};
enum { kSumWb, kSumBb, kSumWa, kSumBa, kSumGate, kSums };

__device__ __forceinline__ void copy16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the `later` youngest groups have arrived.
template <int LATER>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// Sums over a team, the same bits in all of its threads.
struct Team {
    int index, lane, warp, warps, threads;
    float *slots;  // [2][warps][4]
    int turn;
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int off = 16; off; off >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
        if (warps == 1) return;
        float *s = slots + turn * warps * 4;
        turn ^= 1;  // (the next sum but one writes here again, behind the next one's barrier)
        if (!lane)
#pragma unroll
            for (int k = 0; k < K; ++k) s[warp * 4 + k] = v[k];
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(threads) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0.f;
        for (int w = 0; w < warps; ++w)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += s[w * 4 + k];
    }
};

template <class T>
__device__ __forceinline__ void load8(const T *p, int count, bool wide, float (&v)[8]) {
    if (wide && count == 8) {
        constexpr int N = Pack<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            const Pack<T> q = ((const Pack<T> *)p)[i];
#pragma unroll
            for (int e = 0; e < N; ++e) v[i * N + e] = widen(q.v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < count ? widen(p[e]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T *p, int count, bool wide, const float (&v)[8]) {
    if (wide && count == 8) {
        constexpr int N = Pack<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            Pack<T> q;
#pragma unroll
            for (int e = 0; e < N; ++e) q.v[e] = narrowed<T>(v[i * N + e]);
            ((Pack<T> *)p)[i] = q;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) p[e] = narrowed<T>(v[e]);
    }
}
// Weights, biases and gates: f32, through L1.
__device__ __forceinline__ void weights8(const float *p, int count, bool wide, float none, float (&v)[8]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = none;
    } else if (wide && count == 8) {
        const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < count ? __ldg(p + e) : 0.f;
    }
}

// The rows a team goes through: of each of its shares (a group's rows, every `step`-th from `first` on).
struct Walk {
    int share, shares, stride, row, step, end;  // shares: groups * splits
    int splits, group_rows;
    __device__ __forceinline__ void enter() {
        const int group = share / splits;
        row = group * group_rows + share % splits;
        end = (group + 1) * group_rows;
        step = splits;
    }
    __device__ __forceinline__ bool more() const { return share < shares; }
    __device__ __forceinline__ bool last_of_share() const { return row + step >= end; }
    __device__ __forceinline__ void next() {
        if (!last_of_share()) {
            row += step;
            return;
        }
        share += stride;
        if (more()) enter();
    }
};
__device__ __forceinline__ Walk walk_of(const NormsArgs &a, int unit, int units) {
    Walk w;
    w.splits = a.splits;
    w.group_rows = a.group_rows;
    w.shares = a.rows / a.group_rows * a.splits;
    w.stride = units;
    w.share = unit;
    if (w.more()) w.enter();
    return w;
}

// One of a row's operands, eight columns at a time: out of the ring, or straight from memory.
template <class T, bool RING>
struct Operand {
    const T *base;  // at the thread's first column
    long long pitch;
    char *slot;     // its place in a stage, `slots` bytes between a thread's pieces
    int piece, run; // bytes between pieces; elements between the thread's runs
    template <int NV>
    __device__ __forceinline__ void ask(int row, int stage_at, const int (&count)[NV]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (count[v])
#pragma unroll
                for (int i = 0; i < 8 / Pack<T>::N; ++i)
                    copy16(slot + stage_at + (v * (8 / Pack<T>::N) + i) * piece, base + row * pitch + v * run + i * Pack<T>::N);
    }
    __device__ __forceinline__ void get(int row, int stage_at, int v, int count, bool wide, float (&x)[8]) const {
        if (RING) {
            constexpr int N = Pack<T>::N;
#pragma unroll
            for (int i = 0; i < 8 / N; ++i) {
                const Pack<T> q = *(const Pack<T> *)(slot + stage_at + (v * (8 / N) + i) * piece);
#pragma unroll
                for (int e = 0; e < N; ++e) x[i * N + e] = count ? widen(q.v[e]) : 0.f;
            }
        } else {
            load8(base + row * pitch + v * run, count, wide, x);
        }
    }
};
template <class T>
__host__ __device__ constexpr int pieces(int nv) { return nv * 8 * (int)sizeof(T) / 16; }

struct Place {
    int column, run;  // of the thread's first run; elements between its runs
    Team team;
    int unit, units;
};
__device__ __forceinline__ Place place_of(const NormsArgs &a, float *slots) {
    Place p;
    const int t = (int)threadIdx.x % a.team, index = (int)threadIdx.x / a.team, warps = a.team / 32;
    p.column = 8 * t;
    p.run = 8 * a.team;
    p.team = Team{index, t & 31, t >> 5, warps, a.team, slots + index * 2 * warps * 4, 0};
    p.unit = (int)blockIdx.x * a.teams + index;
    p.units = (int)gridDim.x * a.teams;
    return p;
}
constexpr int kSlotFloats = 2 * 4 * (kMaxThreads / 32);

// RING: rows come through shared memory (8 | dim, 16-byte boundaries).  Otherwise they are read where they are used, as vectors if `wide`.
template <class TX, class T, int NV, bool RING>
__global__ void __launch_bounds__(kMaxThreads) block_norms_kernel(const NormsArgs a, const bool wide, const bool wide_weights) {
    extern __shared__ __align__(16) char ring[];
    __shared__ float slots[kSlotFloats];
    grid_dependency_sync();
    Place at = place_of(a, slots);
    Team &team = at.team;
    int count[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) count[v] = max(0, min(8, a.dim - at.column - v * at.run));
    const bool branch = a.y.p != nullptr;
    const int stage_bytes = (int)blockDim.x * 16 * (pieces<TX>(NV) + (branch ? pieces<T>(NV) : 0)), piece = (int)blockDim.x * 16;
    const Operand<TX, RING> x{(const TX *)a.x.p + at.column, a.x.pitch, ring + threadIdx.x * 16, piece, at.run};
    const Operand<T, RING> y{(const T *)a.y.p + at.column, a.y.pitch, ring + threadIdx.x * 16 + pieces<TX>(NV) * piece, piece, at.run};
    const Key key = key_of(a.d);
    const float per = 1.f / (float)a.dim;
    Walk now = walk_of(a, at.unit, at.units), ahead = now;
    constexpr int kAhead = 3;  // rows asked for before the present one's are waited for
    int put = 0, take = 0;
    auto ask = [&]() {
        if (ahead.more()) {
            x.ask(ahead.row, put, count);
            if (branch) y.ask(ahead.row, put, count);
            put = put + stage_bytes == (kAhead + 1) * stage_bytes ? 0 : put + stage_bytes;
            ahead.next();
        }
        copies_end();
    };
    if (RING)
        for (int i = 0; i < kAhead; ++i) ask();
    while (now.more()) {
        const int row = now.row;
        if (RING) {
            ask();
            copies_wait<kAhead>();
        }
        float r[NV][8];
        float mean_a = 0.f, rstd_a = 1.f, mean_b = 0.f, rstd_b = 1.f;
        if (branch) {
#pragma unroll
            for (int v = 0; v < NV; ++v) y.get(row, take, v, count[v], wide, r[v]);
            if (a.after == SAGE_NORM_LAYER) {
                float s[1] = {0.f};
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[0] += r[v][e];
                team.sum(s);
                mean_a = s[0] * per;
            }
            if (a.after != SAGE_NORM_NONE) {
                float s[1] = {0.f};
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float c = e < count[v] ? r[v][e] - mean_a : 0.f;
                        s[0] = fmaf(c, c, s[0]);
                    }
                team.sum(s);
                rstd_a = rsqrtf(fmaf(s[0], per, a.eps));
            }
        }
        const float *gate = a.gate ? a.gate + row / a.group_rows * a.gate_pitch : nullptr;
        float total[1] = {0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = at.column + v * at.run;
            float xs[8];
            x.get(row, take, v, count[v], wide, xs);
            if (branch) {
                float w[8], b[8], g[8];
                weights8(a.wa ? a.wa + col : nullptr, count[v], wide_weights, 1.f, w);
                weights8(a.ba ? a.ba + col : nullptr, count[v], wide_weights, 0.f, b);
                weights8(gate ? gate + col : nullptr, count[v], wide_weights, 1.f, g);
                const unsigned keep = count[v] ? keep_from(a.d, key, (unsigned long long)row * a.dim + col) : 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float n = fmaf((r[v][e] - mean_a) * rstd_a, w[e], b[e]);
                    r[v][e] = fmaf(xs[e], a.scale, keep >> e & 1u ? n * a.d.factor * g[e] : 0.f);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] = xs[e] * a.scale;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                r[v][e] = e < count[v] ? widen(narrowed<TX>(r[v][e])) : 0.f;  // what the next reader of `out` sees: the gradient starts from that too
                total[0] += r[v][e];
            }
            if (a.out.p && count[v]) store8((TX *)a.out.p + row * a.out.pitch + col, count[v], wide, r[v]);
        }
        if (a.before == SAGE_NORM_LAYER) {
            team.sum(total);
            mean_b = total[0] * per;
        }
        if (a.before != SAGE_NORM_NONE) {
            float s[1] = {0.f};
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = e < count[v] ? r[v][e] - mean_b : 0.f;
                    s[0] = fmaf(c, c, s[0]);
                }
            team.sum(s);
            rstd_b = rsqrtf(fmaf(s[0], per, a.eps));
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!count[v]) continue;
                const int col = at.column + v * at.run;
                float w[8], b[8];
                weights8(a.wb ? a.wb + col : nullptr, count[v], wide_weights, 1.f, w);
                weights8(a.bb ? a.bb + col : nullptr, count[v], wide_weights, 0.f, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] = fmaf((r[v][e] - mean_b) * rstd_b, w[e], b[e]);
                store8((T *)a.h.p + row * a.h.pitch + col, count[v], wide, r[v]);
            }
        }
        if (a.stats && (threadIdx.x % a.team) < 4) {
            const int i = (int)threadIdx.x % a.team;
            a.stats[row * a.stats_pitch + i] = i == 0 ? mean_a : i == 1 ? rstd_a : i == 2 ? mean_b : rstd_b;
        }
        if (RING) take = take + stage_bytes == (kAhead + 1) * stage_bytes ? 0 : take + stage_bytes;
        now.next();
    }
}

template <class TX, class T, int NV, bool RING>
__global__ void __launch_bounds__(kMaxThreads) block_norms_grad_kernel(const NormsArgs a, const bool wide, const bool wide_weights) {
    extern __shared__ __align__(16) char ring[];
    __shared__ float slots[kSlotFloats];
    grid_dependency_sync();
    Place at = place_of(a, slots);
    Team &team = at.team;
    int count[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) count[v] = max(0, min(8, a.dim - at.column - v * at.run));
    const bool branch = a.y.p != nullptr, second = a.gh.p != nullptr, carried = a.go.p != nullptr;
    const int piece = (int)blockDim.x * 16;
    char *place = ring + threadIdx.x * 16;
    const Operand<TX, RING> r{(const TX *)a.out.p + at.column, a.out.pitch, place, piece, at.run};
    place += second ? pieces<TX>(NV) * piece : 0;
    const Operand<T, RING> gh{(const T *)a.gh.p + at.column, a.gh.pitch, place, piece, at.run};
    place += second ? pieces<T>(NV) * piece : 0;
    const Operand<TX, RING> go{(const TX *)a.go.p + at.column, a.go.pitch, place, piece, at.run};
    place += carried ? pieces<TX>(NV) * piece : 0;
    const Operand<T, RING> y{(const T *)a.y.p + at.column, a.y.pitch, place, piece, at.run};
    place += branch ? pieces<T>(NV) * piece : 0;
    const int stage_bytes = (int)(place - ring - threadIdx.x * 16);
    const Key key = key_of(a.d);
    const float per = 1.f / (float)a.dim;
    float sum[kSums][NV][8];
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[s][v][e] = 0.f;
    Walk now = walk_of(a, at.unit, at.units), ahead = now;
    const int ring_bytes = a.stages * stage_bytes;
    int put = 0, take = 0;
    auto ask = [&]() {
        if (ahead.more()) {
            if (second) {
                r.ask(ahead.row, put, count);
                gh.ask(ahead.row, put, count);
            }
            if (carried) go.ask(ahead.row, put, count);
            if (branch) y.ask(ahead.row, put, count);
            put = put + stage_bytes == ring_bytes ? 0 : put + stage_bytes;
            ahead.next();
        }
        copies_end();
    };
    if (RING)
        for (int i = 1; i < a.stages; ++i) ask();
    while (now.more()) {
        const int row = now.row;
        if (RING) {
            ask();
            if (a.stages == 4) copies_wait<3>();
            else if (a.stages == 2) copies_wait<1>();
            else copies_wait<0>();
        }
        const float *st = a.stats + row * a.stats_pitch;
        const float mean_a = __ldg(st), rstd_a = __ldg(st + 1), mean_b = __ldg(st + 2), rstd_b = __ldg(st + 3);
        float s1[2] = {0.f, 0.f};
        if (second) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float u[8], g[8], w[8];
                r.get(row, take, v, count[v], wide, u);
                gh.get(row, take, v, count[v], wide, g);
                weights8(a.wb ? a.wb + at.column + v * at.run : nullptr, count[v], wide_weights, 1.f, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float n = (u[e] - mean_b) * rstd_b, q = g[e] * w[e];  // (g is zero behind the row's end)
                    sum[kSumWb][v][e] = fmaf(g[e], n, sum[kSumWb][v][e]);
                    sum[kSumBb][v][e] += g[e];
                    s1[0] = fmaf(q, n, s1[0]);
                    s1[1] += q;
                }
            }
            if (a.before != SAGE_NORM_NONE) team.sum(s1);
        }
        const float along_u = s1[0] * per, mean_q = a.before == SAGE_NORM_LAYER ? s1[1] * per : 0.f;
        const float *gate = a.gate ? a.gate + row / a.group_rows * a.gate_pitch : nullptr;
        float q[NV][8], s2[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = at.column + v * at.run;
            float G[8];
            if (carried) {
                go.get(row, take, v, count[v], wide, G);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) G[e] = 0.f;
            }
            if (second) {
                float u[8], g[8], w[8];
                r.get(row, take, v, count[v], wide, u);
                gh.get(row, take, v, count[v], wide, g);
                weights8(a.wb ? a.wb + col : nullptr, count[v], wide_weights, 1.f, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) G[e] = fmaf(rstd_b, fmaf(g[e], w[e], -mean_q) - (u[e] - mean_b) * rstd_b * along_u, G[e]);
            }
            if (a.dx.p && count[v]) {
                float d[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = G[e] * a.scale;
                store8((TX *)a.dx.p + row * a.dx.pitch + col, count[v], wide, d);
            }
            if (!branch) continue;
            float w[8], b[8], gt[8], ys[8];
            y.get(row, take, v, count[v], wide, ys);
            weights8(a.wa ? a.wa + col : nullptr, count[v], wide_weights, 1.f, w);
            weights8(a.ba ? a.ba + col : nullptr, count[v], wide_weights, 0.f, b);
            weights8(gate ? gate + col : nullptr, count[v], wide_weights, 1.f, gt);
            const unsigned keep = count[v] ? keep_from(a.d, key, (unsigned long long)row * a.dim + col) : 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float n = (ys[e] - mean_a) * rstd_a;
                const float kept = keep >> e & 1u && e < count[v] ? G[e] * a.d.factor : 0.f;
                sum[kSumGate][v][e] += keep >> e & 1u ? kept * fmaf(n, w[e], b[e]) : 0.f;
                const float t = kept * gt[e];
                sum[kSumBa][v][e] += t;
                sum[kSumWa][v][e] = fmaf(t, n, sum[kSumWa][v][e]);
                q[v][e] = t * w[e];
                s2[0] = fmaf(q[v][e], n, s2[0]);
                s2[1] += q[v][e];
            }
        }
        if (branch && a.dy.p) {
            if (a.after != SAGE_NORM_NONE) team.sum(s2);
            const float along_v = s2[0] * per, mean_t = a.after == SAGE_NORM_LAYER ? s2[1] * per : 0.f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!count[v]) continue;
                if (a.after != SAGE_NORM_NONE) {
                    float ys[8];
                    y.get(row, take, v, count[v], wide, ys);
#pragma unroll
                    for (int e = 0; e < 8; ++e) q[v][e] = rstd_a * (q[v][e] - mean_t - (ys[e] - mean_a) * rstd_a * along_v);
                }
                store8((T *)a.dy.p + row * a.dy.pitch + at.column + v * at.run, count[v], wide, q[v]);
            }
        }
        if (a.gate_partial && now.last_of_share()) {
            float *to = a.gate_partial + (long long)now.share * a.dim;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                store8(to + at.column + v * at.run, count[v], wide, sum[kSumGate][v]);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[kSumGate][v][e] = 0.f;
            }
        }
        if (RING) take = take + stage_bytes == ring_bytes ? 0 : take + stage_bytes;
        now.next();
    }
    if (!a.partial) return;
    copies_wait<0>();
    // The teams' sums, team by team, through the ring's memory (a wish at a time: dim floats)
    float *shared = (float *)ring;
#pragma unroll
    for (int s = 0; s < kSums; ++s) {
        if (!(a.sums >> s & 1)) continue;
        for (int t = 0; t < a.teams; ++t) {
            __syncthreads();
            if (t != team.index) continue;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < count[v]) {
                        const int col = at.column + v * at.run + e;
                        const float all = t ? shared[col] + sum[s][v][e] : sum[s][v][e];
                        if (t + 1 == a.teams) a.partial[((long long)blockIdx.x * kSums + s) * a.dim + col] = all;
                        else shared[col] = all;
                    }
        }
    }
}

// y[j] = the sum over i of x[i * pitch + j], in a fixed order: eight runs of i, then their sums.
struct Join {
    const float *x[kSums];
    float *y[kSums];
    int count[kSums];       // addends
    long long pitch[kSums];
    int dim;
};
constexpr int kJoinParts = 16;
__global__ void __launch_bounds__(32 * kJoinParts) block_norms_join_kernel(const Join a) {
    __shared__ float part[kJoinParts][33];
    grid_dependency_sync();
    const int s = (int)blockIdx.y, lane = (int)threadIdx.x & 31, w = (int)threadIdx.x >> 5, col = (int)blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (col < a.dim) {
        const float *x = a.x[s] + col;
#pragma unroll 4
        for (int i = w; i < a.count[s]; i += kJoinParts) sum += x[i * a.pitch[s]];
    }
    part[w][lane] = sum;
    __syncthreads();
    if (w || col >= a.dim) return;
#pragma unroll
    for (int i = 1; i < kJoinParts; ++i) sum += part[i][lane];
    a.y[s][col] = sum;
}
// Gates of several groups: y[g, j] = the sum over `splits` rows of x.
__global__ void __launch_bounds__(256) block_norms_gates_kernel(const float *x, float *y, int splits, int dim, long long total, long long pitch) {
    grid_dependency_sync();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long g = i / dim, col = i - g * dim;
        float sum = 0.f;
#pragma unroll 4
        for (int s = 0; s < splits; ++s) sum += x[(g * splits + s) * dim + col];
        y[g * pitch + col] = sum;
    }
}

bool boundary(const Rows &r, long long size) { return (uintptr_t)r.p % 16 == 0 && r.pitch * size % 16 == 0; }
bool boundary(const float *p) { return (uintptr_t)p % 16 == 0; }

Rows of(const RowsArg &r) { return Rows{r.ptr, r.rows > 1 ? r.pitch : r.cols}; }

// Threads of a row, and how many rows a CTA works on at a time.
int shape_of(NormsArgs *a) {
    const int runs = (a->dim + 7) / 8;
    const int nv = runs <= kMaxThreads ? 1 : runs <= 2 * kMaxThreads ? 2 : 4;
    a->team = ((runs + nv - 1) / nv + 31) / 32 * 32;
    a->teams = std::min(kMaxThreads / a->team, kMaxTeams);
    return nv;
}

NormsArgs args_of(const BlockNorms &n, long long rows, long long dim) {
    NormsArgs a{};
    a.wa = n.after_weight;
    a.ba = n.after_bias;
    a.wb = n.before_weight;
    a.bb = n.before_bias;
    a.gate = n.gate.ptr ? (const float *)n.gate.ptr : nullptr;
    const long long groups = n.gate.ptr ? n.gate.rows : 1;
    a.gate_pitch = n.gate.pitch;
    a.after = n.after;
    a.before = n.before;
    a.eps = n.eps;
    a.scale = n.scale;
    a.d = n.drop;
    a.rows = (int)rows;
    a.dim = (int)dim;
    a.group_rows = (int)(rows / groups);
    return a;
}

bool weights_wide(const NormsArgs &a) {
    return a.dim % 4 == 0 && boundary(a.wa) && boundary(a.ba) && boundary(a.wb) && boundary(a.bb) && boundary(a.gate) && (!a.gate || a.rows == a.group_rows || a.gate_pitch % 4 == 0);
}

template <class F>
sage_status with_types(int x, int t, F f) {
    return with_type(t, [&](auto b) {
        typedef decltype(b) T;
        return x == t ? f(T(), T()) : f(float(), T());
    });
}

}  // namespace

sage_status block_norms(Context &ctx, const BlockNorms &n, const RowsArg &x, const RowsArg &y, const RowsArg &out, const RowsArg &h, const RowsArg &stats) {
    if (!x.rows) return SAGE_OK;
    NormsArgs a = args_of(n, x.rows, x.cols);
    a.x = of(x);
    a.y = of(y);
    a.out = of(out);
    a.h = of(h);
    a.stats = (float *)stats.ptr;
    a.stats_pitch = stats.rows > 1 ? stats.pitch : 4;
    const int t = y.ptr ? y.dtype : h.ptr ? h.dtype : x.dtype, sx = x.dtype == SAGE_F32 ? 4 : 2, st = t == SAGE_F32 ? 4 : 2;
    const int nv = shape_of(&a), threads = a.team * a.teams;
    const bool wide = a.dim % 8 == 0 && boundary(a.x, sx) && boundary(a.out, sx) && boundary(a.y, st) && boundary(a.h, st);
    const size_t smem = (size_t)threads * nv * 8 * (sx + (y.ptr ? st : 0)) * 4;
    const bool ring = wide && nv <= 2 && smem <= 200 * 1024;
    const int units = (a.rows + a.teams - 1) / a.teams, grid = std::min(units, ctx.sm_count * (ring && smem > 100 * 1024 ? 1 : 2));
    a.splits = std::max(1, std::min(a.group_rows, grid * a.teams / (a.rows / a.group_rows)));
    ctx.note_launch("block_norms");
    if (ctx.dry()) return SAGE_OK;
    return with_types(x.dtype, t, [&](auto tx, auto tt) {
        typedef decltype(tx) TX;
        typedef decltype(tt) T;
        const auto run = [&](auto kernel, size_t bytes) {
            if (bytes) {
                sage_status s = ctx.check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024), "block_norms");
                if (s) return s;
            }
            return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), bytes, a, wide, weights_wide(a)), "block_norms");
        };
        if (ring) return nv == 1 ? run(block_norms_kernel<TX, T, 1, true>, smem) : run(block_norms_kernel<TX, T, 2, true>, smem);
        return nv == 1 ? run(block_norms_kernel<TX, T, 1, false>, 0) : nv == 2 ? run(block_norms_kernel<TX, T, 2, false>, 0) : run(block_norms_kernel<TX, T, 4, false>, 0);
    });
}

sage_status block_norms_grad(Context &ctx, const BlockNorms &n, const RowsArg &out, const RowsArg &y, const RowsArg &stats, const RowsArg &g_out, const RowsArg &g_h, const RowsArg &dx,
                             const RowsArg &dy, const BlockNormsSums &sums) {
    const long long rows = stats.rows, dim = n.dim;
    float *const to[kSums] = {sums.before_weight, sums.before_bias, sums.after_weight, sums.after_bias, (float *)sums.gate.ptr};
    const long long groups = n.gate.ptr ? n.gate.rows : 1;
    if (!rows) {  // sums of nothing
        for (int s = 0; s < kSums; ++s) {
            if (!to[s] || (s == kSumGate && !groups)) continue;
            ctx.note_memset();
            if (ctx.dry()) continue;
            const long long pitch = s == kSumGate && groups > 1 ? sums.gate.pitch : dim;
            sage_status st = ctx.check_cuda(cudaMemset2DAsync(to[s], (size_t)pitch * 4, 0, (size_t)dim * 4, (size_t)(s == kSumGate ? groups : 1), ctx.stream()), "block_norms_grad");
            if (st) return st;
        }
        return SAGE_OK;
    }
    NormsArgs a = args_of(n, rows, dim);
    a.out = of(out);
    a.y = of(y);
    a.go = of(g_out);
    a.gh = of(g_h);
    a.dx = of(dx);
    a.dy = of(dy);
    a.stats = (float *)stats.ptr;
    a.stats_pitch = rows > 1 ? stats.pitch : 4;
    const int tx = n.x_dtype, t = n.dtype, sx = tx == SAGE_F32 ? 4 : 2, st = t == SAGE_F32 ? 4 : 2;
    const int nv = shape_of(&a), threads = a.team * a.teams;
    const bool wide = a.dim % 8 == 0 && boundary(a.out, sx) && boundary(a.go, sx) && boundary(a.dx, sx) && boundary(a.y, st) && boundary(a.gh, st) && boundary(a.dy, st);
    const size_t stage = (size_t)threads * nv * 8 * ((a.gh.p ? sx + st : 0) + (a.go.p ? sx : 0) + (a.y.p ? st : 0));
    a.stages = stage * 4 <= 200 * 1024 ? 4 : stage * 2 <= 200 * 1024 ? 2 : 1;
    const bool ring = wide && nv <= 2 && stage * a.stages <= 200 * 1024 && stage;
    const int grid = std::min((a.rows + a.teams - 1) / a.teams, ctx.sm_count);
    a.splits = std::max(1, std::min(a.group_rows, grid * a.teams / (a.rows / a.group_rows)));
    const bool by_group = a.gate && groups > 1 && to[kSumGate];
    int partials = 0;
    Join join{};
    for (int s = 0; s < kSums; ++s)
        if (to[s] && !(s == kSumGate && by_group)) {
            a.sums |= 1 << s;
            join.y[partials++] = to[s];
        }
    const size_t partial_bytes = partials ? (size_t)grid * kSums * dim * 4 : 0, gate_bytes = by_group ? (size_t)(groups * a.splits) * dim * 4 : 0, first = (partial_bytes + 255) / 256 * 256;
    Block *scratch = nullptr;
    if (partial_bytes + gate_bytes) {
        scratch = ctx.allocator().alloc(first + gate_bytes);
        if (!scratch) return ctx.fail(SAGE_ERR_OOM, "block_norms_grad: out of memory");
    }
    a.partial = partials ? (float *)scratch->ptr : nullptr;
    a.gate_partial = by_group ? (float *)(scratch->ptr + first) : nullptr;
    join.dim = a.dim;
    for (int s = 0, i = 0; s < kSums; ++s)
        if (a.sums >> s & 1) {
            join.x[i] = a.partial + (long long)s * dim;
            join.count[i] = grid;
            join.pitch[i++] = (long long)kSums * dim;
        }
    ctx.note_launch("block_norms_grad");
    if (partials) ctx.note_launch("block_norms_join");
    if (by_group) ctx.note_launch("block_norms_gates");
    sage_status status = SAGE_OK;
    if (!ctx.dry()) {
        const size_t smem = std::max(ring ? stage * a.stages : 0, partials && a.teams > 1 ? (size_t)dim * 4 : 0);
        status = with_types(tx, t, [&](auto txv, auto tv) {
            typedef decltype(txv) TX;
            typedef decltype(tv) T;
            const auto run = [&](auto kernel) {
                sage_status s = ctx.check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024), "block_norms_grad");
                if (s) return s;
                return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), smem, a, wide, weights_wide(a)), "block_norms_grad");
            };
            if (ring) return nv == 1 ? run(block_norms_grad_kernel<TX, T, 1, true>) : run(block_norms_grad_kernel<TX, T, 2, true>);
            return nv == 1 ? run(block_norms_grad_kernel<TX, T, 1, false>) : nv == 2 ? run(block_norms_grad_kernel<TX, T, 2, false>) : run(block_norms_grad_kernel<TX, T, 4, false>);
        });
        if (!status && partials)
            status = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), block_norms_join_kernel, dim3((unsigned)((dim + 31) / 32), (unsigned)partials), dim3(32 * kJoinParts), 0, join), "block_norms_join");
        if (!status && by_group) {
            const long long total = groups * dim;
            status = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), block_norms_gates_kernel, dim3((unsigned)std::min((total + 255) / 256, (long long)ctx.sm_count * 8)), dim3(256), 0,
                                                     (const float *)a.gate_partial, (float *)sums.gate.ptr, a.splits, a.dim, total, sums.gate.pitch),
                                    "block_norms_gates");
        }
    }
    if (scratch) ctx.allocator().free(scratch);
    return status;
}

}  // namespace k
}  // namespace sage
