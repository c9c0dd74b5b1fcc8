// What the norms around a block (block_norms.cu) and their gradient (block_norms_grad.cu) have in common: teams of threads that go through rows.
//
// A thread owns NV runs of eight neighbouring columns and a team of threads a row, so that the sums over rows stay in registers, a sum over a row is
// one shuffle tree and, in teams of several warps, one exchange in shared memory, and a block of dropout's mask is one draw.  Forward, a team takes one
// row; in the gradient teams go through rows in steps of their number, and what a thread reads of its team's next rows is copied into places of its own in
// shared memory while the present row is worked on (no barrier: only the thread that asked reads them).  Arithmetic is on pairs of columns, two f32
// operations an instruction.
#pragma once
#include <algorithm>

#include "counter_random.h"
#include "eight.h"
#include "language.h"
#include "launch.h"

namespace sage {
namespace k {
namespace norms {

constexpr int kMaxThreads = 512, kMaxTeams = 15;  // of a CTA; named barriers 1 to 15
constexpr int kRingBytes = 216 * 1024;            // of an SM's shared memory, for rows on their way

struct Rows {
    void *p;
    long long pitch;
    unsigned bytes;  // of a pitch, where that is less than 4 GB
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
    int stages;            // of the ring: a row worked on, the others on their way
    int splits;            // of a group's rows
    float *partial;        // backward: [CTA][sum][dim]
    float *gate_partial;   // ... and for gates of several groups [group * splits + split][dim]
    int sums;              // bits: which of kSums are wanted
};
enum { kSumWb, kSumBb, kSumWa, kSumBa, kSumGate, kSums };

__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the `stages - 1` youngest groups have arrived (two stages or four).
__device__ __forceinline__ void copies_wait(int stages) {
    if (stages == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// Sums over a team, two at a time, the same bits in all of its threads.
struct Team {
    int index, lane, warp, warps, threads;
    float2 *slots;  // [2][16], zero where there are no warps
    int turn;
    __device__ __forceinline__ void open() {
        if (warps == 1) return;
        if (!warp) slots[lane] = make_float2(0.f, 0.f);
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(threads) : "memory");
    }
    __device__ __forceinline__ float2 sum(float2 v) {
#pragma unroll
        for (int off = 16; off; off >>= 1) v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, off), __shfl_xor_sync(0xffffffffu, v.y, off)));
        if (warps == 1) return v;
        if (!lane) slots[turn + warp] = v;
        return met();
    }
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (warps == 1) return v;
        if (!lane) slots[turn + warp].x = v;
        return met().x;
    }
    __device__ __forceinline__ float2 met() {
        const float4 *q = (const float4 *)(slots + turn);
        turn ^= 16;  // (the next sum but one writes here again, behind the next one's barrier)
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(threads) : "memory");
        const auto eight = [&](int at) {
            const float4 a = q[at], b = q[at + 1], c = q[at + 2], d = q[at + 3];
            return add2(add2(add2(make_float2(a.x, a.y), make_float2(a.z, a.w)), add2(make_float2(b.x, b.y), make_float2(b.z, b.w))),
                        add2(add2(make_float2(c.x, c.y), make_float2(c.z, c.w)), add2(make_float2(d.x, d.y), make_float2(d.z, d.w))));
        };
        float2 t = eight(0);
        if (warps > 8) t = add2(t, eight(4));
        return t;
    }
};
constexpr int kSlots = 32 * kMaxTeams;

template <class T>
__device__ __forceinline__ void load8(const T *p, int count, bool wide, float2 (&v)[4]) {
    Eight<T> q;
    if (wide && count == 8) {
#pragma unroll
        for (int i = 0; i < Eight<T>::kPacks; ++i) q.p[i] = ((const Pack<T> *)p)[i];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) q.p[e / Pack<T>::N].v[e % Pack<T>::N] = e < count ? p[e] : narrowed<T>(0.f);
    }
    q.open(v);
}
template <class T>
__device__ __forceinline__ void store8(T *p, int count, bool wide, const float2 (&v)[4]) {
    Eight<T> q;
    q.close(v);
    if (wide && count == 8) {
#pragma unroll
        for (int i = 0; i < Eight<T>::kPacks; ++i) ((Pack<T> *)p)[i] = q.p[i];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) p[e] = q.p[e / Pack<T>::N].v[e % Pack<T>::N];
    }
}
// Weights, biases and gates: f32, through L1.  There is one.
__device__ __forceinline__ void weights8(const float *p, int count, bool wide, float2 (&v)[4]) {
    if (wide && count == 8) {
        const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
        v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_float2(2 * i < count ? __ldg(p + 2 * i) : 0.f, 2 * i + 1 < count ? __ldg(p + 2 * i + 1) : 0.f);
    }
}
// Columns behind the row's end hold nothing.
__device__ __forceinline__ void only(float2 (&v)[4], int count) {
    if (count == 8) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(2 * i < count ? v[i].x : 0.f, 2 * i + 1 < count ? v[i].y : 0.f);
}
__device__ __forceinline__ void only_kept(float2 (&v)[4], unsigned keep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(keep >> (2 * i) & 1u ? v[i].x : 0.f, keep >> (2 * i + 1) & 1u ? v[i].y : 0.f);
}

// The rows a team goes through: of each of its shares (a group's rows, every `splits`-th from the share's first on).
struct Walk {
    int share, shares, stride, row, end, group;  // shares: groups * splits
    int splits, group_rows;
    __device__ __forceinline__ void enter() {
        group = share / splits;
        row = group * group_rows + share % splits;
        end = (group + 1) * group_rows;
    }
    __device__ __forceinline__ bool more() const { return share < shares; }
    __device__ __forceinline__ bool last_of_share() const { return end - row <= splits; }
    __device__ __forceinline__ void next() {
        if (!last_of_share()) {
            row += splits;
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
    w.row = w.end = w.group = 0;
    if (w.more()) w.enter();
    return w;
}

template <class T>
__host__ __device__ constexpr int pieces(int nv) { return nv * 8 * (int)sizeof(T) / 16; }

// One of a row's operands, eight columns at a time.
template <class T>
struct Operand {
    const T *base;  // at the thread's first column
    long long pitch;
    int run;        // elements between its runs
    __device__ __forceinline__ void get(int row, int v, int count, bool wide, float2 (&x)[4]) const { load8(base + row * pitch + v * run, count, wide, x); }
};

struct Place {
    int column, run;  // of the thread's first run; elements between its runs
    Team team;
    int unit, units;
};
__device__ __forceinline__ Place place_of(const NormsArgs &a, float2 *slots) {
    Place p;
    const int index = (int)threadIdx.x / a.team, t = (int)threadIdx.x - index * a.team;
    p.column = 8 * t;
    p.run = 8 * a.team;
    p.team = Team{index, t & 31, t >> 5, a.team / 32, a.team, slots + index * 32, 0};
    p.team.open();
    p.unit = (int)blockIdx.x * a.teams + index;
    p.units = (int)gridDim.x * a.teams;
    return p;
}
// Which of a thread's eight columns of a row stay.
__device__ __forceinline__ unsigned kept(const Dropout &d, Key key, int row, int dim, int col) { return keep_from(d, key, (unsigned long long)row * dim + col); }

// ---- rows that come through shared memory: 8 | dim, rows on 32-byte (16 bits: 16-byte) boundaries, less than 4 GB apart.  All but a thread's last run of columns are
// there; `last` says whether that one is.  Addresses are made from the kernel's parameters where they are used: held in registers they
// took more of them than the sums over rows do.
template <class T>
__device__ __forceinline__ char *at_row(const Rows &r, int row, int col) {
    return (char *)r.p + ((unsigned long long)(unsigned)row * r.bytes + (unsigned)(col * (int)sizeof(T)));
}
template <class T>
__device__ __forceinline__ void ring_ask(const char *from, unsigned to, unsigned piece) {
#pragma unroll
    for (int i = 0; i < Eight<T>::kPacks; ++i) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * piece), "l"(from + i * 16) : "memory");
}
template <class T>
__device__ __forceinline__ void ring_get(unsigned from, int v, unsigned piece, float2 (&x)[4]) {
    Eight<T> q;
#pragma unroll
    for (int i = 0; i < Eight<T>::kPacks; ++i) {
        uint4 u;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(from + (v * Eight<T>::kPacks + i) * piece) : "memory");
        *(uint4 *)&q.p[i] = u;
    }
    q.open(x);
}
template <class T>
__device__ __forceinline__ void put8(char *to, const float2 (&v)[4]) {
    Eight<T> q;
    q.close(v);
    q.store(to);
}
__device__ __forceinline__ void get8(const float *p, float2 (&v)[4]) {  // weights, biases, gates
    const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
    v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
}
// Eight elements of a row in one access (f32: 32 bytes).
inline bool boundary(const Rows &r, long long size) { return (uintptr_t)r.p % (8 * size) == 0 && r.pitch % 8 == 0 && r.pitch * size < 0x100000000ll; }
inline bool boundary(const float *p) { return (uintptr_t)p % 16 == 0; }
inline Rows of(const RowsArg &r) {
    const long long pitch = r.rows > 1 ? r.pitch : r.cols;
    return Rows{r.ptr, pitch, (unsigned)(pitch * (r.dtype == SAGE_F32 ? 4 : 2))};
}

// Threads of a row: of the numbers of runs a thread may own, the one that leaves the fewest without columns, and of those the largest, since what a row
// costs each thread is shared by its columns.
inline int shape_of(NormsArgs *a, int least, int most) {
    const int runs = (a->dim + 7) / 8;
    int slots = 0;
    for (int n = least; n <= most; ++n) {
        const int team = std::max(32, ((runs + n - 1) / n + 31) / 32 * 32), taken = team * ((runs + team - 1) / team);
        if (team > kMaxThreads || (slots && taken > slots)) continue;
        slots = taken;
        a->team = team;
    }
    return (runs + a->team - 1) / a->team;  // all of a thread's runs but the last are whole
}
// How many teams a CTA has and how many CTAs there are, and how deep the ring: `operand_bytes` of what a column reads, `registers` of a thread.  As many
// teams at once as an SM's registers hold (each quarter of it has 16384), in few CTAs, which leave few sums behind.
inline int grid_of(Context &ctx, NormsArgs *a, int nv, size_t operand_bytes, int registers, bool ring, size_t *smem) {
    const int team_warps = a->team / 32, warps = 16384 / (registers * 32) * 4;
    int fit = 0;
    a->teams = 1;
    for (int t = 1; t * a->team <= 1024 && t <= kMaxTeams; ++t) {
        const int ctas = warps / (t * team_warps);
        if (ctas && ctas * t >= fit * a->teams) {
            fit = ctas;
            a->teams = t;
        }
    }
    fit = std::max(1, fit);
    const size_t stage = (size_t)a->team * nv * 8 * operand_bytes;  // of a team
    a->stages = 4;
    if (ring) {
        if (stage * 4 * a->teams * fit > (size_t)kRingBytes) a->stages = 2;
        while (fit > 1 && stage * a->stages * a->teams * fit > (size_t)kRingBytes) --fit;
        while (a->teams > 1 && stage * a->stages * a->teams > (size_t)kRingBytes) --a->teams;
    }
    *smem = ring ? stage * a->stages * a->teams : 0;
    while (a->teams > 1 && (a->rows + a->teams - 1) / a->teams < ctx.sm_count) --a->teams;  // few rows: on all SMs
    const int grid = (int)std::min<long long>((a->rows + a->teams - 1) / a->teams, (long long)ctx.sm_count * fit);
    if (ring) *smem = stage * a->stages * a->teams;
    a->splits = std::max(1, std::min(a->group_rows, grid * a->teams / (a->rows / a->group_rows)));
    return grid;
}

inline NormsArgs args_of(const BlockNorms &n, long long rows, long long dim) {
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

inline bool weights_wide(const NormsArgs &a) {
    return boundary(a.wa) && boundary(a.ba) && boundary(a.wb) && boundary(a.bb) && boundary(a.gate) && (!a.gate || a.rows == a.group_rows || a.gate_pitch % 4 == 0);
}

template <class F>
sage_status with_types(int x, int t, F f) {
    return with_type(t, [&](auto b) {
        typedef decltype(b) T;
        return x == t ? f(T(), T()) : f(float(), T());
    });
}

}  // namespace norms
}  // namespace k
}  // namespace sage
