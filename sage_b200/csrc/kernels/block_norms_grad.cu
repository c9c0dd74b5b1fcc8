// The gradient of the norms around a block (block_norms.cu), for arrivals go (of out) and gh (of h), with u = the unit rows of B's operand, v of A's:
//   q = gh wb;   G = go + rstd (q - mean(q u) u [- mean q], layer norms);   dx = c G
//   K = G keep / (1 - p);   d gate = sum over rows of K n;   t = K gate;   dy from t as G - go from gh
// and the weights' and biases' gradients: sums over rows of gh u, gh, t v, t.
//
// Bound by memory, with as many operations beside it as the instruction slots hold: sums over rows take eight registers for each run of columns and kind, of
// which programs without a norm after the block and without a gate (FULL false) have two.  They are joined in a fixed order: team by team within a
// CTA, then CTA by CTA in a second launch.  16376 x 2056 bf16 with everything 132 us (3.0 TB/s, 49 % of the issue slots; with a gate's
// and a bias's sums made row by row 165); 33.5 M elements in rows of 2048, two rms
// norms 92 us, a norm before alone 83 (0.67 and 0.62 of the memory's rate by what must be read and written); 4096 x 768 f32 24 us.
#include <type_traits>

#include "block_norms.h"

namespace sage {
namespace k {
namespace norms {
namespace {

constexpr int kRegisters = 112;  // of a thread of the general form

// Gates: none; one row of them for all rows that a team goes through, which then multiplies sums instead of rows (with P = sum of K v, Q = sum of K the gate's sum
// is wa P + ba Q, the weight's gate P, the bias's gate Q); rows of their own for each group of rows.
enum { kUngated, kGateOnce, kGateEach };
// Which sums over rows a kernel keeps, and where.
template <bool FULL, int BIASES, int GATE>  // BIASES: 1 the one before, 2 both
struct Kinds {
    __host__ __device__ constexpr int at(int kind) const {
        const bool there[kSums] = {true, BIASES >= 1, FULL, FULL && BIASES == 2, FULL && GATE != kUngated};
        if (!there[kind]) return -1;
        int n = 0;
        for (int k = 0; k < kind; ++k) n += there[k] ? 1 : 0;
        return n;
    }
    __host__ __device__ constexpr int count() const {
        int n = 0;
        for (int k = 0; k < kSums; ++k) n += at(k) >= 0 ? 1 : 0;
        return n;
    }
};

// The teams' sums of a CTA, team by team, through shared memory (a kind at a time: dim floats).
template <class KINDS, int KEPT, int NV>
__device__ __forceinline__ void join_teams(const NormsArgs &a, const Place &at, float2 (&sum)[KEPT][NV][4], const int (&count)[NV], bool wide, float *shared) {
#pragma unroll
    for (int kind = 0; kind < kSums; ++kind) {
        constexpr KINDS kept{};
        if (kept.at(kind) < 0 || !(a.sums >> kind & 1)) continue;
        const int s = kept.at(kind) < 0 ? 0 : kept.at(kind);
        for (int t = 0; t < a.teams; ++t) {
            if (a.teams > 1) __syncthreads();
            if (t != at.team.index) continue;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int col = at.column + v * at.run;
                float2 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = sum[s][v][i];
                if (t && count[v]) {
                    float2 y[4];
                    load8(shared + col, count[v], wide, y);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = add2(x[i], y[i]);
                }
                store8(t + 1 == a.teams ? a.partial + ((long long)blockIdx.x * kSums + kind) * a.dim + col : shared + col, count[v], wide, x);
            }
        }
    }
}

// The gradient of an element that is dropped, told from a zero of one that stays by its sign (the draw's words, kept until they are asked again, cost 10 to 17 % of the time).
constexpr float kDropped = -0.f;
__device__ __forceinline__ bool is_dropped(float g) { return __float_as_uint(g) == 0x80000000u; }

__host__ __device__ constexpr int ring_registers(int nv, bool full) { return full ? (nv == 1 ? 96 : 128) : nv == 1 ? 80 : nv == 2 ? 96 : 128; }

// What models call: both gradients arrive, there is a norm before the next block and norms have weights; whole runs of columns on
// 32-byte (16 bits: 16-byte) boundaries.
template <class TX, class T, int NV, bool FULL, int BIASES, int GATE>
__global__ void __maxnreg__(ring_registers(NV, FULL)) block_norms_grad_ring_kernel(const NormsArgs a) {
    extern __shared__ __align__(16) char ring[];
    __shared__ __align__(16) float2 slots[kSlots];
    Place at = place_of(a, slots);
    grid_dependency_sync();
    Team &team = at.team;
    const int col = at.column, run = at.run;
    const bool last = col + (NV - 1) * run < a.dim;
    // a stage: out, gh, go and (FULL) y
    const unsigned piece = blockDim.x * 16;
    constexpr int kGh = pieces<TX>(NV), kGo = kGh + pieces<T>(NV), kY = kGo + pieces<TX>(NV), kStage = kY + (FULL ? pieces<T>(NV) : 0);
    const int wcol = last ? col + (NV - 1) * run : 0;  // of the last run's weights: threads without one work on zeros, and on any weights
    const unsigned stage = kStage * piece, ring0 = (unsigned)__cvta_generic_to_shared(ring) + threadIdx.x * 16, ring1 = ring0 + a.stages * stage;
    if (!last)
        for (int s = 0; s < a.stages; ++s) {
            const auto clear = [&](int first, int packs) {
                for (int p = first + (NV - 1) * packs; p < first + NV * packs; ++p) *(uint4 *)(ring + threadIdx.x * 16 + s * stage + p * piece) = make_uint4(0u, 0u, 0u, 0u);
            };
            clear(0, Eight<TX>::kPacks);
            clear(kGh, Eight<T>::kPacks);
            clear(kGo, Eight<TX>::kPacks);
            if (FULL) clear(kY, Eight<T>::kPacks);
        }
    __shared__ RoundKeys keys;
    if (a.d.bar) {
        round_keys(&keys, Key{__ldg(a.d.seed), __ldg(a.d.seed + a.d.seed_stride)}, (int)threadIdx.x);
        __syncthreads();
    }
    const float per = 1.f / (float)a.dim;
    const float2 zero = make_float2(0.f, 0.f);
    constexpr Kinds<FULL, BIASES, GATE> kept{};
    constexpr int kKept = kept.count(), kWb = 0, kBb = BIASES >= 1 ? kept.at(kSumBb) : 0, kWa = FULL ? kept.at(kSumWa) : 0, kBa = FULL && BIASES == 2 ? kept.at(kSumBa) : 0, kGate = FULL && GATE != kUngated ? kept.at(kSumGate) : 0;
    float2 sum[kKept][NV][4];
#pragma unroll
    for (int s = 0; s < kKept; ++s)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[s][v][i] = zero;
    const int shares = a.rows / a.group_rows * a.splits;
    for (int share = at.unit; share < shares; share += at.units) {
        const int group = share / a.splits, end = (group + 1) * a.group_rows, row0 = group * a.group_rows + share % a.splits;
        unsigned put = ring0, take = ring0;
        int ahead = row0;
        const auto ask = [&]() {
            if (ahead < end) {
                const unsigned long long x_at = (unsigned long long)(unsigned)ahead * a.out.bytes + (unsigned)(col * (int)sizeof(TX)), t_at = (unsigned long long)(unsigned)ahead * a.gh.bytes + (unsigned)(col * (int)sizeof(T));
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (v + 1 < NV || last) {
                        const unsigned x_run = (unsigned)(v * run * (int)sizeof(TX)), t_run = (unsigned)(v * run * (int)sizeof(T));
                        ring_ask<TX>((const char *)a.out.p + x_at + x_run, put + v * Eight<TX>::kPacks * piece, piece);
                        ring_ask<T>((const char *)a.gh.p + t_at + t_run, put + (kGh + v * Eight<T>::kPacks) * piece, piece);
                        ring_ask<TX>((const char *)a.go.p + x_at + x_run, put + (kGo + v * Eight<TX>::kPacks) * piece, piece);
                        if (FULL) ring_ask<T>((const char *)a.y.p + t_at + t_run, put + (kY + v * Eight<T>::kPacks) * piece, piece);
                    }
                put = put + stage == ring1 ? ring0 : put + stage;
                ahead += a.splits;
            }
            copies_end();
        };
        for (int i = 1; i < a.stages; ++i) ask();
        float next[4];
#pragma unroll
        for (int i = FULL ? 0 : 2; i < 4; ++i) next[i] = __ldg(a.stats + row0 * a.stats_pitch + i);
        for (int row = row0; row < end; row += a.splits) {
            const float mean_a = FULL ? next[0] : 0.f, rstd_a = FULL ? next[1] : 1.f, mean_b = next[2], rstd_b = next[3];
            // Unit rows are x * rstd + these: a rounding of mean / deviation more than (x - mean) * rstd, no larger than that of the mean itself, which the statistics hold in 32 bits
            // (the difference first: 16376 x 2056 132 -> 146 us, 16384 x 2048 with two rms norms 92 -> 94).
            const float from_a = -mean_a * rstd_a, from_b = -mean_b * rstd_b;
            if (end - row > a.splits)
#pragma unroll
                for (int i = FULL ? 0 : 2; i < 4; ++i) next[i] = __ldg(a.stats + (row + a.splits) * a.stats_pitch + i);
            ask();
            copies_wait(a.stages);
            const unsigned long long x_at = (unsigned long long)(unsigned)row * a.out.bytes + (unsigned)(col * (int)sizeof(TX)), t_at = (unsigned long long)(unsigned)row * a.gh.bytes + (unsigned)(col * (int)sizeof(T));
            float2 q[NV][4], along = zero, all = zero;  // what arrives through the norm
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float2 u[4], w[4];
                ring_get<TX>(take, v, piece, u);
                ring_get<T>(take + kGh * piece, v, piece, q[v]);
                get8(a.wb + (v + 1 < NV ? col + v * run : wcol), w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u[i] = fma2(u[i], both(rstd_b), both(from_b));
                    sum[kWb][v][i] = fma2(q[v][i], u[i], sum[kWb][v][i]);
                    if (BIASES >= 1) sum[kBb][v][i] = add2(sum[kBb][v][i], q[v][i]);
                    q[v][i] = mul2(q[v][i], w[i]);
                    along = fma2(q[v][i], u[i], along);
                    all = add2(all, q[v][i]);
                }
            }
            const float2 s1 = team.sum(make_float2(along.x + along.y, all.x + all.y));
            const float along_u = s1.x * per, mean_q = a.before == SAGE_NORM_LAYER ? s1.y * per : 0.f;
            float2 along_t = zero, all_t = zero;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const bool there = v + 1 < NV || last;
                const int at_col = v + 1 < NV ? col + v * run : wcol;
                const float through = there ? rstd_b : 0.f;
                float2 G[4], u[4];
                ring_get<TX>(take + kGo * piece, v, piece, G);
                ring_get<TX>(take, v, piece, u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u[i] = fma2(u[i], both(rstd_b), both(from_b));
                    G[i] = fma2(fma2(u[i], both(-along_u), add2(q[v][i], both(-mean_q))), both(through), G[i]);
                    u[i] = mul2(G[i], both(a.scale));
                }
                if (a.dx.p && there) put8<TX>((char *)a.dx.p + x_at + (unsigned)(v * run * (int)sizeof(TX)), u);
                if (a.d.bar) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) G[i] = fma2(G[i], both(a.d.factor), zero);  // (no zero of those that stay is negative)
                    drop8(G, philox(keys, ((unsigned long long)(unsigned)row * (unsigned)a.dim + at_col) >> 3, a.d.site), a.d.bar, FULL ? kDropped : 0.f);
                }
                if (!FULL) {
                    if (a.dy.p && there) put8<T>((char *)a.dy.p + t_at + (unsigned)(v * run * (int)sizeof(T)), G);
                    continue;
                }
                float2 n[4], w[4], b[4];
                ring_get<T>(take + kY * piece, v, piece, n);
                if (a.after != SAGE_NORM_NONE) {
                    get8(a.wa + at_col, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) n[i] = fma2(n[i], both(rstd_a), both(from_a));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = both(1.f);
                    if (a.d.bar)  // a value that is dropped may be anything (a norm would have spread it)
#pragma unroll
                        for (int i = 0; i < 4; ++i) n[i] = make_float2(is_dropped(G[i].x) ? 0.f : n[i].x, is_dropped(G[i].y) ? 0.f : n[i].y);
                }
                if (GATE == kGateEach) {
                    float2 by[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) by[i] = mul2(n[i], w[i]);
                    if (a.ba) {
                        get8(a.ba + at_col, b);
#pragma unroll
                        for (int i = 0; i < 4; ++i) by[i] = add2(by[i], b[i]);
                    }
                    get8(a.gate + (long long)group * a.gate_pitch + at_col, b);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[kGate][v][i] = fma2(G[i], by[i], sum[kGate][v][i]);
                        G[i] = mul2(G[i], b[i]);
                    }
                }
                if (GATE == kGateOnce) get8(a.gate + (long long)group * a.gate_pitch + at_col, b);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (BIASES == 2) sum[kBa][v][i] = add2(sum[kBa][v][i], G[i]);
                    sum[kWa][v][i] = fma2(G[i], n[i], sum[kWa][v][i]);
                    if (GATE == kGateOnce) G[i] = mul2(G[i], b[i]);
                    q[v][i] = mul2(G[i], w[i]);
                    along_t = fma2(q[v][i], n[i], along_t);
                    all_t = add2(all_t, q[v][i]);
                }
            }
            if (FULL && a.dy.p) {
                float2 s2 = zero;
                if (a.after != SAGE_NORM_NONE) s2 = team.sum(make_float2(along_t.x + along_t.y, all_t.x + all_t.y));
                const float along_v = s2.x * per, mean_t = a.after == SAGE_NORM_LAYER ? s2.y * per : 0.f;
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (v + 1 < NV || last) {
                        if (a.after != SAGE_NORM_NONE) {
                            float2 n[4];
                            ring_get<T>(take + kY * piece, v, piece, n);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                q[v][i] = mul2(fma2(fma2(n[i], both(rstd_a), both(from_a)), both(-along_v), add2(q[v][i], both(-mean_t))), both(rstd_a));
                        }
                        put8<T>((char *)a.dy.p + t_at + (unsigned)(v * run * (int)sizeof(T)), q[v]);
                    }
            }
            take = take + stage == ring1 ? ring0 : take + stage;
        }
        if (FULL && GATE == kGateOnce) {  // the team's only share
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at_col = v + 1 < NV ? col + v * run : wcol;
                float2 f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = both(1.f);
                if (a.after != SAGE_NORM_NONE) get8(a.wa + at_col, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[kGate][v][i] = mul2(sum[kWa][v][i], f[i]);
                if (BIASES == 2 && a.ba) {
                    get8(a.ba + at_col, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[kGate][v][i] = fma2(sum[kBa][v][i], f[i], sum[kGate][v][i]);
                }
                get8(a.gate + (long long)group * a.gate_pitch + at_col, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[kWa][v][i] = mul2(sum[kWa][v][i], f[i]);
                    if (BIASES == 2) sum[kBa][v][i] = mul2(sum[kBa][v][i], f[i]);
                }
            }
        }
        if (FULL && GATE != kUngated && a.gate_partial) {
            float *to = a.gate_partial + (long long)share * a.dim + col;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (v + 1 < NV || last) store8(to + v * run, 8, true, sum[kGate][v]);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[kGate][v][i] = zero;
            }
        }
    }
    if (!a.partial) return;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    int count[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) count[v] = v + 1 < NV || last ? 8 : 0;
    join_teams<Kinds<FULL, BIASES, GATE>>(a, at, sum, count, true, (float *)ring);
}

// Any layout, and operands that are absent (a model's first norm has no y, its last no g_out) or norms without weights: rows are read where they are used, as vectors if `wide`.  8192 x 4096
// bf16, two rms norms 98 us above, without g_out 278 here, without weights 284; a norm before alone without y 119.
template <class TX, class T, int NV, bool FULL>
__global__ void __maxnreg__(kRegisters) block_norms_grad_kernel(const NormsArgs a, const bool wide, const bool wide_weights) {
    extern __shared__ __align__(16) char ring[];
    __shared__ __align__(16) float2 slots[kSlots];
    Place at = place_of(a, slots);
    grid_dependency_sync();
    Team &team = at.team;
    int count[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) count[v] = max(0, min(8, a.dim - at.column - v * at.run));
    const bool branch = a.y.p != nullptr, second = a.gh.p != nullptr, carried = a.go.p != nullptr;
    const Operand<TX> r{(const TX *)a.out.p + at.column, a.out.pitch, at.run}, go{(const TX *)a.go.p + at.column, a.go.pitch, at.run};
    const Operand<T> gh{(const T *)a.gh.p + at.column, a.gh.pitch, at.run}, y{(const T *)a.y.p + at.column, a.y.pitch, at.run};
    const Key key = key_of(a.d);
    const float per = 1.f / (float)a.dim;
    const float2 zero = make_float2(0.f, 0.f);
    constexpr int kKept = FULL ? (int)kSums : 2;
    float2 sum[kKept][NV][4];
#pragma unroll
    for (int s = 0; s < kKept; ++s)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[s][v][i] = zero;
    Walk now = walk_of(a, at.unit, at.units);
    while (now.more()) {
        const int row = now.row;
        const float *st = a.stats + row * a.stats_pitch;
        const float mean_a = __ldg(st), rstd_a = __ldg(st + 1), mean_b = __ldg(st + 2), rstd_b = __ldg(st + 3);
        // (drawn here: nothing waits for it, and the sums below wait for others)
        unsigned keep[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) keep[v] = a.d.bar && count[v] ? kept(a.d, key, row, a.dim, at.column + v * at.run) : 0xffu;
        float2 s1 = zero;
        if (second) {
            float2 along = zero, all = zero;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!count[v]) continue;
                float2 u[4], g[4], w[4];
                r.get(row, v, count[v], wide, u);
                gh.get(row, v, count[v], wide, g);  // (zero behind the row's end)
                if (a.wb) weights8(a.wb + at.column + v * at.run, count[v], wide_weights, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 n = mul2(add2(u[i], both(-mean_b)), both(rstd_b)), q = a.wb ? mul2(g[i], w[i]) : g[i];
                    sum[kSumWb][v][i] = fma2(g[i], n, sum[kSumWb][v][i]);
                    sum[kSumBb][v][i] = add2(sum[kSumBb][v][i], g[i]);
                    along = fma2(q, n, along);
                    all = add2(all, q);
                }
            }
            s1 = make_float2(along.x + along.y, all.x + all.y);
            if (a.before != SAGE_NORM_NONE) s1 = team.sum(s1);
        }
        const float along_u = s1.x * per * rstd_b, mean_q = a.before == SAGE_NORM_LAYER ? s1.y * per : 0.f;
        const float *gate = FULL && a.gate ? a.gate + now.group * a.gate_pitch : nullptr;
        float2 q[NV][4], along_t = zero, all_t = zero;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (!count[v]) continue;
            const int col = at.column + v * at.run;
            float2 G[4];
            if (carried) {
                go.get(row, v, count[v], wide, G);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) G[i] = zero;
            }
            if (second) {
                float2 u[4], g[4], w[4];
                r.get(row, v, count[v], wide, u);
                gh.get(row, v, count[v], wide, g);
                if (a.wb) weights8(a.wb + col, count[v], wide_weights, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 n = mul2(add2(u[i], both(-mean_b)), both(rstd_b));
                    const float2 e = a.wb ? fma2(g[i], w[i], both(-mean_q)) : add2(g[i], both(-mean_q));
                    G[i] = add2(G[i], fma2(n, both(-along_u), mul2(e, both(rstd_b))));
                }
            }
            if (a.dx.p) {
                float2 d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = mul2(G[i], both(a.scale));
                store8((TX *)a.dx.p + row * a.dx.pitch + col, count[v], wide, d);
            }
            if (!branch) continue;
            if (a.d.bar) {
#pragma unroll
                for (int i = 0; i < 4; ++i) G[i] = mul2(G[i], both(a.d.factor));
                only_kept(G, keep[v]);
            }
            if (!FULL) {
                if (a.dy.p) store8((T *)a.dy.p + row * a.dy.pitch + col, count[v], wide, G);
                continue;
            }
            only(G, count[v]);
            float2 n[4], w[4], b[4], t[4];
            y.get(row, v, count[v], wide, n);
            if (a.wa) weights8(a.wa + col, count[v], wide_weights, w);
            if (gate) {
                if (a.ba) weights8(a.ba + col, count[v], wide_weights, b);
                weights8(gate + col, count[v], wide_weights, t);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                n[i] = mul2(add2(n[i], both(-mean_a)), both(rstd_a));
                if (gate) {
                    float2 by = a.wa ? a.ba ? fma2(n[i], w[i], b[i]) : mul2(n[i], w[i]) : a.ba ? add2(n[i], b[i]) : n[i];
                    if (a.d.bar) by = make_float2(keep[v] >> (2 * i) & 1u ? by.x : 0.f, keep[v] >> (2 * i + 1) & 1u ? by.y : 0.f);  // (a value that is dropped may be anything)
                    sum[kSumGate][v][i] = fma2(G[i], by, sum[kSumGate][v][i]);
                    t[i] = mul2(t[i], G[i]);
                } else {
                    t[i] = G[i];
                }
                sum[kSumBa][v][i] = add2(sum[kSumBa][v][i], t[i]);
                sum[kSumWa][v][i] = fma2(t[i], n[i], sum[kSumWa][v][i]);
                q[v][i] = a.wa ? mul2(t[i], w[i]) : t[i];
                along_t = fma2(q[v][i], n[i], along_t);
                all_t = add2(all_t, q[v][i]);
            }
        }
        if (FULL && branch && a.dy.p) {
            float2 s2 = make_float2(along_t.x + along_t.y, all_t.x + all_t.y);
            if (a.after != SAGE_NORM_NONE) s2 = team.sum(s2);
            const float along_v = s2.x * per * rstd_a, mean_t = a.after == SAGE_NORM_LAYER ? s2.y * per : 0.f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!count[v]) continue;
                if (a.after != SAGE_NORM_NONE) {
                    float2 n[4];
                    y.get(row, v, count[v], wide, n);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        q[v][i] = fma2(mul2(add2(n[i], both(-mean_a)), both(rstd_a)), both(-along_v), mul2(add2(q[v][i], both(-mean_t)), both(rstd_a)));
                }
                store8((T *)a.dy.p + row * a.dy.pitch + at.column + v * at.run, count[v], wide, q[v]);
            }
        }
        if (FULL && a.gate_partial && now.last_of_share()) {
            float *to = a.gate_partial + (long long)now.share * a.dim;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                store8(to + at.column + v * at.run, count[v], wide, sum[FULL ? kSumGate : 0][v]);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[FULL ? kSumGate : 0][v][i] = zero;
            }
        }
        now.next();
    }
    if (!a.partial) return;
    join_teams<Kinds<FULL, FULL ? 2 : 1, kGateEach>>(a, at, sum, count, wide, (float *)ring);
}

// The sums that CTAs, and shares of a group's rows, left: y[j] = the sum over i of x[i * pitch + j], in a fixed order: warp by warp every 32nd, then
// the warps'.  A row of blocks for each kind, and for each group of a gate.
struct Join {
    const float *x[kSums];
    float *y[kSums];
    int kinds, count;         // addends
    long long pitch;
    const float *gate_x;      // gates of several groups: `splits` addends each, dim apart
    float *gate_y;
    long long gate_pitch;
    int splits, dim;
};
constexpr int kJoinParts = 32;
__global__ void __launch_bounds__(32 * kJoinParts) block_norms_join_kernel(const __grid_constant__ Join a) {
    __shared__ float2 part[kJoinParts][32];
    grid_dependency_sync();
    const int lane = (int)threadIdx.x & 31, w = (int)threadIdx.x >> 5, col = ((int)blockIdx.x * 32 + lane) * 2, s = (int)blockIdx.y;
    const bool kind = s < a.kinds;
    const int count = kind ? a.count : a.splits;
    const long long group = s - a.kinds, pitch = kind ? a.pitch : a.dim;
    const float *x = (kind ? a.x[s] : a.gate_x + group * a.splits * a.dim) + col;
    const bool two = a.dim % 2 == 0 && col < a.dim, one = col < a.dim;  // (the partial sums lie on 256-byte boundaries)
    float2 sum = make_float2(0.f, 0.f);
    if (two) {
        const float2 *p = (const float2 *)x;
        const long long step = pitch / 2;
        int i = w;
        for (; i + 7 * kJoinParts < count; i += 8 * kJoinParts) {
            float2 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[(i + k * kJoinParts) * step];
#pragma unroll
            for (int k = 0; k < 8; ++k) sum = add2(sum, v[k]);
        }
#pragma unroll 4
        for (; i < count; i += kJoinParts) sum = add2(sum, p[i * step]);
    } else if (one) {
        for (int i = w; i < count; i += kJoinParts) sum = add2(sum, make_float2(x[i * pitch], col + 1 < a.dim ? x[i * pitch + 1] : 0.f));
    }
    part[w][lane] = sum;
    __syncthreads();
    if (w || !one) return;
#pragma unroll
    for (int k = 1; k < kJoinParts; ++k) sum = add2(sum, part[k][lane]);
    float *y = (kind ? a.y[s] : a.gate_y + group * a.gate_pitch) + col;
    y[0] = sum.x;
    if (col + 1 < a.dim) y[1] = sum.y;
}

}  // namespace
}  // namespace norms

sage_status block_norms_grad(Context &ctx, const BlockNorms &n, const RowsArg &out, const RowsArg &y, const RowsArg &stats, const RowsArg &g_out, const RowsArg &g_h, const RowsArg &dx,
                             const RowsArg &dy, const BlockNormsSums &sums) {
    using namespace norms;
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
    // Without a norm after the block or a gate its values are not read, and two kinds of sums are kept.
    const bool full = a.y.p && (a.after != SAGE_NORM_NONE || a.gate);
    // Runs of eight columns to a thread.  Two where rows are long: what a row costs each thread is then shared by twice the columns; four kinds of sums of
    // two runs fit its registers, five (gates that change on a team's way) do not.  33.5 M elements bf16, one run | two, us: five kinds, 768 columns 131 | 161, 1024 140 | 140,
    // 1536 144 | 147, 2048 156 | 152, 4096 187 | 166; four kinds 1024 128 | 120, 1536 135 | 118; two norms alone, 2048 columns 127 | 95, 4096 151 | 101; a norm before
    // alone, 4096 columns 104 | 89.
    const bool many = full && a.gate && to[kSumBb] && groups > ctx.sm_count;
    const int least = a.dim > (many ? 1536 : full ? 1024 : 2048) ? 2 : 1, most = least == 2 || (full && !many) ? 2 : 1, nv = a.dim > 8 * kMaxThreads * 2 ? shape_of(&a, 4, 4) : shape_of(&a, least, most);
    const bool wide = a.dim % 8 == 0 && boundary(a.out, sx) && boundary(a.go, sx) && boundary(a.dx, sx) && boundary(a.y, st) && boundary(a.gh, st) && boundary(a.dy, st);
    size_t smem;
    const size_t bytes = (a.gh.p ? sx + st : 0) + (a.go.p ? sx : 0) + (full ? st : 0);
    // Rows of the stream have one pitch, those of the block another.
    const auto like = [](const Rows &r, const Rows &of) { return !r.p || r.pitch == of.pitch; };
    const bool usual = a.y.p && a.gh.p && a.go.p && a.wb && like(a.go, a.out) && like(a.dx, a.out) && like(a.y, a.gh) && like(a.dy, a.gh) && (a.wa || a.after == SAGE_NORM_NONE);
    const bool ring = wide && usual && weights_wide(a) && !(full && nv > 2) && grid_of(ctx, &a, nv, bytes, ring_registers(nv, full), true, &smem) && smem <= kRingBytes;
    const int grid = grid_of(ctx, &a, nv, bytes, ring ? ring_registers(nv, full) : kRegisters, ring, &smem), threads = a.team * a.teams;
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
            join.x[i++] = a.partial + (long long)s * dim;
        }
    ctx.note_launch("block_norms_grad");
    join.kinds = partials;
    join.count = grid;
    join.pitch = (long long)kSums * dim;
    join.splits = a.splits;
    if (by_group) {
        join.gate_x = a.gate_partial;
        join.gate_y = (float *)sums.gate.ptr;
        join.gate_pitch = sums.gate.pitch;
    }
    const long long joins = partials + (by_group ? groups : 0), once = 32768;  // rows of blocks, as many as a launch may have
    for (long long at = 0; at < joins; at += once) ctx.note_launch("block_norms_join");
    sage_status status = SAGE_OK;
    if (!ctx.dry()) {
        if (partials && a.teams > 1) smem = std::max(smem, (size_t)dim * 4);
        status = with_types(tx, t, [&](auto txv, auto tv) {
            typedef decltype(txv) TX;
            typedef decltype(tv) T;
            const auto by_ring = [&](auto kernel) {
                sage_status s = ctx.check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes), "block_norms_grad");
                return s ? s : ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), smem, a), "block_norms_grad");
            };
            const auto any = [&](auto kernel) { return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), smem, a, wide, weights_wide(a)), "block_norms_grad"); };
            if (ring) {
                const auto of_full = [&](auto biases, auto gate) {
                    constexpr int B = decltype(biases)::value, G = decltype(gate)::value;
                    return nv == 1 ? by_ring(block_norms_grad_ring_kernel<TX, T, 1, true, B, G>) : by_ring(block_norms_grad_ring_kernel<TX, T, 2, true, B, G>);
                };
                const auto of_biases = [&](auto gate) {
                    const bool both = to[kSumBa] || (a.ba && decltype(gate)::value == kGateOnce);
                    return both ? of_full(std::integral_constant<int, 2>(), gate) : to[kSumBb] ? of_full(std::integral_constant<int, 1>(), gate) : of_full(std::integral_constant<int, 0>(), gate);
                };
                if (full && !a.gate) return of_biases(std::integral_constant<int, kUngated>());
                if (full) return groups * a.splits <= (long long)grid * a.teams ? of_biases(std::integral_constant<int, kGateOnce>()) : of_biases(std::integral_constant<int, kGateEach>());
                return nv == 1 ? by_ring(block_norms_grad_ring_kernel<TX, T, 1, false, 1, kUngated>) : nv == 2 ? by_ring(block_norms_grad_ring_kernel<TX, T, 2, false, 1, kUngated>) : by_ring(block_norms_grad_ring_kernel<TX, T, 4, false, 1, kUngated>);
            }
            if (full) return nv == 1 ? any(block_norms_grad_kernel<TX, T, 1, true>) : nv == 2 ? any(block_norms_grad_kernel<TX, T, 2, true>) : any(block_norms_grad_kernel<TX, T, 4, true>);
            return nv == 1   ? any(block_norms_grad_kernel<TX, T, 1, false>)
                   : nv == 2 ? any(block_norms_grad_kernel<TX, T, 2, false>)
                             : any(block_norms_grad_kernel<TX, T, 4, false>);
        });
        for (long long at = 0; at < joins && !status; at += once) {
            status = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), block_norms_join_kernel, dim3((unsigned)((dim + 63) / 64), (unsigned)std::min(once, joins - at)), dim3(32 * kJoinParts), 0, join), "block_norms_join");
            const long long done = std::min(once, joins - at) - join.kinds;  // groups
            join.kinds = 0;
            if (join.gate_x) {
                join.gate_x += done * a.splits * dim;
                join.gate_y += done * join.gate_pitch;
            }
        }
    }
    if (scratch) ctx.allocator().free(scratch);
    return status;
}

}  // namespace k
}  // namespace sage
