// The norms before and after a block of a model, with what joins the block to the residual stream, row by row:
//   n = A(y)              A, B: none, x / sqrt(mean(x^2) + eps) or (x - mean x) / sqrt(mean((x - mean x)^2) + eps), then a weight and a bias
//   out = c x + gate * dropout(n)
//   h = B(out)            (of `out` as it is stored)
// Bound by memory: each operand is read and each result written once (block_norms.h says how).  16384 x 4096, stream f32, blocks bf16: 135-144 us, 5.6-6.0 TB/s;
// 4096 x 768 f32 with dropout 12.3 us, 4.1 TB/s, a launch and one round of rows.
#include "block_norms.h"

namespace sage {
namespace k {
namespace norms {
namespace {

constexpr int kRegisters = 80;  // of a thread of the general form
__host__ __device__ constexpr int wide_registers(int nv) { return nv <= 2 ? 64 : nv == 3 ? 72 : 96; }

// Whole runs of eight columns on 32-byte (16 bits: 16-byte) boundaries: a team takes one row, all of whose columns are asked for before anything waits.  Teams enough for
// the memory's latency are there at once, and the weights stay in L1 (with rows brought through rings in shared memory by teams that stay,
// 16384 x 4096 took 232 us: what is left of L1 then does not hold the weights).
__device__ __forceinline__ void prefetch_row(const char *p, int bytes) { asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory"); }

template <class TX, class T, int NV>
__global__ void __maxnreg__(wide_registers(NV)) block_norms_wide_kernel(const NormsArgs a, const int ahead) {
    __shared__ __align__(16) float2 slots[kSlots];
    Place at = place_of(a, slots);
    grid_dependency_sync();
    Team &team = at.team;
    const int col = at.column, run = at.run, row = at.unit;
    if (row >= a.rows) return;  // (the whole team)
    const bool last = col + (NV - 1) * run < a.dim, branch = a.y.p != nullptr;
    Eight<TX> xs[NV];
    Eight<T> ys[NV];
    const char *from_y = at_row<T>(a.y, row, col), *from_x = at_row<TX>(a.x, row, col);
    if (branch)
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v + 1 < NV || last) ys[v].load(from_y + v * run * (int)sizeof(T));
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (v + 1 < NV || last) xs[v].load(from_x + v * run * (int)sizeof(TX));
    if (!col && row < a.rows - ahead) {  // the rows of the CTAs that come when these have gone, into L2
        prefetch_row(at_row<TX>(a.x, row + ahead, 0), a.dim * (int)sizeof(TX));
        if (branch) prefetch_row(at_row<T>(a.y, row + ahead, 0), a.dim * (int)sizeof(T));
    }
    const Key key = key_of(a.d);
    const float per = 1.f / (float)a.dim;
    float2 r[NV][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[NV - 1][i] = make_float2(0.f, 0.f);
    // mean and 1 / deviation of the row in r, as the norm takes them (columns that are not there hold zeros)
    const auto moments = [&](int kind, float *mean, float *rstd) {
        if (kind == SAGE_NORM_NONE) return;
        if (kind == SAGE_NORM_LAYER) {
            float2 t = r[0][0];
#pragma unroll
            for (int i = 1; i < 4 * NV; ++i) t = add2(t, r[i / 4][i % 4]);
            *mean = team.sum(t.x + t.y) * per;
        }
        float2 t = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v + 1 < NV || last)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 c = add2(r[v][i], both(-*mean));
                    t = fma2(c, c, t);
                }
        *rstd = rsqrtf(fmaf(team.sum(t.x + t.y), per, a.eps));
    };
    const auto normed = [&](float2 (&c)[4], float mean, float rstd, const float *w, const float *b, int at_col) {
        float2 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = mul2(add2(c[i], both(-mean)), both(rstd));
        if (w) {
            get8(w + at_col, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = mul2(c[i], f[i]);
        }
        if (b) {
            get8(b + at_col, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = add2(c[i], f[i]);
        }
    };
    float mean_a = 0.f, rstd_a = 1.f, mean_b = 0.f, rstd_b = 1.f;
    if (branch) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v + 1 < NV || last) ys[v].open(r[v]);
        moments(a.after, &mean_a, &rstd_a);
    }
    const float *gate = a.gate;
    if (gate && a.group_rows < a.rows) gate += row / a.group_rows * a.gate_pitch;
    char *out = a.out.p ? at_row<TX>(a.out, row, col) : nullptr;
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (v + 1 < NV || last) {
            const int at_col = col + v * run;
            float2 x[4];
            xs[v].open(x);
            if (branch) {
                if (a.after != SAGE_NORM_NONE) normed(r[v], mean_a, rstd_a, a.wa, a.ba, at_col);
                if (gate) {
                    float2 g[4];
                    get8(gate + at_col, g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[v][i] = mul2(r[v][i], g[i]);
                }
                if (a.d.bar) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[v][i] = mul2(r[v][i], both(a.d.factor));
                    drop8(r[v], philox(key, ((unsigned long long)(unsigned)row * (unsigned)a.dim + at_col) >> 3, a.d.site), a.d.bar);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) r[v][i] = fma2(x[i], both(a.scale), r[v][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) r[v][i] = mul2(x[i], both(a.scale));
            }
            xs[v].close(r[v]);
            if (out) xs[v].store(out + v * run * (int)sizeof(TX));
            if (sizeof(TX) == 2) xs[v].open(r[v]);  // what the next reader of `out` sees: the gradient starts from that too
        }
    moments(a.before, &mean_b, &rstd_b);
    if (a.before != SAGE_NORM_NONE) {
        char *h = at_row<T>(a.h, row, col);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v + 1 < NV || last) {
                normed(r[v], mean_b, rstd_b, a.wb, a.bb, col + v * run);
                put8<T>(h + v * run * (int)sizeof(T), r[v]);
            }
    }
    if (a.stats && col < 32) {
        const int i = col / 8;
        a.stats[row * a.stats_pitch + i] = i == 0 ? mean_a : i == 1 ? rstd_a : i == 2 ? mean_b : rstd_b;
    }
}

// Any layout: rows are read where they are used, as vectors if `wide`.
template <class TX, class T, int NV>
__global__ void __maxnreg__(kRegisters) block_norms_kernel(const NormsArgs a, const bool wide, const bool wide_weights) {
    __shared__ __align__(16) float2 slots[kSlots];
    Place at = place_of(a, slots);
    grid_dependency_sync();
    Team &team = at.team;
    int count[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) count[v] = max(0, min(8, a.dim - at.column - v * at.run));
    const bool branch = a.y.p != nullptr;
    const Operand<TX> x{(const TX *)a.x.p + at.column, a.x.pitch, at.run};
    const Operand<T> y{(const T *)a.y.p + at.column, a.y.pitch, at.run};
    const Key key = key_of(a.d);
    const float per = 1.f / (float)a.dim;
    // mean and 1 / deviation of the row in r, as the norm takes them
    float2 r[NV][4];
    auto moments = [&](int kind, float *mean, float *rstd) {
        if (kind == SAGE_NORM_NONE) return;
        if (kind == SAGE_NORM_LAYER) {
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) t = add2(t, r[v][i]);
            *mean = team.sum(t.x + t.y) * per;
        }
        float2 t = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (!count[v]) continue;
            float2 c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = add2(r[v][i], both(-*mean));
            only(c, count[v]);
#pragma unroll
            for (int i = 0; i < 4; ++i) t = fma2(c[i], c[i], t);
        }
        *rstd = rsqrtf(fmaf(team.sum(t.x + t.y), per, a.eps));
    };
    // (r - mean) * rstd, times the weight, plus the bias
    auto normed = [&](float2 (&c)[4], float mean, float rstd, const float *w, const float *b, int col, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = mul2(add2(c[i], both(-mean)), both(rstd));
        float2 f[4];
        if (w) {
            weights8(w + col, n, wide_weights, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = mul2(c[i], f[i]);
        }
        if (b) {
            weights8(b + col, n, wide_weights, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = add2(c[i], f[i]);
        }
    };
    for (int row = at.unit; row < a.rows; row += at.units) {
        float mean_a = 0.f, rstd_a = 1.f, mean_b = 0.f, rstd_b = 1.f;
        if (branch) {
#pragma unroll
            for (int v = 0; v < NV; ++v) y.get(row, v, count[v], wide, r[v]);
            moments(a.after, &mean_a, &rstd_a);
        }
        const float *gate = a.gate ? a.gate + row / a.group_rows * a.gate_pitch : nullptr;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (!count[v]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) r[v][i] = make_float2(0.f, 0.f);
                continue;
            }
            const int col = at.column + v * at.run;
            float2 xs[4];
            x.get(row, v, count[v], wide, xs);
            if (branch) {
                if (a.after != SAGE_NORM_NONE) normed(r[v], mean_a, rstd_a, a.wa, a.ba, col, count[v]);
                if (gate) {
                    float2 g[4];
                    weights8(gate + col, count[v], wide_weights, g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[v][i] = mul2(r[v][i], g[i]);
                }
                if (a.d.bar) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[v][i] = mul2(r[v][i], both(a.d.factor));
                    only_kept(r[v], kept(a.d, key, row, a.dim, col));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) r[v][i] = fma2(xs[i], both(a.scale), r[v][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) r[v][i] = mul2(xs[i], both(a.scale));
            }
            if (a.out.p) store8((TX *)a.out.p + row * a.out.pitch + col, count[v], wide, r[v]);
            if (sizeof(TX) == 2) {  // what the next reader of `out` sees: the gradient starts from that too
                Eight<TX> q;
                q.close(r[v]);
                q.open(r[v]);
            }
            only(r[v], count[v]);
        }
        moments(a.before, &mean_b, &rstd_b);
        if (a.before != SAGE_NORM_NONE) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!count[v]) continue;
                const int col = at.column + v * at.run;
                normed(r[v], mean_b, rstd_b, a.wb, a.bb, col, count[v]);
                store8((T *)a.h.p + row * a.h.pitch + col, count[v], wide, r[v]);
            }
        }
        if (a.stats && at.column < 32) {
            const int i = at.column / 8;
            a.stats[row * a.stats_pitch + i] = i == 0 ? mean_a : i == 1 ? rstd_a : i == 2 ? mean_b : rstd_b;
        }
    }
}

}  // namespace
}  // namespace norms

sage_status block_norms(Context &ctx, const BlockNorms &n, const RowsArg &x, const RowsArg &y, const RowsArg &out, const RowsArg &h, const RowsArg &stats) {
    using namespace norms;
    if (!x.rows) return SAGE_OK;
    NormsArgs a = args_of(n, x.rows, x.cols);
    a.x = of(x);
    a.y = of(y);
    a.out = of(out);
    a.h = of(h);
    a.stats = (float *)stats.ptr;
    a.stats_pitch = stats.rows > 1 ? stats.pitch : 4;
    const int t = y.ptr ? y.dtype : h.ptr ? h.dtype : x.dtype, sx = x.dtype == SAGE_F32 ? 4 : 2, st = t == SAGE_F32 ? 4 : 2;
    const int nv = shape_of(&a, 1, 4);
    const bool wide = a.dim % 8 == 0 && boundary(a.x, sx) && boundary(a.out, sx) && boundary(a.y, st) && boundary(a.h, st);
    const bool vectors = wide && weights_wide(a);
    size_t none;
    a.teams = std::max(1, std::min(128 / a.team, kMaxTeams));
    const int grid = vectors ? (a.rows + a.teams - 1) / a.teams : grid_of(ctx, &a, nv, 0, kRegisters, false, &none), threads = a.team * a.teams;  // (grid_of sets the teams)
    const int ahead = ctx.sm_count * (65536 / (wide_registers(nv) * threads)) * a.teams;  // rows that are worked on at once
    ctx.note_launch("block_norms");
    if (ctx.dry()) return SAGE_OK;
    return with_types(x.dtype, t, [&](auto tx, auto tt) {
        typedef decltype(tx) TX;
        typedef decltype(tt) T;
        const auto by_vectors = [&](auto kernel) { return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), 0, a, ahead), "block_norms"); };
        const auto any = [&](auto kernel) { return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3((unsigned)grid), dim3((unsigned)threads), 0, a, wide, weights_wide(a)), "block_norms"); };
        if (vectors)
            return nv == 1 ? by_vectors(block_norms_wide_kernel<TX, T, 1>) : nv == 2 ? by_vectors(block_norms_wide_kernel<TX, T, 2>) : nv == 3 ? by_vectors(block_norms_wide_kernel<TX, T, 3>) : by_vectors(block_norms_wide_kernel<TX, T, 4>);
        return nv == 1 ? any(block_norms_kernel<TX, T, 1>) : nv == 2 ? any(block_norms_kernel<TX, T, 2>) : nv == 3 ? any(block_norms_kernel<TX, T, 3>) : any(block_norms_kernel<TX, T, 4>);
    });
}

}  // namespace k
}  // namespace sage
