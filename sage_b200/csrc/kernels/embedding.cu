// Token embedding: y[t, :] = scale * table[ids[t], :], and its gradient by table rows.
#include <cuda_runtime.h>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

// ------------------------------------------------------------------------------------------ lookup
// A thread moves V elements at a time (16 bytes of the table, or one element where rows do not lie on 16-byte boundaries), four of
// them in flight.  Bound by memory: the tokens' rows read, the results written.
constexpr int kLookups = 4;
template <class T, class Y, int V>
__global__ void __launch_bounds__(256) embedding_kernel(const T *__restrict__ table, long long vocab, long long ld, const int *__restrict__ ids, long long ids_stride, float scale, Y *__restrict__ y,
                                                        long long ldy, long long tokens, unsigned per_row) {
    grid_dependency_sync();
    // Units of V elements, `per_row` to a row, are numbered through; the block's first in 64 bits, the others from there in 32.
    const unsigned long long first = (unsigned long long)blockIdx.x * (256 * kLookups);
    const unsigned long long row0 = first / per_row;
    const unsigned rest = (unsigned)(first - row0 * per_row) + threadIdx.x;
    Pack<T> v[kLookups];
    long long at[kLookups];
    bool some[kLookups];
#pragma unroll
    for (int u = 0; u < kLookups; ++u) {
        const unsigned unit = rest + u * 256, rows = unit / per_row, c = (unit - rows * per_row) * V;
        const long long t = (long long)row0 + rows;
        at[u] = -1;
        some[u] = false;
        if (t < tokens) {
            const int id = ids[t * ids_stride];
            some[u] = id >= 0 && id < vocab;
            at[u] = t * ldy + c;
            if (some[u]) {
                const T *p = table + id * ld + c;
                if (V > 1) v[u] = *reinterpret_cast<const Pack<T> *>(p);
                else v[u].v[0] = *p;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kLookups; ++u) {
        if (at[u] < 0) continue;
        if constexpr (V == 1) {
            y[at[u]] = narrowed<Y>(some[u] ? widen(v[u].v[0]) * scale : 0.f);
        } else {
            constexpr int P = V / Pack<Y>::N;  // a narrow table's row into f32 takes two stores
#pragma unroll
            for (int p = 0; p < P; ++p) {
                Pack<Y> o;
#pragma unroll
                for (int j = 0; j < Pack<Y>::N; ++j) o.v[j] = narrowed<Y>(some[u] ? widen(v[u].v[p * Pack<Y>::N + j]) * scale : 0.f);
                *reinterpret_cast<Pack<Y> *>(y + at[u] + p * Pack<Y>::N) = o;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ gradient
// Tokens are sorted by table row (those of a row in their order), then rows are summed in pieces of a fixed length of that order, so
// that a frequent token's thousands of rows are spread like any others.  Two launches, no sums by atomics: the same bits every time.

// Sorting.  Each of 2^bits blocks owns the table rows whose numbers end in its own (frequent tokens have low numbers: neighbours go to
// different blocks) and reads all ids: its warps, each over a contiguous share of the tokens, count its rows' tokens, the counts become
// places (in front of them all tokens of the blocks before), and a second pass puts the tokens there.  A hundred times the ids out of L2
// instead of a radix sort's passes through memory and launches.
constexpr int kSortWarps = 32, kSortRows = 1536;  // rows of a block at most: their counts fill shared memory
__global__ void __launch_bounds__(kSortWarps * 32) embedding_sort_kernel(const int *__restrict__ ids, long long ids_stride, int tokens, int vocab, int bits, int2 *__restrict__ spans, int *__restrict__ total,
                                                                         int *__restrict__ order, int *__restrict__ sorted, unsigned *__restrict__ arrived, int counters) {
    extern __shared__ int places[];  // [warp][row of the block]
    __shared__ int warp_sums[kSortWarps], below_all;
    constexpr int U = 8;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const unsigned own = blockIdx.x, ending = (1u << bits) - 1;
    const int rows = (int)(((unsigned)vocab - own + ending) >> bits);
    for (int i = threadIdx.x; i < kSortWarps * rows; i += kSortWarps * 32) places[i] = 0;
    grid_dependency_sync();
    for (int i = blockIdx.x * (kSortWarps * 32) + threadIdx.x; i < counters; i += gridDim.x * (kSortWarps * 32)) arrived[i] = 0;
    __syncthreads();
    const int share = ((tokens + kSortWarps - 1) / kSortWarps + 31) / 32 * 32, begin = (int)min((long long)warp * share, (long long)tokens), end = (int)min(begin + (long long)share, (long long)tokens);
    int *mine = places + warp * rows, below = 0;
    for (int t0 = begin; t0 < end; t0 += 32 * U) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = t0 + u * 32 + lane < end ? ids[(t0 + u * 32 + lane) * ids_stride] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool some = (unsigned)id[u] < (unsigned)vocab;
            below += some && (id[u] & ending) < own;
            if (some && (id[u] & ending) == own) atomicAdd(mine + (id[u] >> bits), 1);  // a count: any order
        }
    }
    for (int o = 16; o; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
    if (lane == 0) warp_sums[warp] = below;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) below_all = s;
    }
    __syncthreads();
    int next = below_all;  // place of the next row's first token
    for (int r0 = 0; r0 < rows; r0 += kSortWarps * 32) {
        const int r = r0 + threadIdx.x;
        int count = 0;
        if (r < rows)
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) count += places[w * rows + r];
        int sum = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += left;
        }
        if (lane == 31) warp_sums[warp] = sum;
        __syncthreads();
        int ahead = lane < warp ? warp_sums[lane] : 0, all = warp_sums[lane];
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        int at = next + ahead + sum - count;
        next += all;
        if (r < rows) {
            spans[((long long)r << bits) + own] = make_int2(at, at + count);
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = places[w * rows + r];
                places[w * rows + r] = at;
                at += c;
            }
        }
        __syncthreads();
    }
    if (own == ending && threadIdx.x == 0) *total = next;
    for (int t0 = begin; t0 < end; t0 += 32 * U) {
        int id[U], from[U];
        unsigned same[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = t0 + u * 32 + lane < end ? ids[(t0 + u * 32 + lane) * ids_stride] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = (unsigned)id[u] < (unsigned)vocab && (id[u] & ending) == own;
            const unsigned all = __ballot_sync(0xffffffffu, in);
            same[u] = 0;
            __syncwarp();  // places of u - 1 are taken
            if (in) {
                same[u] = __match_any_sync(all, id[u]);
                if (lane == __ffs(same[u]) - 1) from[u] = atomicAdd(mine + (id[u] >> bits), __popc(same[u]));  // one lane for each row: in the order of u
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = __shfl_sync(0xffffffffu, from[u], same[u] ? __ffs(same[u]) - 1 : lane);
            if (same[u]) {
                const int place = at + __popc(same[u] & ((1u << lane) - 1));
                order[place] = t0 + u * 32 + lane;
                sorted[place] = id[u];
            }
        }
    }
}

// Summing.  A block takes 256 tokens of the sorted order, 32 to a warp, and 32 lanes' columns; the rows of g that end in a warp's 32 go
// straight to the table, the others are joined over the warps in shared memory, and what goes on beyond the block's 256 is left in
// `partial` (slot 2 c: of a row that began before block c, 2 c + 1: of one that goes on behind it); the last block of such a row to
// arrive adds the pieces up, in their order.  Further blocks write the rows that no token reaches.
// Bound by memory: g once, the table once.
constexpr int kSumWarps = 8, kSumTokens = 32 * kSumWarps, kZeroRows = 64;
struct EmbeddingGrad {
    const void *g;
    long long ldg;
    float *dtable;
    long long ld;
    int dim, vocab, slices, chunks, add;
    float scale;
    const int2 *spans;  // a row's places in the order
    const int *total, *order, *sorted;
    float *partial;
    unsigned *arrived;
};

template <class T, bool WIDE>
struct Columns {  // a lane's columns of a slice: N in a row, or N that lie 32 apart
    static constexpr int N = 16 / (int)sizeof(T);
    int first, dim;
    __device__ Columns(int slice, int dim_) : first(slice * 32 * N + (threadIdx.x % 32) * (WIDE ? N : 1)), dim(dim_) {}
    __device__ __forceinline__ int column(int j) const { return first + (WIDE ? j : 32 * j); }
    __device__ __forceinline__ bool has(int j) const { return column(j) < dim; }
    __device__ __forceinline__ Pack<T> load(const T *row) const {
        Pack<T> v;
        if (WIDE) {
            if (first < dim) v = *reinterpret_cast<const Pack<T> *>(row + first);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (has(j)) v.v[j] = row[column(j)];
        }
        return v;
    }
};

template <class T, bool WIDE>
__global__ void __launch_bounds__(kSumTokens) embedding_grad_kernel(const __grid_constant__ EmbeddingGrad a) {
    typedef Columns<T, WIDE> C;
    constexpr int N = C::N, U = 8;
    __shared__ float head[kSumWarps][32 * N], tail[kSumWarps][32 * N];
    __shared__ int head_row[kSumWarps], tail_row[kSumWarps], head_ends[kSumWarps];  // rows: -1 = none
    __shared__ int spans[2], last[2];  // rows that go on beyond the block (-1 = none): began before it, or in it
    grid_dependency_sync();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if ((int)blockIdx.x >= a.chunks * a.slices) {  // rows without a token
        const long long v0 = (long long)(blockIdx.x - a.chunks * a.slices) * kZeroRows, v1 = min(v0 + kZeroRows, (long long)a.vocab);
        const long long first = v0 + warp * (kZeroRows / kSumWarps);  // the warp's rows, looked up at once
        int2 span = make_int2(0, 1);
        if (lane < kZeroRows / kSumWarps && first + lane < v1) span = a.spans[first + lane];
        for (unsigned todo = __ballot_sync(0xffffffffu, span.x == span.y); todo; todo &= todo - 1) {
            float *row = a.dtable + (first + __ffs(todo) - 1) * a.ld;
            if (WIDE)
                for (int c = lane * 4; c < a.dim; c += 128) *reinterpret_cast<float4 *>(row + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            else
                for (int c = lane; c < a.dim; c += 32) row[c] = 0.f;
        }
        return;
    }
    const int chunk = blockIdx.x / a.slices, slice = blockIdx.x - chunk * a.slices, total = *a.total;
    if (chunk * kSumTokens >= total) return;
    const C cols(slice, a.dim);
    auto output = [&](int v, const float (&x)[N]) {
        float *row = a.dtable + v * a.ld;
        if (WIDE) {
            if (cols.first >= a.dim) return;
#pragma unroll
            for (int q = 0; q < N; q += 4) {
                const float4 o = make_float4(x[q] * a.scale, x[q + 1] * a.scale, x[q + 2] * a.scale, x[q + 3] * a.scale);
                // One addition to each element in all, made in L2: reading the row first would stop the warp at the end of every row.
                if (a.add) asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(row + cols.first + q), "f"(o.x), "f"(o.y), "f"(o.z), "f"(o.w) : "memory");
                else *reinterpret_cast<float4 *>(row + cols.first + q) = o;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (cols.has(j)) {
                    if (a.add) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(row + cols.column(j)), "f"(x[j] * a.scale) : "memory");
                    else row[cols.column(j)] = x[j] * a.scale;
                }
        }
    };
    auto keep = [&](float *to, const float (&x)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) to[j * 32 + lane] = x[j];
    };

    // the warp's 32 places
    const int from = chunk * kSumTokens + warp * 32, n = min(32, total - from);
    int first_row = -1, tail_kept = -1, ends = 0;
    if (n > 0) {
        const int row = lane < n ? a.sorted[from + lane] : -1, token = lane < n ? a.order[from + lane] : 0;
        const int before = from > 0 ? a.sorted[from - 1] : -1, after = from + n < total ? a.sorted[from + n] : -1;
        const int left = __shfl_up_sync(0xffffffffu, row, 1);
        const unsigned starts = __ballot_sync(0xffffffffu, lane < n && row != (lane ? left : before));
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.f;
        bool began_before = !(starts & 1);
        for (int i0 = 0; i0 < n; i0 += U) {
            Pack<T> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = __shfl_sync(0xffffffffu, token, (i0 + u) & 31);
                if (i0 + u < n) v[u] = cols.load((const T *)a.g + t * a.ldg);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i >= n) break;
                if (i && starts >> i & 1) {  // the row so far is complete
                    const int done = __shfl_sync(0xffffffffu, row, i - 1);
                    if (began_before) {
                        first_row = done;
                        ends = 1;
                        keep(head[warp], sum);
                    } else {
                        output(done, sum);
                    }
                    began_before = false;
#pragma unroll
                    for (int j = 0; j < N; ++j) sum[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] += widen(v[u].v[j]);
            }
        }
        const int done = __shfl_sync(0xffffffffu, row, n - 1);
        if (began_before) {
            first_row = done;
            ends = done != after;
            keep(head[warp], sum);
        } else if (done == after) {
            tail_kept = done;
            keep(tail[warp], sum);
        } else {
            output(done, sum);
        }
    }
    if (lane == 0) {
        head_row[warp] = first_row;
        head_ends[warp] = ends;
        tail_row[warp] = tail_kept;
    }
    __syncthreads();

    // over the warps
    const long long stride = (long long)a.slices * 32 * N;  // of the partial sums, padded to whole slices
    float *partial = a.partial + slice * 32 * N + lane;
    if (warp == 0) {
        float sum[N];
        int open = -1, spans_before = -1, spans_after = -1;
        bool began_before = false;
        auto leave = [&](int slot) {
#pragma unroll
            for (int j = 0; j < N; ++j) __stcg(partial + slot * stride + j * 32, sum[j]);
        };
        for (int w = 0; w < kSumWarps; ++w) {
            if (head_row[w] >= 0) {
                if (w == 0) began_before = true;
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] = (w ? sum[j] : 0.f) + head[w][j * 32 + lane];
                open = head_row[w];
                if (head_ends[w]) {
                    if (began_before) {
                        spans_before = open;
                        leave(2 * chunk);
                    } else {
                        output(open, sum);
                    }
                    open = -1;
                    began_before = false;
                }
            }
            if (tail_row[w] >= 0) {
                open = tail_row[w];
                began_before = false;
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] = tail[w][j * 32 + lane];
            }
        }
        if (open >= 0) {
            leave(2 * chunk + (began_before ? 0 : 1));
            (began_before ? spans_before : spans_after) = open;
        }
        __threadfence();
        __syncwarp();
        if (lane == 0) {
            spans[0] = spans_before;
            spans[1] = spans_after;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                last[k] = 0;
                if (spans[k] < 0) continue;
                const int2 at = a.spans[spans[k]];
                const int c0 = at.x / kSumTokens, c1 = (at.y - 1) / kSumTokens;
                last[k] = atomicAdd(a.arrived + (long long)c0 * a.slices + slice, 1u) == (unsigned)(c1 - c0);
            }
            __threadfence();
        }
    }
    __syncthreads();
    for (int k = 0; k < 2; ++k) {
        if (!last[k]) continue;  // the same for the whole block
        const int v = spans[k], c0 = a.spans[v].x / kSumTokens, pieces = (a.spans[v].y - 1) / kSumTokens - c0 + 1;
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.f;
        const int p1 = (int)((long long)pieces * (warp + 1) / kSumWarps);
#pragma unroll 4
        for (int p = (int)((long long)pieces * warp / kSumWarps); p < p1; ++p) {
            const float *from_piece = partial + (2 * (long long)(c0 + p) + (p == 0)) * stride;
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += __ldcg(from_piece + j * 32);
        }
        keep(head[warp], sum);
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < kSumWarps; ++w)
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] += head[w][j * 32 + lane];
            output(v, sum);
        }
        __syncthreads();
    }
}

}  // namespace

bool on_16(const void *p, long long pitch, size_t size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch * (long long)size % 16 == 0; }

sage_status embedding(Context &ctx, const RowsArg &table, const VectorArg &ids, float scale, const RowsArg &y) {
    if (!y.rows || !y.cols) return SAGE_OK;
    ctx.note_launch("embedding");
    if (ctx.dry()) return SAGE_OK;
    return with_type(table.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_type(y.dtype, [&](auto o) {
            typedef decltype(o) Y;
            if constexpr (sizeof(Y) < sizeof(T)) return ctx.fail(SAGE_ERR_INVALID, "embedding: y is narrower than the table");
            else {
                constexpr int V = 16 / (int)sizeof(T);
                const bool wide = y.cols % V == 0 && on_16(table.ptr, table.pitch, sizeof(T)) && on_16(y.ptr, y.pitch, sizeof(Y));
                const unsigned per_row = (unsigned)(wide ? y.cols / V : y.cols);
                const long long each = 256 * kLookups;
                long long most = (0x7fffffffll * each) / per_row;  // rows of one launch
                for (long long at = 0; at < y.rows; at += most) {
                    const long long rows = y.rows - at < most ? y.rows - at : most;
                    const dim3 grid((unsigned)((rows * per_row + each - 1) / each));
                    sage_status st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? embedding_kernel<T, Y, V> : embedding_kernel<T, Y, 1>, grid, dim3(256), 0, (const T *)table.ptr, table.rows,
                                                                     table.pitch, (const int *)ids.ptr + at * ids.stride, ids.stride, scale, (Y *)y.ptr + at * y.pitch, y.pitch, rows, per_row),
                                                    "embedding");
                    if (st) return st;
                }
                return (sage_status)SAGE_OK;
            }
        });
    });
}

sage_status embedding_grad(Context &ctx, const RowsArg &g, const VectorArg &ids, float scale, bool add, const RowsArg &dtable) {
    const long long vocab = dtable.rows, dim = dtable.cols, tokens = g.rows;
    if (!vocab || !dim || (add && !tokens)) return SAGE_OK;
    const long long n = g.dtype == SAGE_F32 ? 4 : 8, slices = (dim + 32 * n - 1) / (32 * n), chunks = (tokens + kSumTokens - 1) / kSumTokens;
    const long long zero_blocks = add ? 0 : (vocab + kZeroRows - 1) / kZeroRows;
    if (chunks * slices + zero_blocks > 0x7fffffffll || chunks * kSumTokens > 0x7fff0000ll) return ctx.fail(SAGE_ERR_INVALID, "embedding_grad: too many rows");
    const auto rounded = [](long long words) { return (words + 63) / 64 * 64; };
    const long long starts = rounded(2 * vocab + 1), places = rounded(tokens), counters = rounded(chunks * slices);
    Block *scratch = ctx.allocator().alloc((size_t)(starts + 2 * places + counters + 2 * chunks * slices * 32 * n) * 4);
    if (!scratch) return ctx.fail(SAGE_ERR_OOM, "embedding_grad: out of memory");
    EmbeddingGrad a;
    int *words = (int *)scratch->ptr;
    a.spans = (const int2 *)words;
    a.total = words + 2 * vocab;
    a.order = words + starts;
    a.sorted = a.order + places;
    a.arrived = (unsigned *)(words + starts + 2 * places);
    a.partial = (float *)(a.arrived + counters);
    a.g = g.ptr;
    a.ldg = g.pitch;
    a.dtable = (float *)dtable.ptr;
    a.ld = dtable.pitch;
    a.dim = (int)dim;
    a.vocab = (int)vocab;
    a.slices = (int)slices;
    a.chunks = (int)chunks;
    a.add = add;
    a.scale = scale;
    const bool wide = dim % n == 0 && on_16(g.ptr, g.pitch, 16 / n) && on_16(dtable.ptr, dtable.pitch, 4);
    int bits = 0;  // about one block for each SM; more where shared memory does not hold the counts of that many rows
    while ((2ll << bits) <= vocab && ((2 << bits) <= ctx.sm_count || ((vocab - 1) >> bits) + 1 > kSortRows)) ++bits;
    const size_t smem = (size_t)(((vocab - 1) >> bits) + 1) * kSortWarps * 4;
    sage_status st = SAGE_OK;
    ctx.note_launch("embedding_sort");
    ctx.note_launch("embedding_grad");
    if (!ctx.dry()) {
        st = ctx.check_cuda(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortRows * kSortWarps * 4), "embedding_sort");
        if (!st)
            st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), embedding_sort_kernel, dim3(1u << bits), dim3(kSortWarps * 32), smem, (const int *)ids.ptr, ids.stride,
                                                 (int)tokens, (int)vocab, bits, (int2 *)a.spans, (int *)a.total, (int *)a.order, (int *)a.sorted, a.arrived, (int)counters),
                                "embedding_sort");
        if (!st)
            st = with_type(g.dtype, [&](auto t) {
                typedef decltype(t) T;
                return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? embedding_grad_kernel<T, true> : embedding_grad_kernel<T, false>, dim3((unsigned)(chunks * slices + zero_blocks)),
                                                       dim3(kSumTokens), 0, a),
                                      "embedding_grad");
            });
    }
    ctx.allocator().free(scratch);
    return st;
}

}  // namespace k
}  // namespace sage
