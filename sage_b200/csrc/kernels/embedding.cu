// Token embedding: y[t, :] = scale * table[ids[t], :], and its gradient by table rows.
#include <cuda_runtime.h>

#include <algorithm>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

// ------------------------------------------------------------------------------------------ lookup
// A thread moves V elements at a time (16 bytes of the table, or one element where rows do not lie on 16-byte boundaries), four of
// them in flight.  Bound by memory: the tokens' rows read, the results written (32768 x 4096 bf16: 91 us, 5.9 TB/s; 8 x 768: 4.0, a launch).
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
// Tokens are sorted by table row (those of a row in a fixed order), then rows are summed in pieces of a fixed length of that order, so
// that a frequent token's thousands of rows are spread like any others.  Two or three launches, no sums by atomics: the same bits every time.

constexpr int kZeroRows = 8;  // of a block that writes zeros: about one to a warp (94 MB with 64 rows a block 30 us, with 6 to 12 18 us)
// Zeros into the rows of the table, 16 bytes at a time where they lie on such boundaries.
struct Zeros {
    float *dtable;
    long long ld;
    int dim, wide;
    // Those of the block's `count` rows from `first` on; with `spans` those that no token reaches.
    __device__ __forceinline__ void rows(long long first, int count, int vocab, const int2 *spans) const {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32, each = (count + warps - 1) / warps;
        const long long end = min(first + count, (long long)vocab);
        first += warp * each;  // the warp's rows, looked up 32 at once
        for (long long v0 = first; v0 < min(first + each, end); v0 += 32) {
            bool empty = v0 + lane < min(first + each, end);
            if (empty && spans) {
                const int2 span = spans[v0 + lane];
                empty = span.x == span.y;
            }
            for (unsigned todo = __ballot_sync(0xffffffffu, empty); todo; todo &= todo - 1) {
                float *row = dtable + (v0 + __ffs(todo) - 1) * ld;
                if (wide)
                    for (int c = lane * 4; c < dim; c += 128) *reinterpret_cast<float4 *>(row + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                else
                    for (int c = lane; c < dim; c += 32) row[c] = 0.f;
            }
        }
    }
};

// Sorting.  Each of 2^bits blocks owns the table rows whose numbers end in its own (frequent tokens have low numbers: neighbours go to
// different blocks).  Its warps, each over a share of the tokens, count its rows' tokens, the counts become places (in front of them
// all tokens of the blocks before), and a second pass puts the tokens there.  Up to kDealFrom tokens every block reads all ids for that: one
// launch, but the ids once for each sorting block out of L2, 128 times for tables of up to 131 072 rows.  Above, a launch in front deals the ids out,
// 1024 to a block, so that a sorting block finds its tokens of them together.  The whole gradient, added, undealt and dealt: 16 384 x 768 f32 into
// 30 522 rows 31 and 36 us, 32 768 44 and 49, 65 536 70 and 72, 131 072 151 and 113; 32 768 x 256 bf16 into 131 072 rows 32 and 32; 262 144 x 256 f32 into as many
// 244 and 166.  Dealing knows 2^kDealBits sorting blocks, those of up to 524 288 rows.  Larger tables have 1024 and more, which read all ids
// whatever their number: 65 536 x 128 f32 into 524 288 rows 53 us, into one row more 95; 262 144 103 us, into 1 048 576 rows 293.
constexpr int kSortWarps = 32, kSortRows = 1024, kSortList = 256;  // rows of a block and own tokens of a warp that shared memory holds
constexpr int kDealFrom = 16384, kDealTokens = 1024, kDealThreads = 256, kDealBits = 9;

// Block s orders ids [1024 s, 1024 (s + 1)) by their sorting block: dealt[1024 s + starts[s][b]] onwards {token, id} of sorting block b.
__global__ void __launch_bounds__(kDealThreads) embedding_deal_kernel(const int *__restrict__ ids, long long ids_stride, int tokens, int vocab, int bits, int2 *__restrict__ dealt, int *__restrict__ starts) {
    constexpr int W = kDealThreads / 32, U = kDealTokens / kDealThreads, PER = (1 << kDealBits) / kDealThreads;
    __shared__ int counts[W << kDealBits], warp_sums[W];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, blocks = 1 << bits;
    for (int i = threadIdx.x; i < W * blocks; i += kDealThreads) counts[i] = 0;
    grid_dependency_sync();
    int id[U], rank[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = blockIdx.x * kDealTokens + warp * (32 * U) + u * 32 + lane;
        id[u] = t < tokens ? ids[t * ids_stride] : -1;
        if ((unsigned)id[u] >= (unsigned)vocab) id[u] = -1;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int to = id[u] & (blocks - 1);
        const unsigned some = __ballot_sync(0xffffffffu, id[u] >= 0);
        unsigned same = 1u << lane;
        int from = 0;
        __syncwarp();
        if (id[u] >= 0) {
            same = __match_any_sync(some, to);
            if (lane == __ffs(same) - 1) from = atomicAdd(counts + warp * blocks + to, __popc(same));  // one lane for each sorting block
        }
        rank[u] = __shfl_sync(0xffffffffu, from, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1));
    }
    __syncthreads();
    // counts -> places: sorting blocks one after the other, in each the warps; a thread has PER sorting blocks in a row
    int count[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int b = threadIdx.x * PER + k;
        count[k] = 0;
        if (b < blocks)
            for (int w = 0; w < W; ++w) count[k] += counts[w * blocks + b];
        sum += count[k];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += left;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int at = upto - sum;
    for (int w = 0; w < warp; ++w) at += warp_sums[w];
    int *start = starts + (long long)blockIdx.x * (blocks + 1);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int b = threadIdx.x * PER + k;
        if (b >= blocks) break;
        start[b] = at;
        if (b == blocks - 1) start[blocks] = at + count[k];
        for (int w = 0; w < W; ++w) {
            const int c = counts[w * blocks + b];
            counts[w * blocks + b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (id[u] >= 0)
            dealt[(long long)blockIdx.x * kDealTokens + counts[warp * blocks + (id[u] & (blocks - 1))] + rank[u]] = make_int2(blockIdx.x * kDealTokens + warp * (32 * U) + u * 32 + lane, id[u]);
}

// Where a sorting block's tokens come from.
enum Source { kStrided, kQuads, kDealt };
struct Ids {
    const int *ids;
    long long stride;
    const int2 *dealt;
    const int *starts;
    int tokens, vocab;
};

template <Source FROM>
__global__ void __launch_bounds__(kSortWarps * 32) embedding_sort_kernel(const Ids in_all, int bits, int2 *__restrict__ spans, int *__restrict__ total, int *__restrict__ order, int *__restrict__ sorted,
                                                                         unsigned *__restrict__ arrived, int counters, const Zeros zeros, int late_rows) {
    if (blockIdx.x >> bits) {  // blocks behind the sorting ones: the table's last rows, a row to a warp, are zero until sums are written
        grid_dependency_sync();
        zeros.rows(late_rows + (long long)(blockIdx.x - (1u << bits)) * (blockDim.x / 32), blockDim.x / 32, in_all.vocab, nullptr);
        return;
    }
    extern __shared__ int2 lists[];  // [warp][kSortList] {token, id}, then [warp][row of the block] counts, later places
    int *places = reinterpret_cast<int *>(lists + blockDim.x / 32 * kSortList);
    __shared__ int warp_sums[kSortWarps], below_all;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32, tokens = in_all.tokens, vocab = in_all.vocab;
    const unsigned own = blockIdx.x, ending = (1u << bits) - 1;
    const int rows = (int)(((unsigned)vocab - own + ending) >> bits);
    for (int i = threadIdx.x; i < warps * rows; i += blockDim.x) places[i] = 0;
    grid_dependency_sync();
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < counters; i += (ending + 1) * blockDim.x) arrived[i] = 0;
    __syncthreads();
    int2 *list = lists + warp * kSortList;
    int *mine = places + warp * rows, below = 0, found = 0;
    // The warp's share, 32 tokens at a time: f(token, id, is it the block's own).  In an order that depends on nothing but their number.
    auto each = [&](auto f) {
        if constexpr (FROM == kDealt) {
            const int sources = (tokens + kDealTokens - 1) / kDealTokens, share = (sources + warps - 1) / warps;
            int lanes = 32;  // that share a source
            while (lanes > 1 && 32 / lanes < share) lanes /= 2;
            for (int s0 = warp * share; s0 < min((warp + 1) * share, sources); s0 += 32 / lanes) {
                const int s = s0 + lane / lanes;
                int from = 0, to = 0;
                if (s < min((warp + 1) * share, sources)) {
                    const int *start = in_all.starts + (long long)s * (ending + 2) + own;
                    from = start[0];
                    to = start[1];
                }
                const int2 *p = in_all.dealt + (long long)s * kDealTokens;
                constexpr int U = 4;
                for (int i = from + lane % lanes; __any_sync(0xffffffffu, i < to); i += U * lanes) {
                    int2 t[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) t[u] = i + u * lanes < to ? p[i + u * lanes] : make_int2(0, -1);
#pragma unroll
                    for (int u = 0; u < U; ++u) f(t[u].x, t[u].y, t[u].y >= 0);
                }
            }
        } else {
            constexpr int U = 4;
            const int share = ((tokens + warps - 1) / warps + 127) / 128 * 128, begin = (int)min((long long)warp * share, (long long)tokens), end = (int)min(begin + (long long)share, (long long)tokens);
            for (int t0 = begin; t0 < end; t0 += 128 * U) {  // four tokens to a lane
                int id[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int t = t0 + u * 128 + lane * 4;
                    if (FROM == kQuads && t + 3 < end) {
                        const int4 q = *reinterpret_cast<const int4 *>(in_all.ids + t);
                        id[u][0] = q.x;
                        id[u][1] = q.y;
                        id[u][2] = q.z;
                        id[u][3] = q.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) id[u][j] = t + j < end ? in_all.ids[(t + j) * in_all.stride] : -1;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool some = (unsigned)id[u][j] < (unsigned)vocab;
                        if (some && ((unsigned)id[u][j] & ending) < own) ++below;
                        f(t0 + u * 128 + lane * 4 + j, id[u][j], some && ((unsigned)id[u][j] & ending) == own);
                    }
            }
        }
    };
    each([&](int t, int id, bool in) {
        const unsigned all = __ballot_sync(0xffffffffu, in);
        if (!all) return;
        if (in) {
            atomicAdd(mine + (id >> bits), 1);  // a count: any order
            const int at = found + __popc(all & ((1u << lane) - 1));
            if (at < kSortList) list[at] = make_int2(t, id);
        }
        found += __popc(all);
    });
    if constexpr (FROM == kDealt)  // a source's first place for this block: as many of its tokens are of the blocks before
        for (int s = threadIdx.x; s < (tokens + kDealTokens - 1) / kDealTokens; s += blockDim.x) below += in_all.starts[(long long)s * (ending + 2) + own];
    for (int o = 16; o; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
    if (lane == 0) warp_sums[warp] = below;
    __syncthreads();
    if (warp == 0) {
        int s = lane < warps ? warp_sums[lane] : 0;
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) below_all = s;
    }
    __syncthreads();
    int next = below_all;  // place of the next row's first token
    for (int r0 = 0; r0 < rows; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        int count = 0;
        if (r < rows)
#pragma unroll 8
            for (int w = 0; w < warps; ++w) count += places[w * rows + r];
        int sum = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += left;
        }
        if (lane == 31) warp_sums[warp] = sum;
        __syncthreads();
        int all = lane < warps ? warp_sums[lane] : 0, ahead = lane < warp ? all : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        int at = next + ahead + sum - count;
        next += all;
        if (r < rows) {
            spans[((long long)r << bits) + own] = make_int2(at, at + count);
            if (count)
#pragma unroll 8
                for (int w = 0; w < warps; ++w) {
                    const int c = places[w * rows + r];
                    places[w * rows + r] = at;
                    at += c;
                }
        }
        __syncthreads();
    }
    if (own == ending && threadIdx.x == 0) *total = next;
    // 32 tokens of the warp's own at a time, from its list, or from all of its share where the list was too short
    auto put = [&](int t, int id, bool in) {
        const unsigned all = __ballot_sync(0xffffffffu, in);
        if (!all) return;
        __syncwarp();
        unsigned same = 1u << lane;
        int from = 0;
        if (in) {
            same = __match_any_sync(all, id);
            if (lane == __ffs(same) - 1) from = atomicAdd(mine + (id >> bits), __popc(same));  // one lane for each row
        }
        const int at = __shfl_sync(0xffffffffu, from, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1));
        if (in) {
            order[at] = t;
            sorted[at] = id;
        }
    };
    if (found <= kSortList) {
        __syncwarp();
        for (int i = 0; i < found; i += 32) {
            const bool in = i + lane < found;
            const int2 t = in ? list[i + lane] : make_int2(0, 0);
            put(t.x, t.y, in);
        }
    } else {
        each(put);
    }
}

// Summing.  A block takes `length` tokens of the sorted order and four columns for each of its threads, and adds the rows of g up one
// after the other; a row of the table that ends is written, what goes on beyond the block's tokens is left in `partial` (slot 2 c: of a
// row that began before block c, 2 c + 1: of one that goes on behind it), and the last block of such a row to arrive adds the pieces up,
// in their order.  Further blocks write the rows that no token reaches.
// Bound by memory: g once, the table once.  Each thread copies its own columns of the next tokens into shared memory asynchronously (no
// barriers, and no registers that wait for them): kAhead rows of the block in flight, five blocks of 256 threads on an SM.
// The whole gradient of 4096 x 768 f32 into 30522 rows: 22.5 us, of which sorting is 8; of 65521 x 1000 bf16 added to 50021 rows: 66 us, of which
// sorting is 15; of 65536 x 4096 bf16 added to 131072: 208 us, 5.6 TB/s.
struct EmbeddingGrad {
    const void *g;
    long long ldg;
    Zeros table;
    int vocab, tokens, slices, chunks, length, add, late_rows;
    float scale;
    const int2 *spans;  // a row's places in the order
    const int *total, *order, *sorted;
    float *partial;
    unsigned *arrived;
};
constexpr int kMaxLength = 256, kAhead = 8;

template <class T>
struct alignas(4 * sizeof(T)) Four {
    T v[4];
};
// The thread's columns: four in a row, or (rows that do not lie on such boundaries) four that lie blockDim.x apart.
template <bool WIDE>
struct Columns {
    int first, dim;
    __device__ Columns(int slice, int dim_) : first(slice * blockDim.x * 4 + threadIdx.x * (WIDE ? 4 : 1)), dim(dim_) {}
    __device__ __forceinline__ int column(int j) const { return first + (WIDE ? j : j * (int)blockDim.x); }
    __device__ __forceinline__ bool has(int j) const { return column(j) < dim; }
};

template <class T, bool WIDE>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const __grid_constant__ EmbeddingGrad a) {
    extern __shared__ char ahead[];  // WIDE: [kAhead][thread] of Four<T>
    __shared__ int rows[kMaxLength + 2], tokens[kMaxLength], last[2], first_piece[2];
    grid_dependency_sync();
    if ((int)blockIdx.x >= a.chunks * a.slices) {
        a.table.rows((long long)(blockIdx.x - a.chunks * a.slices) * kZeroRows, kZeroRows, a.late_rows, a.spans);
        return;
    }
    const int chunk = blockIdx.x / a.slices, slice = blockIdx.x - chunk * a.slices, from = chunk * a.length;
    const int total = *a.total;  // not waited for before what it decides about has been asked for
    for (int i = threadIdx.x; i < a.length + 2; i += blockDim.x) {  // rows[i + 1]: of the i-th token, and of those in front and behind; -1 = none
        const int place = from + i - 1, inside = min(max(place, 0), a.tokens - 1);
        const int row = a.sorted[inside], token = a.order[inside];  // behind the last place: not used
        rows[i] = place >= 0 && place < total ? row : -1;
        if (i > 0 && i <= a.length) tokens[i - 1] = place < total ? token : 0;
    }
    if (from >= total) return;  // the whole block
    const int n = min(a.length, total - from);
    __syncthreads();
    int2 span = make_int2(0, 1);  // of the block's first and last row, for their first two threads, which may need them at the end
    if (threadIdx.x < 2) span = a.spans[rows[threadIdx.x ? n : 1]];
    const Columns<WIDE> cols(slice, a.table.dim);
    const T *g = (const T *)a.g + cols.first;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    auto output = [&](int v) {
        float *row = a.table.dtable + v * a.table.ld;
        // Added: one addition to each element in all, made in L2; reading the row first would stop the thread at the end of every row.
        if (WIDE) {
            if (cols.first >= cols.dim) return;
            const float4 o = make_float4(sum[0] * a.scale, sum[1] * a.scale, sum[2] * a.scale, sum[3] * a.scale);
            if (a.add) asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(row + cols.first), "f"(o.x), "f"(o.y), "f"(o.z), "f"(o.w) : "memory");
            else *reinterpret_cast<float4 *>(row + cols.first) = o;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!cols.has(j)) continue;
                if (a.add) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(row + cols.column(j)), "f"(sum[j] * a.scale) : "memory");
                else row[cols.column(j)] = sum[j] * a.scale;
            }
        }
    };
    const long long stride = (long long)a.slices * blockDim.x * 4;  // of the partial sums: [slot][slice][column][thread]
    float *partial = a.partial + (long long)slice * blockDim.x * 4 + threadIdx.x;
    auto leave = [&](int slot) {
#pragma unroll
        for (int j = 0; j < 4; ++j) __stcg(partial + slot * stride + j * blockDim.x, sum[j]);
    };
    const bool before = rows[0] == rows[1];  // the first row began in front
    bool first = true;                       // ... and goes on
    auto ended = [&](int i) {                // the row of tokens [.., i)
        if (first && before) leave(2 * chunk);
        else output(rows[i]);
        first = false;
        sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
    };
    if (WIDE) {
        Four<T> *mine = reinterpret_cast<Four<T> *>(ahead) + threadIdx.x;
        const bool some = cols.first < cols.dim;
        const unsigned place = (unsigned)__cvta_generic_to_shared(mine), step = blockDim.x * sizeof(Four<T>);
        auto fetch = [&](int i, int u) {
            if (some && i < n) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(place + u * step), "l"(g + tokens[i] * a.ldg), "n"((int)sizeof(Four<T>)) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int u = 0; u < kAhead; ++u) fetch(u, u);
        int row = rows[1];
        for (int i0 = 0; i0 < n; i0 += kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {  // the places of the ring at fixed offsets: 2 us less in both of the cases above
                const int i = i0 + u;
                if (i >= n) break;
                asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
                const int now = rows[i + 1];
                if (now != row) {
                    ended(i);
                    row = now;
                }
                const Four<T> v = mine[u * blockDim.x];
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += widen(v.v[j]);
                asm volatile("" ::"f"(sum[0]), "f"(sum[1]), "f"(sum[2]), "f"(sum[3]) : "memory");  // read before the place is taken again
                fetch(i + kAhead, u);
            }
        }
    } else {
        constexpr int U = 8;
        for (int i0 = 0; i0 < n; i0 += U) {
            T v[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i0 + u < n && cols.has(j)) v[u][j] = g[tokens[i0 + u] * a.ldg + j * (int)blockDim.x];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i >= n) break;
                if (i && rows[i + 1] != rows[i]) ended(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += widen(v[u][j]);
            }
        }
    }
    int spans_before = before ? rows[1] : -1, spans_after = -1;
    if (rows[n + 1] != rows[n] && !(first && before)) {
        output(rows[n]);
    } else if (first && before) {
        leave(2 * chunk);
    } else {
        leave(2 * chunk + 1);
        spans_after = rows[n];
    }
    if (spans_before < 0 && spans_after < 0) return;  // the whole block
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
        const int v = threadIdx.x ? spans_after : spans_before;
        last[threadIdx.x] = 0;
        if (v >= 0) {
            const int c0 = span.x / a.length, c1 = (span.y - 1) / a.length;
            last[threadIdx.x] = atomicAdd(a.arrived + (long long)c0 * a.slices + slice, 1u) == (unsigned)(c1 - c0) ? c1 - c0 + 1 : 0;
            first_piece[threadIdx.x] = c0;
        }
        __threadfence();
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        if (!last[k]) continue;
        const int v = k ? spans_after : spans_before, c0 = first_piece[k], pieces = last[k];
        sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll 8
        for (int p = 0; p < pieces; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += __ldcg(partial + (2 * (long long)(c0 + p) + (p == 0)) * stride + j * blockDim.x);
        output(v);
    }
}

}  // namespace

// Do all rows start at a multiple of `boundary` bytes?
bool on_boundary(const void *p, long long pitch, size_t size, size_t boundary) { return reinterpret_cast<uintptr_t>(p) % boundary == 0 && (size_t)pitch * size % boundary == 0; }

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
                const bool wide = y.cols % V == 0 && on_boundary(table.ptr, table.pitch, sizeof(T), 16) && on_boundary(y.ptr, y.pitch, sizeof(Y), 16);
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
    if (tokens > kMaxRows) return ctx.fail(SAGE_ERR_INVALID, "embedding_grad: too many tokens");
    const size_t size = g.dtype == SAGE_F32 ? 4 : 2;
    const bool wide = dim % 4 == 0 && on_boundary(g.ptr, g.pitch, size, 4 * size) && on_boundary(dtable.ptr, dtable.pitch, 4, 16);
    // Four columns a thread, up to 256 threads (eight 16-bit columns in half the threads: 65521 x 1000 bf16 113 us instead of 80).  So many tokens a
    // block that there are seven blocks for each SM, of which five of 256 threads are resident: sums of few rows begin while others wait (four,
    // seven, eight for each: 72, 67, 70 us).
    const long long threads = dim >= 1024 ? 256 : ((dim + 3) / 4 + 31) / 32 * 32, slices = (dim + 4 * threads - 1) / (4 * threads);
    long long length = (tokens * slices + ctx.sm_count * 7 - 1) / (ctx.sm_count * 7);
    length = length < 16 ? 16 : length > kMaxLength ? kMaxLength : (length + 7) / 8 * 8;
    const long long chunks = (tokens + length - 1) / length;
    // Rows that no token reaches become zero beside the sums.  24 MB of the table are cleared beside the sorting already, which leaves the memory
    // idle, whether tokens reach them or not: the last rows, since frequent tokens have low numbers (with 0, 12, 24 and 48 MB: 512 x 768
    // into 30522 rows 21.1, 19.9, 19.4, 20.1 us; 4096 24.9, 23.6, 22.7, 23.6; 16384 44.7, 43.4, 40.2, 41.9; 65536 74.5, 74.6, 72.2, 72.5; 4096 x 1024 into
    // 131072 86.3, 84.6, 83.3, 82.6; 8192 x 512 into 8000, 16 MB in all, 20.2, 21.0, 21.5, 21.8; 32768 x 4096 into 131072 403, 409, 408, 406).
    const long long early_rows = add ? 0 : std::min(vocab, (24ll << 20) / (dim * 4)), late_rows = add ? 0 : vocab - early_rows, zero_blocks = (late_rows + kZeroRows - 1) / kZeroRows;
    if (chunks * slices + zero_blocks > 0x7fffffffll) return ctx.fail(SAGE_ERR_INVALID, "embedding_grad: too many rows");
    const auto rounded = [](long long words) { return (words + 63) / 64 * 64; };
    const long long starts = rounded(2 * vocab + 1), places = rounded(tokens), counters = rounded(chunks * slices);
    Block *scratch = ctx.allocator().alloc((size_t)(starts + 2 * places + counters + 2 * chunks * slices * threads * 4) * 4);
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
    a.table = Zeros{(float *)dtable.ptr, dtable.pitch, (int)dim, (int)(dim % 4 == 0 && on_boundary(dtable.ptr, dtable.pitch, 4, 16))};
    a.vocab = (int)vocab;
    a.tokens = (int)tokens;
    a.slices = (int)slices;
    a.chunks = (int)chunks;
    a.length = (int)length;
    a.add = add;
    a.late_rows = (int)late_rows;
    a.scale = scale;
    int bits = 0;  // about one sorting block for each SM; more where shared memory does not hold the counts of that many rows
    while ((2ll << bits) <= vocab && ((2 << bits) <= ctx.sm_count || ((vocab - 1) >> bits) + 1 > kSortRows)) ++bits;
    const int warps = tokens <= 8192 ? 8 : kSortWarps;  // few ids: the counts of a warp cost more than its share of the ids
    const size_t smem = (size_t)((((vocab - 1) >> bits) + 1) + 2 * kSortList) * warps * 4;
    const bool deal = tokens > kDealFrom && bits <= kDealBits;
    Ids source = {(const int *)ids.ptr, ids.stride, nullptr, nullptr, (int)tokens, (int)vocab};
    Block *dealt = nullptr;
    const long long sources = (tokens + kDealTokens - 1) / kDealTokens;
    sage_status st = SAGE_OK;
    if (deal) {
        dealt = ctx.allocator().alloc((size_t)(sources * kDealTokens * 8 + sources * ((1ll << bits) + 1) * 4));
        if (!dealt) {
            ctx.allocator().free(scratch);
            return ctx.fail(SAGE_ERR_OOM, "embedding_grad: out of memory");
        }
        source.dealt = (const int2 *)dealt->ptr;
        source.starts = (const int *)(source.dealt + sources * kDealTokens);
        ctx.note_launch("embedding_deal");
        if (!ctx.dry())
            st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), embedding_deal_kernel, dim3((unsigned)sources), dim3(kDealThreads), 0, source.ids, source.stride, source.tokens, source.vocab, bits,
                                                 (int2 *)source.dealt, (int *)source.starts),
                                "embedding_deal");
    }
    ctx.note_launch("embedding_sort");
    const long long blocks = chunks * slices + zero_blocks;  // none: no tokens, and all of the table cleared early
    if (blocks) ctx.note_launch("embedding_grad");
    if (!ctx.dry() && !st) {
        const auto sort = deal ? embedding_sort_kernel<kDealt> : ids.stride == 1 && reinterpret_cast<uintptr_t>(ids.ptr) % 16 == 0 ? embedding_sort_kernel<kQuads> : embedding_sort_kernel<kStrided>;
        st = ctx.check_cuda(cudaFuncSetAttribute(sort, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSortRows + 2 * kSortList) * kSortWarps * 4), "embedding_sort");
        if (!st)
            st = ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), sort, dim3((1u << bits) + (unsigned)((early_rows + warps - 1) / warps)), dim3(warps * 32), smem, source, bits, (int2 *)a.spans, (int *)a.total, (int *)a.order, (int *)a.sorted,
                                                 a.arrived, (int)counters, a.table, (int)late_rows),
                                "embedding_sort");
        if (!st && blocks)
            st = with_type(g.dtype, [&](auto t) {
                typedef decltype(t) T;
                const size_t smem_ahead = wide ? kAhead * threads * sizeof(Four<T>) : 0;  // 32 KB at most
                return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? embedding_grad_kernel<T, true> : embedding_grad_kernel<T, false>,
                                                       dim3((unsigned)blocks), dim3((unsigned)threads), smem_ahead, a),
                                      "embedding_grad");
            });
    }
    if (dealt) ctx.allocator().free(dealt);
    ctx.allocator().free(scratch);
    return st;
}

}  // namespace k
}  // namespace sage
