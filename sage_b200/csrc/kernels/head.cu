// Log probabilities of given tokens straight from hidden states, x = scale hidden weight^T, without keeping the logits, and the gradient:
//   log p_j = x_j - m - ln S,  m = max x,  S = sum exp(x_j - m),  H = ln S - sum (x_j - m) exp(x_j - m) / S
//   q_j = gl (delta(j, id) - p_j) - ge p_j (ln p_j + H);   dhidden = scale q weight,   dweight = scale q^T hidden
//
// 16-bit operands (head_device.h).  Forward: one product whose tiles are finished in registers; each half tile leaves a row's {m, S, sum} and a second
// launch joins them.  Gradient: the vocabulary in pieces; of each piece the product again, q into a buffer (16 bits: q is an operand of two
// products, rounded like the operands beside it; the sums of both are f32), then its two products.
// Bound by the tensor cores: 2 rows vocab width operations forward, three times that for the gradient, which makes the logits again.
// f32 operands: the same products of their pieces, which a pass over them makes first.
#include <algorithm>
#include <cmath>

#include "eight.h"
#include "head_device.h"
#include "language.h"

namespace sage {
void *driver_symbol(const char *name);  // runtime/context.cc
namespace k {
namespace head {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr size_t kPartBytes = (size_t)512 << 20;   // what half tiles leave of a run of rows
constexpr size_t kPieceBytes = (size_t)256 << 20;  // a piece of q

__device__ __forceinline__ float exp2_of(float x) { return exp2f(x); }

// One row's sums, joined: (m, S, A) with A = sum (x - m) c2 2^((x - m) c2).
struct Sums {
    float m, s, a;
};
__device__ __forceinline__ Sums joined(Sums x, Sums y, float c2) {
    const float m = fmaxf(x.m, y.m);  // of two numbers the larger; nan only beside sums that are nan
    const float fx = x.m == -INFINITY ? 0.f : (x.m - m) * c2, fy = y.m == -INFINITY ? 0.f : (y.m - m) * c2;
    const float ex = x.m == -INFINITY ? 1.f : exp2_of(fx), ey = y.m == -INFINITY ? 1.f : exp2_of(fy);  // (sums of nothing are zero, or nan)
    const float ax = ex > 0.f ? fmaf(x.s * ex, fx, x.a * ex) : x.s * ex, ay = ey > 0.f ? fmaf(y.s * ey, fy, y.a * ey) : y.s * ey;
    return Sums{m, x.s * ex + y.s * ey, ax + ay};
}

struct Values {
    float *log_probs, *entropy, *stats;
    long long log_probs_stride, entropy_stride, stats_pitch;
};

// 32 rows a block: its warps share the parts of all of them, a lane to a row, then a warp takes a row, a lane to what each warp found.
__global__ void __launch_bounds__(1024) head_join_kernel(const float4 *parts, int count, int rows, const float *asked, const int *ids, long long ids_stride, int vocab, float scale, float c2,
                                                         Values y) {
    __shared__ Sums all[32][33];
    grid_dependency_sync();
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    Sums x{-INFINITY, 0.f, 0.f};
    if ((int)blockIdx.x * 32 + lane < rows) {
#pragma unroll 4
        for (int i = warp; i < count; i += warps) {
            const float4 p = __ldg(parts + (long long)i * rows + (int)blockIdx.x * 32 + lane);
            x = joined(x, Sums{p.x, p.y, p.z}, c2);
        }
    }
    all[warp][lane] = x;
    __syncthreads();
    for (int r = warp; r < 32; r += warps) {
        const int row = (int)blockIdx.x * 32 + r;
        if (row >= rows) return;
        x = lane < warps ? all[lane][r] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            const Sums o{__shfl_xor_sync(0xffffffffu, x.m, off), __shfl_xor_sync(0xffffffffu, x.s, off), __shfl_xor_sync(0xffffffffu, x.a, off)};
            x = lane & off ? joined(o, x, c2) : joined(x, o, c2);  // (the same order on both sides: the same bits)
        }
        if (lane) continue;
        const bool none = x.m == -INFINITY && x.s == 0.f;  // no token has a chance
        const float ln_s = logf(x.s);
        const int id = __ldg(ids + row * ids_stride);
        const bool scored = id >= 0 && id < vocab;
        if (y.log_probs) y.log_probs[row * y.log_probs_stride] = !scored ? 0.f : none ? -INFINITY : (asked[row] - x.m) * scale - ln_s;
        if (y.entropy) y.entropy[row * y.entropy_stride] = none ? 0.f : ln_s - kLn2 * x.a / x.s;
        if (y.stats) {
            y.stats[row * y.stats_pitch] = x.m;
            y.stats[row * y.stats_pitch + 1] = x.s;
        }
    }
}

// Few rows (one token of each of a few sequences): a warp takes four rows of the weights at a time, straight from memory in order, with the hidden states in
// shared memory.  Bound by the weights' bytes.  A lane sums its columns in f32; of the 4 x RB sums of a warp every lane ends up with one (half of
// what it has goes to another lane at each step), and keeps the sums of exponentials for those of its place, or (Q) makes of its logit its part of the gradient: from
// logits of the tensor cores, which differ in their last places, p = exp(x - m) / S of a likely token would be off by as much.
struct FewProbs {
    const float4 *about;  // head_rows_kernel's
    const float *gl;
    const unsigned *gmax;
    float alpha;          // f32
    unsigned short *q;    // 16 bits; f32: three planes of pieces
    long long pitch, plane;
    int first;            // token that the weights' first row stands for
};
template <class T, int RB, bool Q>
__global__ void __launch_bounds__(256, 2) head_few_kernel(const T *hidden, long long hidden_pitch, const T *weight, long long weight_pitch, int rows, int vocab, int width, const int *ids,
                                                          long long ids_stride, float c2, float4 *parts, float *asked, const FewProbs to) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Sums all[8][RB];
    grid_dependency_sync();
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, runs = width / 8;
    Eight<T> *states = (Eight<T> *)smem;
    for (int i = (int)threadIdx.x; i < RB * runs; i += 256) {
        const int r = i / runs;
        if (r < rows) states[i].load_once((const char *)(hidden + r * hidden_pitch + (i - r * runs) * 8));
        else states[i].clear();
    }
    __syncthreads();
    constexpr int N = 4 * RB, kLanes = 32 / N;  // sums; lanes that end up with the same one
    const int index = lane / kLanes, mine = index % RB, which = index / RB;
    const int id = mine < rows ? __ldg(ids + mine * ids_stride) : -1;
    float4 about = make_float4(0.f, 0.f, 0.f, 0.f);
    float gl = 0.f;
    if (Q && mine < rows) {
        const float by = sizeof(T) == 4 ? to.alpha : to.gmax ? power_of_two(stored_exponent(to.gmax)) : 1.f;
        about = __ldg(to.about + mine);
        about.z *= by, about.w *= by;
        gl = __ldg(to.gl + mine) * by;
    }
    Sums kept{-INFINITY, 0.f, 0.f};
    for (long long first = 4ll * ((long long)blockIdx.x * 8 + warp); first < vocab; first += 32ll * gridDim.x) {
        const char *row[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) row[k] = (const char *)(weight + min(first + k, vocab - 1ll) * weight_pitch);
        float2 sum[4][RB];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int r = 0; r < RB; ++r) sum[k][r] = make_float2(0.f, 0.f);
#pragma unroll(RB <= 2 ? 4 : 2)
        for (int c = lane; c < runs; c += 32) {
            float2 x[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                Eight<T> v;
                v.load_once(row[k] + (long long)c * (8 * (int)sizeof(T)));
                v.open(x[k]);
            }
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                float2 h[4];
                states[r * runs + c].open(h);
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[k][r] = fma2(x[k][i], h[i], sum[k][r]);
            }
        }
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = sum[i / RB][i % RB].x + sum[i / RB][i % RB].y;
        int n = N;
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            if (n > 1) {
                n /= 2;
                const bool upper = lane & off;
#pragma unroll
                for (int i = 0; i < N / 2; ++i)
                    if (i < n) v[i] = (upper ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + n], off);
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
            }
        }
        const long long token = first + which;
        if (Q) {
            if (token < vocab && mine < rows && lane % kLanes == 0) {
                const float d = fmaf(v[0] - about.x, c2, about.y);
                float q = exp2_of(d) * fmaf(about.w, fmaxf(d, kFar), about.z), none = 0.f;
                if (token + to.first == id) q += gl;
                unsigned short *at = to.q + mine * to.pitch + token;
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) at[k * to.plane] = (unsigned short)take_piece(q, none);
                } else {
                    *(T *)at = narrowed<T>(q);
                }
            }
        } else if (token < vocab) {
            const float x = v[0];
            if (x > kept.m) {
                const float by = kept.m == -INFINITY ? 0.f : (kept.m - x) * c2, f = kept.m == -INFINITY ? 0.f : exp2_of(by);
                kept.a = f > 0.f ? fmaf(kept.s * f, by, kept.a * f) : kept.s * f;  // (zero, or not a number)
                kept.s *= f;
                kept.m = x;
            }
            const float d = (x - (kept.m == -INFINITY ? 0.f : kept.m)) * c2, e = exp2_of(d);
            kept.s += e;
            kept.a = fmaf(e, fmaxf(d, kFar), kept.a);
            if (token == id) asked[mine] = x;
        }
    }
    if constexpr (!Q) {
#pragma unroll
        for (int off = 16; off >= 8; off >>= 1)  // the four weights' rows of a hidden state
            kept = joined(kept, Sums{__shfl_xor_sync(0xffffffffu, kept.m, off), __shfl_xor_sync(0xffffffffu, kept.s, off), __shfl_xor_sync(0xffffffffu, kept.a, off)}, c2);
        if (lane < 8 && lane % kLanes == 0) all[warp][mine] = kept;
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            Sums t = all[0][threadIdx.x];
            for (int w = 1; w < 8; ++w) t = joined(t, all[w][threadIdx.x], c2);
            parts[(long long)blockIdx.x * rows + threadIdx.x] = make_float4(t.m, t.s, t.a, 0.f);
        }
    }
}

// What the gradient needs of each row, once.
__global__ void __launch_bounds__(256) head_rows_kernel(const float *stats, long long stats_pitch, VectorArg entropy, VectorArg gl, VectorArg ge, const int *ids, long long ids_stride, int rows,
                                                        int vocab, float4 *about, float *gls, unsigned *gmax) {
    grid_dependency_sync();
    const int row = (int)blockIdx.x * 256 + (int)threadIdx.x;
    float size = 0.f;
    if (row < rows) {
        const float m = stats[row * stats_pitch], s = stats[row * stats_pitch + 1];
        const int id = __ldg(ids + row * ids_stride);
        const bool none = m == -INFINITY && s == 0.f;
        const float g = gl.ptr && !none && id >= 0 && id < vocab ? ((const float *)gl.ptr)[row * gl.stride] : 0.f;
        const float e = ge.ptr && !none ? ((const float *)ge.ptr)[row * ge.stride] : 0.f, h = e != 0.f ? ((const float *)entropy.ptr)[row * entropy.stride] : 0.f;
        about[row] = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(m, -log2f(s), -fmaf(e, h, g), -e * kLn2);
        gls[row] = g;
        size = fabsf(g) + fabsf(e) * (fabsf(h) + 0.5f);
        if (!(size < INFINITY)) size = 0.f;
    }
    if (gmax) {
#pragma unroll
        for (int off = 16; off; off >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, off));
        if (!(threadIdx.x & 31) && size > 0.f) atomicMax(gmax, __float_as_uint(size));  // (a largest value: in any order)
    }
}

// Rows into others: the sum of `slices` that lie apart, in another type, with another pitch.  WIDE: four elements of `x` on 16-byte (f32) or 8-byte boundaries.
template <class A, class B, bool WIDE>
__global__ void __launch_bounds__(256) head_rows_copy_kernel(const A *x, long long px, B *y, long long py, long long rows, int cols, int slices, long long slice) {
    struct alignas(4 * sizeof(A)) Four {
        A v[4];
    };
    grid_dependency_sync();
    const int per = (cols + 3) / 4;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < rows * per; i += gridDim.x * 256ll) {
        const long long r = rows * per <= 0x7fffffffll ? (int)i / per : i / per, c = (i - r * per) * 4;
        const A *from = x + r * px + c;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (WIDE) {
#pragma unroll 4
            for (int s = 0; s < slices; ++s) {
                const Four f = *(const Four *)(from + s * slice);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += widen(f.v[e]);
            }
        } else {
            for (int s = 0; s < slices; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < cols) v[e] += widen(from[s * slice + e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) y[r * py + c + e] = narrowed<B>(v[e]);
    }
}
template <class A, class B>
sage_status copy_rows(Context &ctx, const A *x, long long px, B *y, long long py, long long rows, int cols, int slices, long long slice) {
    ctx.note_launch("head_rows_copy");
    if (ctx.dry()) return SAGE_OK;
    const long long blocks = std::min<long long>((rows * ((cols + 3) / 4) + 255) / 256, ctx.sm_count * 16ll);
    const bool wide = (uintptr_t)x % (4 * sizeof(A)) == 0 && px % 4 == 0 && cols % 4 == 0 && slice % 4 == 0;
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? head_rows_copy_kernel<A, B, true> : head_rows_copy_kernel<A, B, false>, dim3((unsigned)blocks), dim3(256), 0, x, px, y, py, rows, cols, slices, slice), "head_rows_copy");
}

// Three bf16 pieces of each f32 element of up to two matrices, eight to a thread.
struct ToPieces {
    const float *x;
    __nv_bfloat16 *y;
    long long px, py, plane, groups;  // groups: of eight elements, rows of py / 8
    int cols, wide;                   // wide: whole groups on 16-byte boundaries
};
__global__ void __launch_bounds__(256) head_pieces_kernel(const ToPieces a, const ToPieces b) {
    grid_dependency_sync();
    for (long long n = blockIdx.x * 256ll + threadIdx.x; n < a.groups + b.groups; n += gridDim.x * 256ll) {
        const bool second = n >= a.groups;
        const ToPieces &m = second ? b : a;
        const long long i = second ? n - a.groups : n, per = m.py / 8, r = m.groups <= 0x7fffffffll ? (int)i / (int)per : i / per, c = (i - r * per) * 8;
        const float *from = m.x + r * m.px + c;
        float v[8];
        if (m.wide) {
            const float4 p = *(const float4 *)from, q = *((const float4 *)from + 1);
            v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < m.cols ? from[e] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            unsigned w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = take_piece(v[2 * e], v[2 * e + 1]);
            *(uint4 *)(m.y + k * m.plane + r * m.py + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ------------------------------------------------------------------------------------------ host
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Boxes of `box_rows` rows, `box_bytes` of each, of a matrix (of each of several, `plane` elements apart).
sage_status map_of(Context &ctx, int dtype, const void *base, long long cols, long long rows, long long pitch, int box_rows, CUtensorMap *map, int box_bytes = 128, int planes = 0, long long plane = 0) {
    static const EncodeTiled encode = reinterpret_cast<EncodeTiled>(driver_symbol("cuTensorMapEncodeTiled"));
    if (!encode) return ctx.fail(SAGE_ERR_DEVICE, "cuTensorMapEncodeTiled is not available");
    const int size = dtype == SAGE_F32 ? 4 : 2;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)std::max(planes, 1)}, strides[2] = {(cuuint64_t)(pitch * size), (cuuint64_t)((plane ? plane : pitch) * size)};
    const cuuint32_t box[3] = {(cuuint32_t)(box_bytes / size), (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == SAGE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == SAGE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (encode(map, type, planes ? 3 : 2, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return ctx.fail(SAGE_ERR_DEVICE, "head_log_probs: cuTensorMapEncodeTiled failed");
    return SAGE_OK;
}

// Memory of the call, given back with it: the stream orders its next use.
struct Scratch {
    Context &ctx;
    std::vector<Block *> blocks;
    explicit Scratch(Context &c) : ctx(c) {}
    ~Scratch() {
        for (Block *b : blocks) ctx.allocator().free(b);
    }
    template <class P>
    sage_status get(size_t bytes, P **out) {
        Block *b = ctx.allocator().alloc(bytes);
        if (!b) return ctx.fail(SAGE_ERR_OOM, "head_log_probs: out of memory");
        blocks.push_back(b);
        *out = (P *)b->ptr;
        return SAGE_OK;
    }
};

struct Matrix {  // rows x cols, cols contiguous; f32: in pieces, `plane` elements apart
    const void *p = nullptr;
    long long rows = 0, cols = 0, pitch = 0, plane = 0;
};
bool on_16(const void *p, long long pitch, int size) { return (uintptr_t)p % 16 == 0 && pitch * size % 16 == 0; }

// The operand as TMA reads it: rows on 16-byte boundaries, copied where they are not.
template <class T>
sage_status aligned(Context &ctx, Scratch &scratch, const RowsArg &r, Matrix *m) {
    *m = Matrix{r.ptr, r.rows, r.cols, r.rows > 1 ? r.pitch : (r.cols + 7) / 8 * 8};
    if (on_16(m->p, m->pitch, 2) && m->pitch >= r.cols) return SAGE_OK;
    const long long pitch = (r.cols + 7) / 8 * 8;
    T *to = nullptr;
    sage_status st = scratch.get((size_t)(r.rows * pitch) * 2, &to);
    if (!st) st = copy_rows<T, T>(ctx, (const T *)r.ptr, r.rows > 1 ? r.pitch : r.cols, to, pitch, r.rows, (int)r.cols, 1, 0);
    m->p = to;
    m->pitch = pitch;
    return st;
}

Product shape_of(Context &ctx, long long m, long long n, long long k) {
    Product p{};
    p.m = (int)m;
    p.n = (int)n;
    p.k = (int)k;
    p.bn = n <= 128 || (n + 255) / 256 * 256 - (n + 127) / 128 * 128 > 0 && n < 1024 ? 128 : 256;  // fewer columns that are not there
    p.tiles_m = (int)((m + 255) / 256);
    p.tiles_n = (int)((n + p.bn - 1) / p.bn);
    p.slices = 1;
    p.slice_blocks = p.chain = (int)((k + kK - 1) / kK);
    p.band = 8;
    p.status = ctx.status_word_dev;
    return p;
}

// K-blocks that the tensor cores add up where logits are made, by the values and by the gradient alike: chains of equal length, 512 k at most.
int logits_chain(const Product &p) {
    const int chains = (p.slice_blocks + 7) / 8;
    return (p.slice_blocks + chains - 1) / chains;
}

template <class T, bool A_MN, bool B_MN, End END, bool F32 = false>
sage_status launch(Context &ctx, const char *name, Product p, int dtype, const Matrix &a, const Matrix &b, int out_type, const Matrix &c) {
    ctx.note_launch(name);
    if (ctx.dry()) return SAGE_OK;
    p.band = std::min(p.band, p.tiles_m);
    CUtensorMap ma, mb, mc;
    constexpr int kPlanes = F32 ? 3 : 1;
    sage_status st = map_of(ctx, dtype, a.p, a.cols, a.rows, a.pitch, A_MN ? kK : 128, &ma, 128, kPlanes, a.plane);
    if (!st) st = map_of(ctx, dtype, b.p, b.cols, b.rows, b.pitch, B_MN ? kK : p.bn / 2, &mb, 128, kPlanes, b.plane);
    if (!st && END != kStats) st = map_of(ctx, out_type, c.p, c.cols, c.rows, c.pitch, 32, &mc, F32 && END == kProbs ? 64 : 128);
    else mc = ma;
    if (F32) {
        p.slice_blocks *= kProducts;
        p.chain = kProducts;
    }
    const auto kernel = head_product_kernel<T, A_MN, B_MN, END, F32>;
    if (!st) st = ctx.check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem), name);
    if (st) return st;
    const long long tiles = (long long)p.tiles_m * p.tiles_n * p.slices;
    const unsigned grid = 2 * (unsigned)std::min<long long>(tiles, ctx.sm_count / 2);
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), 2, kernel, dim3(grid), dim3(kBlock), kSmem, ma, mb, mc, p), name);
}

// out = alpha * the product, rounded once.  Pieces of K come in calls of their own, the first with `first`, the last with `last`; where tiles are few, slices
// of K are worked on side by side.  `held`: f32 sums between the calls, made here where they are needed.
struct Result {
    RowsArg out;
    float *sums = nullptr;
    long long pitch = 0;
    int slices = 1, slice_rows = 0;
    bool wide = false;  // sums are kept in f32
};
void plan(Context &ctx, const Product &p, long long k, bool pieces, Result *r) {
    const int pairs = ctx.sm_count / 2, tiles = p.tiles_m * p.tiles_n;
    const int blocks = (int)((k + kK - 1) / kK);
    r->slices = tiles >= pairs ? 1 : std::max(1, std::min(pairs / tiles, blocks / 8));
    r->slice_rows = p.tiles_m * 256;
    r->wide = pieces || r->slices > 1 || !on_16(r->out.ptr, r->out.pitch, r->out.dtype == SAGE_F32 ? 4 : 2);
}
template <class T, bool A_MN, bool B_MN, bool F32 = false>
sage_status multiply(Context &ctx, Scratch &scratch, const char *name, Product p, int dtype, const Matrix &a, const Matrix &b, bool first, bool last, Result *r) {
    sage_status st = SAGE_OK;
    const long long rows = r->out.rows, cols = r->out.cols;
    const bool f32 = r->out.dtype == SAGE_F32, direct = f32 && r->slices == 1 && on_16(r->out.ptr, r->out.pitch, 4);  // sums may be the result itself
    if constexpr (!F32)
        if (!r->wide && !f32) return launch<T, A_MN, B_MN, kNarrow>(ctx, name, p, dtype, a, b, dtype, Matrix{r->out.ptr, rows, cols, r->out.pitch});
    p.add = !first;
    if (direct) return launch<T, A_MN, B_MN, kWide, F32>(ctx, name, p, dtype, a, b, SAGE_F32, Matrix{r->out.ptr, rows, cols, r->out.pitch});
    if (first) {
        r->pitch = (cols + 7) / 8 * 8;
        st = scratch.get((size_t)r->slices * r->slice_rows * r->pitch * 4, &r->sums);
        if (st) return st;
    }
    const int blocks = p.slice_blocks;
    p.slice_blocks = (blocks + r->slices - 1) / r->slices;
    p.slices = (blocks + p.slice_blocks - 1) / p.slice_blocks;
    if (first) r->slices = p.slices;  // (pieces that follow are no longer: a slice of the last one may have nothing to add)
    p.slice_rows = r->slice_rows;
    st = launch<T, A_MN, B_MN, kWide, F32>(ctx, name, p, dtype, a, b, SAGE_F32, Matrix{r->sums, (long long)r->slices * r->slice_rows, cols, r->pitch});
    if (st || !last) return st;
    const long long slice = (long long)r->slice_rows * r->pitch;
    if (f32) return copy_rows<float, float>(ctx, r->sums, r->pitch, (float *)r->out.ptr, r->out.pitch, rows, (int)cols, r->slices, slice);
    return copy_rows<float, T>(ctx, r->sums, r->pitch, (T *)r->out.ptr, r->out.pitch, rows, (int)cols, r->slices, slice);
}

sage_status join(Context &ctx, const float4 *parts, int count, long long rows, const float *asked, const VectorArg &ids, long long vocab, float scale, const Values &y) {
    ctx.note_launch("head_join");
    if (ctx.dry()) return SAGE_OK;
    const int warps = count >= 64 && rows < 32 * 296 ? 32 : 8;
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), head_join_kernel, dim3((unsigned)((rows + 31) / 32)), dim3(32 * warps), 0, parts, count, (int)rows, asked, (const int *)ids.ptr,
                                           ids.stride, (int)vocab, scale, scale * kLog2E, y),
                          "head_join");
}

// Rows that are few enough for dot products, and how many of them a pass over the weights takes: eight, or what 96 KB of shared memory hold.  16-bit operands
// up to four rows (one, four, eight rows of 131072 x 4096 164, 208, 290 us, the tensor cores 203; 30522 x 768 20, 22, 27 and 23); f32 operands up
// to four passes (16 rows of 131072 x 4096 in four 1250 us, the tensor cores, which need the weights in pieces first, 1820; 32 of 50021 x 2048 460 and 475).  The gradient goes the values'
// way (one row of 131072 x 4096 bf16 557 us, by the tensor cores 662; four f32 rows 2850 and 3800, sixteen 4000 and 3790).
long long few(const Head &a) {
    const int size = a.hidden.dtype == SAGE_F32 ? 4 : 2;
    if (a.hidden.cols % 8 || !on_16(a.hidden.ptr, a.hidden.rows > 1 ? a.hidden.pitch : 0, size) || !on_16(a.weight.ptr, a.weight.rows > 1 ? a.weight.pitch : 0, size)) return 0;
    long long pass = 8;
    while (pass && pass * a.hidden.cols * size > 96 * 1024) pass /= 2;
    while (pass > 1 && pass / 2 >= a.hidden.rows) pass /= 2;
    return a.hidden.rows <= (size == 4 ? 4 * pass : std::min(4ll, pass)) ? pass : 0;
}
// Rows [at, at + count) of the operands and results.
RowsArg cut(const RowsArg &r, long long at, long long count) {
    RowsArg c = r;
    if (r.ptr) c.ptr = (char *)r.ptr + at * r.pitch * (r.dtype == SAGE_F32 ? 4 : 2);
    c.rows = count;
    return c;
}
VectorArg cut(const VectorArg &v, long long at) { return v.ptr ? VectorArg{(char *)v.ptr + at * v.stride * 4, v.stride} : v; }

// One pass over the weights for `pass` rows at most.
template <class T, bool Q>
sage_status launch_few(Context &ctx, const Head &a, long long pass, unsigned grid, float4 *parts, float *asked, const FewProbs &to) {
    ctx.note_launch(Q ? "head_few_probs" : "head_few");
    if (ctx.dry()) return SAGE_OK;
    const auto run = [&](auto kernel, int padded) {
        const size_t smem = (size_t)padded * a.hidden.cols * sizeof(T);
        sage_status s = ctx.check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024), "head_few");
        return s ? s
                 : ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), kernel, dim3(grid), dim3(256), smem, (const T *)a.hidden.ptr, a.hidden.pitch, (const T *)a.weight.ptr, a.weight.pitch, (int)a.hidden.rows,
                                                   (int)a.weight.rows, (int)a.hidden.cols, (const int *)a.ids.ptr, a.ids.stride, a.scale * kLog2E, parts, asked, to),
                                  "head_few");
    };
    if constexpr (sizeof(T) == 4)
        if (pass > 4) return run(head_few_kernel<T, 8, Q>, 8);
    return pass > 2 ? run(head_few_kernel<T, 4, Q>, 4) : pass > 1 ? run(head_few_kernel<T, 2, Q>, 2) : run(head_few_kernel<T, 1, Q>, 1);
}
unsigned few_grid(Context &ctx, long long vocab) { return (unsigned)std::min<long long>((vocab + 31) / 32, 2ll * ctx.sm_count); }

template <class T>
sage_status forward_few(Context &ctx, const Head &all, long long pass, const VectorArg &all_log_probs, const VectorArg &all_entropy, const RowsArg &all_stats) {
    for (long long at = 0; at < all.hidden.rows; at += pass) {
        Scratch scratch(ctx);
        Head a = all;
        a.hidden = cut(all.hidden, at, std::min(pass, all.hidden.rows - at));
        a.ids = cut(all.ids, at);
        const VectorArg log_probs = cut(all_log_probs, at), entropy = cut(all_entropy, at);
        const RowsArg stats = cut(all_stats, at, a.hidden.rows);
        const long long rows = a.hidden.rows, vocab = a.weight.rows;
        const unsigned grid = few_grid(ctx, vocab);
        float4 *parts = nullptr;
        float *asked = nullptr;
        sage_status st = scratch.get((size_t)(grid * rows) * 16, &parts);
        if (!st) st = scratch.get((size_t)rows * 4, &asked);
        if (!st) st = launch_few<T, false>(ctx, a, pass, grid, parts, asked, FewProbs{});
        if (!st) st = join(ctx, parts, (int)grid, rows, asked, a.ids, vocab, a.scale, Values{(float *)log_probs.ptr, (float *)entropy.ptr, (float *)stats.ptr, log_probs.stride, entropy.stride, stats.pitch});
        if (st) return st;
    }
    return SAGE_OK;
}
// q of tokens [first, first + count) for few rows, from the values' own dot products.
template <class T>
sage_status probs_few(Context &ctx, const Head &all, long long pass, long long first, long long count, FewProbs to) {
    Head a = all;
    a.weight = cut(all.weight, first, count);
    to.first = (int)first;
    for (long long at = 0; at < all.hidden.rows; at += pass) {
        a.hidden = cut(all.hidden, at, std::min(pass, all.hidden.rows - at));
        a.ids = cut(all.ids, at);
        sage_status st = launch_few<T, true>(ctx, a, pass, few_grid(ctx, count), nullptr, nullptr, to);
        if (st) return st;
        to.about += pass;
        to.gl += pass;
        to.q += pass * to.pitch;
    }
    return SAGE_OK;
}

template <class T>
sage_status forward16(Context &ctx, const Head &a, const VectorArg &log_probs, const VectorArg &entropy, const RowsArg &stats) {
    Scratch scratch(ctx);
    const long long rows = a.hidden.rows, vocab = a.weight.rows, width = a.hidden.cols;
    Matrix w;
    sage_status st = aligned<T>(ctx, scratch, a.weight, &w);
    if (st) return st;
    Product p = shape_of(ctx, rows, vocab, width);
    const long long parts_of_row = 2ll * p.tiles_n;
    const long long most = std::max<long long>(256, (long long)(kPartBytes / (16 * parts_of_row)) / 256 * 256);  // rows at a time
    float4 *parts = nullptr;
    float *asked = nullptr;
    st = scratch.get((size_t)(std::min(rows, most) * parts_of_row) * 16, &parts);
    if (!st) st = scratch.get((size_t)std::min(rows, most) * 4, &asked);
    for (long long at = 0; at < rows && !st; at += most) {
        const long long count = std::min(most, rows - at);
        Matrix x;
        st = aligned<T>(ctx, scratch, cut(a.hidden, at, count), &x);
        if (st) return st;
        p.m = (int)count;
        p.tiles_m = (int)((count + 255) / 256);
        p.band = (int)std::max<long long>(8, ((long long)48 << 20) / (256 * width * 2));  // rows of hidden states that stay in L2 while the weights go by
        const VectorArg ids = cut(a.ids, at);
        p.ids = (const int *)ids.ptr;
        p.ids_stride = ids.stride;
        p.c2 = a.scale * kLog2E;
        p.chain = logits_chain(p);
        p.parts = parts;
        p.asked = asked;
        st = launch<T, false, false, kStats>(ctx, "head_log_probs", p, a.hidden.dtype, x, w, 0, Matrix{});
        const VectorArg lp = cut(log_probs, at), h = cut(entropy, at);
        const RowsArg s = cut(stats, at, count);
        if (!st) st = join(ctx, parts, (int)parts_of_row, count, asked, ids, vocab, a.scale, Values{(float *)lp.ptr, (float *)h.ptr, (float *)s.ptr, lp.stride, h.stride, s.pitch});
    }
    return st;
}

// The rows' part of the gradient; gmax where P is stored by a scale of its own.
sage_status rows_about(Context &ctx, Scratch &scratch, const Head &a, const RowsArg &stats, const VectorArg &entropy, const VectorArg &gl, const VectorArg &ge, bool scaled, float4 **about,
                       float **gls, unsigned **gmax) {
    const long long rows = a.hidden.rows;
    sage_status st = scratch.get((size_t)rows * 16, about);
    if (!st) st = scratch.get((size_t)rows * 4, gls);
    *gmax = nullptr;
    if (!st && scaled) {
        st = scratch.get(4, gmax);
        ctx.note_memset();
        if (!st && !ctx.dry()) st = ctx.check_cuda(cudaMemsetAsync(*gmax, 0, 4, ctx.stream()), "head_log_probs_grad");
    }
    if (st) return st;
    ctx.note_launch("head_rows");
    if (ctx.dry()) return SAGE_OK;
    return ctx.check_cuda(launch_dependent(ctx.pdl && !scaled, ctx.stream(), head_rows_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, (const float *)stats.ptr,
                                           rows > 1 ? stats.pitch : 2, entropy, gl, ge, (const int *)a.ids.ptr, a.ids.stride, (int)rows, (int)a.weight.rows, *about, *gls, *gmax),
                          "head_rows");
}

template <class T>
sage_status grad16(Context &ctx, const Head &a, const RowsArg &stats, const VectorArg &entropy, const VectorArg &gl, const VectorArg &ge, const RowsArg &dhidden, const RowsArg &dweight) {
    Scratch scratch(ctx);
    const long long rows = a.hidden.rows, vocab = a.weight.rows, width = a.hidden.cols;
    const int dtype = a.hidden.dtype;
    Matrix x, w;
    float4 *about;
    float *gls;
    unsigned *gmax;
    T *probs = nullptr;
    // Pieces of equal size, whole tiles
    const long long tiles = (vocab + 255) / 256, most = std::max<long long>(1, (long long)(kPieceBytes / ((size_t)rows * 512))), pieces = (tiles + most - 1) / most,
                    piece = (tiles + pieces - 1) / pieces * 256, pitch = std::min(piece, (vocab + 63) / 64 * 64);
    sage_status st = aligned<T>(ctx, scratch, a.hidden, &x);
    if (!st) st = aligned<T>(ctx, scratch, a.weight, &w);
    if (!st) st = rows_about(ctx, scratch, a, stats, entropy, gl, ge, dtype == SAGE_F16, &about, &gls, &gmax);
    if (!st) st = scratch.get((size_t)(rows * pitch) * 2, &probs);
    const long long pass = few(a);  // rows whose values came from dot products
    Result to_hidden;
    to_hidden.out = dhidden;
    for (long long at = 0; at < vocab && !st; at += piece) {
        const long long n = std::min(piece, vocab - at);
        const bool first = at == 0, last = at + n == vocab;
        const Matrix here{(const T *)w.p + at * w.pitch, n, width, w.pitch}, q{probs, rows, n, pitch};
        Product p = shape_of(ctx, rows, n, width);
        p.ids = (const int *)a.ids.ptr;
        p.ids_stride = a.ids.stride;
        p.first = (int)at;
        p.c2 = a.scale * kLog2E;
        p.rows = about;
        p.gl = gls;
        p.gmax = gmax;
        p.chain = logits_chain(p);
        p.band = (int)std::max<long long>(8, ((long long)48 << 20) / (256 * width * 2));
        if (pass) st = probs_few<T>(ctx, a, pass, at, n, FewProbs{about, gls, gmax, 1.f, (unsigned short *)probs, pitch, 0, 0});
        else st = launch<T, false, false, kProbs>(ctx, "head_probs", p, dtype, x, here, dtype, q);
        if (!st && dhidden.ptr) {
            p = shape_of(ctx, rows, width, n);
            p.gmax = gmax;
            p.alpha = a.scale;
            if (first) plan(ctx, p, n, !last, &to_hidden);
            st = multiply<T, false, true>(ctx, scratch, "head_dhidden", p, dtype, q, here, first, last, &to_hidden);
        }
        if (!st && dweight.ptr) {
            p = shape_of(ctx, n, width, rows);
            p.gmax = gmax;
            p.alpha = a.scale;
            Scratch sums(ctx);  // of this piece alone
            Result r;
            r.out = cut(dweight, at, n);
            plan(ctx, p, rows, false, &r);
            st = multiply<T, true, true>(ctx, sums, "head_dweight", p, dtype, q, x, true, true, &r);
        }
    }
    return st;
}

// ------------------------------------------------------------------------------------------ f32
typedef __nv_bfloat16 Piece;

// The pieces of one or two operands, in planes of their own.
sage_status pieces_of(Context &ctx, Scratch &scratch, const RowsArg &r, Matrix *m, const RowsArg &r2 = RowsArg{}, Matrix *m2 = nullptr) {
    ToPieces to[2] = {};
    sage_status st = SAGE_OK;
    const RowsArg *of[2] = {&r, &r2};
    Matrix *into[2] = {m, m2};
    for (int i = 0; i < 2 && into[i] && !st; ++i) {
        const RowsArg &x = *of[i];
        const long long pitch = (x.cols + 7) / 8 * 8, px = x.rows > 1 ? x.pitch : x.cols;
        st = scratch.get((size_t)(3 * x.rows * pitch) * 2, &to[i].y);
        *into[i] = Matrix{to[i].y, x.rows, x.cols, pitch, x.rows * pitch};
        to[i] = ToPieces{(const float *)x.ptr, to[i].y, px, pitch, x.rows * pitch, x.rows * (pitch / 8), (int)x.cols, x.cols % 8 == 0 && on_16(x.ptr, px, 4)};
    }
    if (st) return st;
    ctx.note_launch("head_pieces");
    if (ctx.dry()) return SAGE_OK;
    const long long blocks = std::min<long long>((to[0].groups + to[1].groups + 255) / 256, ctx.sm_count * 16ll);
    return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), head_pieces_kernel, dim3((unsigned)blocks), dim3(256), 0, to[0], to[1]), "head_pieces");
}

sage_status forward32(Context &ctx, const Head &a, const VectorArg &log_probs, const VectorArg &entropy, const RowsArg &stats) {
    Scratch scratch(ctx);
    const long long rows = a.hidden.rows, vocab = a.weight.rows, width = a.hidden.cols;
    Product p = shape_of(ctx, rows, vocab, width);
    const long long parts_of_row = 2ll * p.tiles_n, most = std::max<long long>(256, (long long)(kPartBytes / (16 * parts_of_row)) / 256 * 256);  // rows at a time
    Matrix x, w;
    sage_status st = rows <= most ? pieces_of(ctx, scratch, a.weight, &w, a.hidden, &x) : pieces_of(ctx, scratch, a.weight, &w);
    if (!st) st = scratch.get((size_t)(std::min(rows, most) * parts_of_row) * 16, &p.parts);
    if (!st) st = scratch.get((size_t)std::min(rows, most) * 4, &p.asked);
    p.c2 = a.scale * kLog2E;
    p.ids_stride = a.ids.stride;
    for (long long at = 0; at < rows && !st; at += most) {
        const long long count = std::min(most, rows - at);
        const VectorArg ids = cut(a.ids, at), lp = cut(log_probs, at), h = cut(entropy, at);
        const RowsArg s = cut(stats, at, count);
        if (rows > most) st = pieces_of(ctx, scratch, cut(a.hidden, at, count), &x);
        p.m = (int)count;
        p.tiles_m = (int)((count + 255) / 256);
        p.band = (int)std::max<long long>(8, ((long long)48 << 20) / (256 * width * 6));
        p.ids = (const int *)ids.ptr;
        if (!st) st = launch<Piece, false, false, kStats, true>(ctx, "head_log_probs", p, SAGE_BF16, x, w, 0, Matrix{});
        if (!st) st = join(ctx, p.parts, (int)parts_of_row, count, p.asked, ids, vocab, a.scale, Values{(float *)lp.ptr, (float *)h.ptr, (float *)s.ptr, lp.stride, h.stride, s.pitch});
    }
    return st;
}

sage_status grad32(Context &ctx, const Head &a, const RowsArg &stats, const VectorArg &entropy, const VectorArg &gl, const VectorArg &ge, const RowsArg &dhidden, const RowsArg &dweight) {
    Scratch scratch(ctx);
    const long long rows = a.hidden.rows, vocab = a.weight.rows, width = a.hidden.cols, padded = (rows + 255) / 256 * 256;
    const long long tiles = (vocab + 255) / 256, most = std::max<long long>(1, (long long)(kPieceBytes / ((size_t)padded * 512 * 3))), pieces = (tiles + most - 1) / most, piece = (tiles + pieces - 1) / pieces * 256,
                    pitch = std::min(piece, (vocab + 63) / 64 * 64);
    float4 *about;
    float *gls;
    unsigned *gmax;
    Piece *probs = nullptr;
    Matrix x, w;
    sage_status st = pieces_of(ctx, scratch, a.hidden, &x, a.weight, &w);
    if (!st) st = rows_about(ctx, scratch, a, stats, entropy, gl, ge, false, &about, &gls, &gmax);
    if (!st) st = scratch.get((size_t)(3 * padded * pitch) * 2, &probs);
    const long long pass = few(a);  // rows whose values came from dot products
    Result to_hidden;
    to_hidden.out = dhidden;
    for (long long at = 0; at < vocab && !st; at += piece) {
        const long long n = std::min(piece, vocab - at);
        const bool first = at == 0, last = at + n == vocab;
        const Matrix here{(const Piece *)w.p + at * w.pitch, n, width, w.pitch, w.plane}, q{probs, rows, n, pitch, padded * pitch};
        Product p = shape_of(ctx, rows, n, width);
        p.ids = (const int *)a.ids.ptr;
        p.ids_stride = a.ids.stride;
        p.first = (int)at;
        p.c2 = a.scale * kLog2E;
        p.rows = about;
        p.gl = gls;
        p.band = (int)std::max<long long>(8, ((long long)48 << 20) / (256 * width * 6));
        p.slice_rows = (int)padded;  // of a plane
        p.alpha = a.scale;
        if (pass) st = probs_few<float>(ctx, a, pass, at, n, FewProbs{about, gls, nullptr, a.scale, (unsigned short *)probs, pitch, padded * pitch, 0});
        else st = launch<Piece, false, false, kProbs, true>(ctx, "head_probs", p, SAGE_BF16, x, here, SAGE_BF16, Matrix{probs, 3 * padded, n, pitch});
        if (!st && dhidden.ptr) {
            p = shape_of(ctx, rows, width, n);
            if (first) plan(ctx, p, n, !last, &to_hidden);
            st = multiply<Piece, false, true, true>(ctx, scratch, "head_dhidden", p, SAGE_BF16, q, here, first, last, &to_hidden);
        }
        if (!st && dweight.ptr) {
            p = shape_of(ctx, n, width, rows);
            Scratch sums(ctx);  // of this piece alone
            Result r;
            r.out = cut(dweight, at, n);
            plan(ctx, p, rows, false, &r);
            st = multiply<Piece, true, true, true>(ctx, sums, "head_dweight", p, SAGE_BF16, q, x, true, true, &r);
        }
    }
    return st;
}

}  // namespace
}  // namespace head

sage_status head_log_probs(Context &ctx, const Head &a, const VectorArg &log_probs, const VectorArg &entropy, const RowsArg &stats) {
    if (!a.hidden.rows) return SAGE_OK;
    if (const long long pass = head::few(a))
        return with_type(a.hidden.dtype, [&](auto t) { return head::forward_few<decltype(t)>(ctx, a, pass, log_probs, entropy, stats); });
    if (a.hidden.dtype == SAGE_F32) return head::forward32(ctx, a, log_probs, entropy, stats);
    return a.hidden.dtype == SAGE_F16 ? head::forward16<__half>(ctx, a, log_probs, entropy, stats) : head::forward16<__nv_bfloat16>(ctx, a, log_probs, entropy, stats);
}

sage_status head_log_probs_grad(Context &ctx, const Head &a, const RowsArg &stats, const VectorArg &entropy, const VectorArg &g_log_probs, const VectorArg &g_entropy, const RowsArg &dhidden,
                                const RowsArg &dweight) {
    RowsArg dh = dhidden, dw = dweight;
    if (dh.rows <= 1) dh.pitch = (dh.cols + 7) / 8 * 8;
    if (dw.rows <= 1) dw.pitch = (dw.cols + 7) / 8 * 8;
    if (!a.hidden.rows) {
        if (!dw.ptr) return SAGE_OK;
        ctx.note_memset();
        const size_t size = dw.dtype == SAGE_F32 ? 4 : 2;
        return ctx.dry() ? SAGE_OK : ctx.check_cuda(cudaMemset2DAsync(dw.ptr, dw.pitch * size, 0, dw.cols * size, (size_t)dw.rows, ctx.stream()), "head_log_probs_grad");
    }
    if (a.hidden.dtype == SAGE_F32) return head::grad32(ctx, a, stats, entropy, g_log_probs, g_entropy, dh, dw);
    if (a.hidden.dtype == SAGE_F16) return head::grad16<__half>(ctx, a, stats, entropy, g_log_probs, g_entropy, dh, dw);
    return head::grad16<__nv_bfloat16>(ctx, a, stats, entropy, g_log_probs, g_entropy, dh, dw);
}

}  // namespace k
}  // namespace sage
