// The products of log probabilities straight from hidden states (head.cu): C = A B^T of 16-bit operands on the tensor cores, f32 sums, with what
// becomes of a tile done while the next one is multiplied.
//
// Two CTAs work on one tile of 256 rows and BN columns (cta_group::2): each loads its 128 rows of A and its half of B's rows, 64 k at a time,
// through a ring of TMA stages; the first of them issues the MMAs, whose sums lie 128 rows to a CTA in tensor memory, two tiles' worth, so that
// eight warps finish a tile while the next one's sums are made: the tensor pipe is 88-94 % busy (8192 x 50021 x 2048 bf16, values 1163-1210 us, 1390-1440 TFLOP/s, where a
// plain product of the library reaches 1376 for seconds on end).  Either operand may be stored with K or with its rows contiguous.
//
// f32 operands (F32), with f32's accuracy: every element is the sum of three bf16 numbers, x = x0 + x1 + x2 (8 bits each, to nearest, 24 in all; what
// rounds to a finite bf16, 3.39e38 at most), which lie in three planes, and of the nine products of pieces the six that reach 2^-24 of the result are made,
//   x2 y0 + x0 y2 + x1 y1 + x1 y0 + x0 y1 + x0 y0,
// in this order for each 64 k, so that the tensor cores, which cut what lies below the last place of a sum, add the small ones to small sums; the sum of
// each 64 k is then added to registers, to nearest.  (Two f16 pieces would need three products, but a scale for each row, and what is far below a row's
// largest would lose bits: the gradient of rare tokens is.  Pieces made inside the product, tile by tile, from f32 operands: 640 x 30522 x 768, values and
// gradient, 1015 us.)
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "gemm_tc_device.inc"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {
namespace head {

using namespace sage_tc;

constexpr int kK = 64;                  // k of a stage: rows of 128 bytes
constexpr int kStages = 6;
constexpr int kEndWarps = 8;
constexpr int kBlock = 64 + 32 * kEndWarps;
constexpr int kOperandBytes = 128 * kK * 2;  // of a CTA and stage; B's may be half of that
constexpr int kStageSize = 2 * kOperandBytes;
constexpr int kOutBytes = 4096;         // 32 rows of 128 bytes for each warp's stores
constexpr size_t kSmem = (size_t)kStages * kStageSize + kEndWarps * kOutBytes + 1024;

enum End {
    kStats,   // of each row and half a tile's columns: largest, sum of exponentials, sum of those times their exponents; the asked-for logit
    kProbs,   // the gradient with respect to the product, 16 bits
    kNarrow,  // alpha times the product, 16 bits
    kWide     // ... in f32, stored or added to what is there
};

struct Product {
    int m, n, k;
    int bn;                       // 256 or 128
    int tiles_m, tiles_n, slices; // slices of K, each a result of its own: `slice_rows` rows further
    int slice_blocks, slice_rows; // K-blocks of a slice
    int chain;                    // K-blocks that the tensor cores add up
    int band;                     // row tiles that column tiles are gone through for
    unsigned *status;
    const int *ids;
    long long ids_stride;
    int first;                    // column n stands for token first + n
    float c2;                     // kStats, kProbs: scale * log2(e)
    float4 *parts;                // kStats: [half tile][m] {largest, sum, sum of products, -}
    float *asked;                 // ... [m]
    const float4 *rows;           // kProbs: [m] {largest, -log2 sum, -(gl + ge H), -ge ln 2}
    const float *gl;              // ... [m]
    const unsigned *gmax;         // f16: the bits of the largest |gl| + |ge| (H + 1/2), for the scale that P is stored with; null: 1
    float alpha;                  // kNarrow, kWide: of the product (f32 operands: kProbs)
    int add;                      // kWide
};

// What P is multiplied by so that its largest possible value is near 2^14: f16 then holds 2^-28 of that as normal numbers.
__device__ __forceinline__ int stored_exponent(const unsigned *gmax) {
    const unsigned e = __ldg(gmax) >> 23;  // of a magnitude below 2^(e - 126)
    return e == 0u || e >= 255u ? 0 : min(126, max(-126, 14 - ((int)e - 126)));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

__device__ __forceinline__ void load_3d_pair(void *dst, const CUtensorMap *map, unsigned bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x),
                 "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap *map, const void *src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void add_2d(const CUtensorMap *map, const void *src, int x, int y) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void mma_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld32(unsigned at, float (&v)[32]) {
    unsigned r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
                   "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kFar = -1000.f;  // an exponent whose power is zero, and whose product with that is too

struct Tile {
    int m0, n0, slice;
};
__device__ __forceinline__ Tile tile_of(const Product &p, int index) {
    const int per = p.tiles_m * p.tiles_n, slice = index / per;
    int r = index - slice * per;
    const int band = r / (p.band * p.tiles_n), height = min(p.band, p.tiles_m - band * p.band);
    r -= band * p.band * p.tiles_n;
    const int n = r / height;
    return Tile{(band * p.band + r - n * height) * 256, n * p.bn, slice};
}

// One operand's rows of a stage: with K contiguous one box of 64 k, otherwise a box of 64 k for every 64 rows.
template <bool MN>
__device__ __forceinline__ void load_rows(char *to, const CUtensorMap *map, unsigned bar, int row, int rows, int k, int plane) {
    if (MN)
        for (int i = 0; i < rows; i += 64) load_3d_pair(to + i * (kK * 2), map, bar, row + i, k, plane);
    else
        load_3d_pair(to, map, bar, k, row, plane);
}
constexpr int kProducts = 6;  // of pieces, for each 64 k of f32 operands

// A warp's 32 rows of 128 bytes as TMA's 128-byte swizzle has them: 16-byte chunk c of row r lies at chunk c ^ (r % 8).
__device__ __forceinline__ void put_chunk(char *out, int row, int chunk, uint4 v) { *(uint4 *)(out + row * 128 + ((chunk ^ (row & 7)) << 4)) = v; }

// ... 32 rows of 64 bytes, its 64-byte swizzle: chunk c of row r at c ^ (r / 2 % 4).
__device__ __forceinline__ void put_chunk64(char *out, int row, int chunk, uint4 v) { *(uint4 *)(out + row * 64 + ((chunk ^ (row >> 1 & 3)) << 4)) = v; }

template <class T>
__device__ __forceinline__ unsigned pair16(float a, float b);
template <>
__device__ __forceinline__ unsigned pair16<__nv_bfloat16>(float a, float b) {
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <>
__device__ __forceinline__ unsigned pair16<__half>(float a, float b) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// The largest bf16 piece of each of two numbers, which keep the rest.  (An infinity is its first piece alone: what is left of it is not a number.)
__device__ __forceinline__ unsigned take_piece(float &a, float &b) {
    const unsigned w = pair16<__nv_bfloat16>(a, b);
    const float x = __uint_as_float(w << 16), y = __uint_as_float(w & 0xffff0000u);
    a = fabsf(x) < INFINITY ? a - x : x == x ? 0.f : x;
    b = fabsf(y) < INFINITY ? b - y : y == y ? 0.f : y;
    return w;
}

// What a row's 32 * count columns from col0 on come to: largest, sum of exponentials, sum of those times their exponents; the asked-for logit where it is here.
template <int N>
__device__ __forceinline__ float4 stats_of(const Product &p, float (&acc)[N][32], int count, int col0, int id, int row) {
    float largest = -INFINITY, sum = 0.f, along = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (j >= count) break;
        const int col = col0 + j * 32;
        if (col + 32 > p.n) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (col + e >= p.n) acc[j][e] = -INFINITY;
        }
        float high = acc[j][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) high = fmaxf(high, acc[j][e]);
        if (high > largest) {  // what there is so far, seen from the new largest
            const float by = largest == -INFINITY ? 0.f : (largest - high) * p.c2, f = largest == -INFINITY ? 0.f : exp2_fast(by);
            along = f > 0.f ? fmaf(sum * f, by, along * f) : 0.f;
            sum *= f;
            largest = high;
        }
        const float from = largest == -INFINITY ? 0.f : largest;
        float s[4] = {0.f, 0.f, 0.f, 0.f}, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const float d = (acc[j][e] - from) * p.c2, x = exp2_fast(d);
            s[e & 3] += x;
            a[e & 3] = fmaf(x, fmaxf(d, kFar), a[e & 3]);
        }
        sum += (s[0] + s[1]) + (s[2] + s[3]);
        along += (a[0] + a[1]) + (a[2] + a[3]);
        const int want = id - col;
        if (__any_sync(0xffffffffu, want >= 0 && want < 32)) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) x = e == want ? acc[j][e] : x;
            if (want >= 0 && want < 32 && col + want < p.n) p.asked[row] = x;
        }
    }
    return make_float4(largest, sum, along, 0.f);
}
// d / d logits of 32 columns, in place of the logits.
__device__ __forceinline__ void probs_of(const Product &p, float (&v)[32], const float4 &about, int want, int row, bool there, float factor) {
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const float d = fmaf(v[e] - about.x, p.c2, about.y), x = exp2_fast(d);
        v[e] = x * fmaf(about.w, fmaxf(d, kFar), about.z);
    }
    if (__any_sync(0xffffffffu, want >= 0 && want < 32)) {
        const float gl = there ? __ldg(p.gl + row) * factor : 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] += e == want ? gl : 0.f;
    }
}

template <class T, bool A_MN, bool B_MN, End END, bool F32>
__global__ void __launch_bounds__(kBlock, 1)
head_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c, const Product p) {
    extern __shared__ __align__(1024) char smem_raw[];
    __shared__ __align__(8) unsigned long long full[kStages], empty[kStages], done[2], freed[2];
    __shared__ unsigned tmem_slot;
    __shared__ volatile int given_up;
    char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = __shfl_sync(0xffffffffu, (int)cluster_rank(), 0), pair = (int)blockIdx.x / 2, pairs = (int)gridDim.x / 2;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&done[b], 1);
            mbar_init(&freed[b], 2 * kEndWarps);  // the leader's: both CTAs' warps
        }
        given_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_slot;  // all of the columns: the same in both CTAs
    grid_dependency_sync();
    const auto give_up = [&](unsigned where) {
        atomicOr(p.status, 0x100u | where);
        given_up = 1;
    };
    const int all = p.tiles_m * p.tiles_n * p.slices, all_blocks = (p.k + kK - 1) / kK * (F32 ? kProducts : 1), half = p.bn / 2;

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        int i = 0;
        bool live = true;
        for (int t = pair; t < all && live && !__any_sync(0xffffffffu, given_up != 0); t += pairs) {
            const Tile tile = tile_of(p, t);
            const int first = tile.slice * p.slice_blocks, last = min(all_blocks, first + p.slice_blocks);
            for (int b = first; b < last; ++b, ++i) {
                const int s = i % kStages;
                if (!mbar_wait_warp(&empty[s], ((i / kStages) & 1) ^ 1)) {
                    if (lane == 0) give_up(1);
                    live = false;
                    break;
                }
                char *to = smem + s * kStageSize;
                const unsigned bar = peer_addr(smem_u32(&full[s]), 0);
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(&full[s], (unsigned)(2 * (128 + half) * kK * 2));
                    const int k = (F32 ? b / kProducts : b) * kK, n = F32 ? b % kProducts : 0;
                    load_rows<A_MN>(to, &map_a, bar, tile.m0 + rank * 128, 128, k, F32 ? (0x001102 >> 4 * n) & 3 : 0);  // 2 0 1 1 0 0
                    load_rows<B_MN>(to + kOperandBytes, &map_b, bar, tile.n0 + rank * half, half, k, F32 ? (0x010120 >> 4 * n) & 3 : 0);  // 0 2 1 0 1 0
                }
                __syncwarp();
            }
        }
        // Copies have landed before the CTA leaves: the leader sees its barriers complete, the other its stages released.
        for (int j = i > kStages ? i - kStages : 0; j < i; ++j)
            if (!mbar_wait_warp(rank == 0 ? &full[j % kStages] : &empty[j % kStages], (j / kStages) & 1) && lane == 0) give_up(2);
    } else if (warp == 1 && rank == 0) {
        // ------------------------------------------------------------------ products
        // D f32, A and B bf16 (1) or f16 (0), which of them have their rows contiguous, N / 8, M / 16
        constexpr unsigned type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const unsigned idesc = (1u << 4) | (type << 7) | (type << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((unsigned)(p.bn >> 3) << 17) | ((256u >> 4) << 24);
        // K contiguous: rows of 128 bytes, eight of them 1024 bytes apart, 16 k are 32 bytes on.  Rows contiguous: k-rows of 64 operand rows, groups
        // of eight k 1024 bytes apart, the next 64 operand rows behind the stage's 64 k, 16 k are 2048 bytes on.
        const unsigned long long desc_a = smem_desc(0u, A_MN ? kK * 128u : 16u, 1024u, 2u), desc_b = smem_desc(0u, B_MN ? kK * 128u : 16u, 1024u, 2u);
        constexpr unsigned kStepA = A_MN ? 128u : 2u, kStepB = B_MN ? 128u : 2u;
        const unsigned base = smem_u32(smem);
        int i = 0, chains = 0;
        bool live = !__any_sync(0xffffffffu, given_up != 0);
        for (int t = pair; t < all && live; t += pairs) {
            const int slice = t / (p.tiles_m * p.tiles_n), first = slice * p.slice_blocks, last = min(all_blocks, first + p.slice_blocks);
            for (int from = first; from < last && live; from += p.chain, ++chains) {
                const int buffer = chains & 1, to = min(last, from + p.chain);
                if (!mbar_wait_warp(&freed[buffer], ((chains >> 1) & 1) ^ 1)) {
                    if (lane == 0) give_up(16);
                    live = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned d = tmem + (unsigned)buffer * 256u;
                for (int b = from; b < to; ++b, ++i) {
                    const int s = i % kStages;
                    if (!mbar_wait_warp(&full[s], (i / kStages) & 1)) {
                        if (lane == 0 && !given_up) give_up(4);
                        live = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned at = base + (unsigned)(s * kStageSize);
                    const unsigned long long a = desc_a + (at >> 4), bb = desc_b + ((at + kOperandBytes) >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kK / 16; ++k) mma_pair(d, a + k * kStepA, bb + k * kStepB, idesc, b > from || k > 0 ? 1u : 0u);
                        umma_commit_pair(&empty[s]);
                        if (b + 1 == to) umma_commit_pair(&done[buffer]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------------ what becomes of a tile
        const int quarter = warp & 3, side = (warp - 2) >> 2;  // a warp reaches the 32 rows of tensor memory that its number gives
        char *out = smem + kStages * kStageSize + (warp - 2) * kOutBytes;
        float factor = 1.f;
        if (END == kProbs) factor = F32 ? p.alpha : p.gmax ? power_of_two(stored_exponent(p.gmax)) : 1.f;  // (the products of f32 operands have no scale: q has it)
        if (END == kNarrow || END == kWide) factor = p.gmax ? p.alpha * power_of_two(-stored_exponent(p.gmax)) : p.alpha;
        int chains = 0;
        bool live = true;
        // Waits for a chain's sums; gives their tensor memory back.
        const auto arrived = [&]() {
            if (!mbar_wait_warp(&done[chains & 1], (chains >> 1) & 1)) {
                if (lane == 0 && !given_up) give_up(8);
                live = false;
                return 0u;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)((chains & 1) * 256 + side * half);
        };
        const auto drained = [&]() {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(&freed[chains & 1]);
                else mbar_arrive_remote_tmem(peer_addr(smem_u32(&freed[chains & 1]), 0));
            }
            ++chains;
        };
        for (int t = pair; t < all && live; t += pairs) {
            const Tile tile = tile_of(p, t);
            const int row0 = tile.m0 + rank * 128 + quarter * 32, row = row0 + lane, col0 = tile.n0 + side * half;
            const bool there = row < p.m;
            int id = -1;
            if ((END == kStats || END == kProbs) && there) {
                id = __ldg(p.ids + row * p.ids_stride);
                id = id < p.first ? -1 : id - p.first;
            }
            if constexpr (END == kStats || END == kProbs || F32) {
                // The tensor cores cut what lies below a sum's last place at every addition: log probabilities of 4096 k in one chain were 4e-6 off.
                // Chains of 512 k at most are added up here, to nearest; the gradient's in the same chains as the values', so that its logits are theirs
                // to the bit and a row's probabilities come from the logits that its sum was made of.
                float acc[4][32];
#pragma unroll
                for (int e = 0; e < 128; ++e) acc[e / 32][e % 32] = 0.f;
                const int first = tile.slice * p.slice_blocks, last = min(all_blocks, first + p.slice_blocks);
#pragma unroll 1
                for (int from = first; from < last && live; from += p.chain) {
                    const unsigned at = arrived();
                    if (!live) break;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j * 32 < half) {
                            float v[32];
                            tmem_ld32(at + j * 32, v);
#pragma unroll
                            for (int e = 0; e < 32; ++e) acc[j][e] += v[e];
                        }
                    drained();
                }
                if (!live) break;
                if constexpr (END == kStats) {
                    const float4 found = stats_of(p, acc, half / 32, col0, id, row);
                    if (there) p.parts[(long long)(tile.n0 / half + side) * p.m + row] = found;
                } else {
                    float4 about = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (END == kProbs && there) {
                        about = __ldg(p.rows + row);
                        about.z *= factor, about.w *= factor;
                    }
                    // 32 columns at a time: the sums as they are, or q in three planes
                    const auto open = [&]() {  // the warp's last store has been read
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                    };
                    const auto close = [&](int col, int y) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (row0 < p.m && col < p.n && elect_one()) {
                            if (END == kWide && p.add) add_2d(&map_c, out, col, y);
                            else store_2d(&map_c, out, col, y);
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                        __syncwarp();
                    };
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j * 32 < half) {
                            const int col = col0 + j * 32;
                            if constexpr (END == kProbs && !F32) {  // 64 columns to a store of 128 bytes
                                probs_of(p, acc[j], about, id - col, row, there, factor);
                                if (j % 2 == 0) open();
#pragma unroll
                                for (int c = 0; c < 4; ++c)
                                    put_chunk(out, lane, 4 * (j % 2) + c, make_uint4(pair16<T>(acc[j][8 * c], acc[j][8 * c + 1]), pair16<T>(acc[j][8 * c + 2], acc[j][8 * c + 3]),
                                                                                     pair16<T>(acc[j][8 * c + 4], acc[j][8 * c + 5]), pair16<T>(acc[j][8 * c + 6], acc[j][8 * c + 7])));
                                if (j % 2) close(col - 32, row0);
                            } else if constexpr (END == kProbs) {
                                probs_of(p, acc[j], about, id - col, row, there, factor);
#pragma unroll 1
                                for (int n = 0; n < 3; ++n) {
                                    open();
#pragma unroll
                                    for (int c = 0; c < 4; ++c)
                                        put_chunk64(out, lane, c, make_uint4(take_piece(acc[j][8 * c], acc[j][8 * c + 1]), take_piece(acc[j][8 * c + 2], acc[j][8 * c + 3]),
                                                                             take_piece(acc[j][8 * c + 4], acc[j][8 * c + 5]), take_piece(acc[j][8 * c + 6], acc[j][8 * c + 7])));
                                    close(col, row0 + n * p.slice_rows);
                                }
                            } else {
                                open();
#pragma unroll
                                for (int c = 0; c < 8; ++c)
                                    put_chunk(out, lane, c, make_uint4(__float_as_uint(acc[j][4 * c]), __float_as_uint(acc[j][4 * c + 1]), __float_as_uint(acc[j][4 * c + 2]), __float_as_uint(acc[j][4 * c + 3])));
                                close(col, row0 + tile.slice * p.slice_rows);
                            }
                        }
                }
            } else {
                const unsigned at = arrived();
                if (!live) break;
                for (int j = 0; j < half; j += 32) {
                    float v[32];
                    tmem_ld32(at + j, v);
                    const int col = col0 + j;
                    constexpr int kPer = END == kWide ? 1 : 2;  // loads of 32 columns to a store of 128 bytes
                    const int part = (j / 32) % kPer;
                    if (part == 0) {  // the warp's last store has been read
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                    }
                    if (END == kWide) {
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            put_chunk(out, lane, c, make_uint4(__float_as_uint(v[4 * c] * factor), __float_as_uint(v[4 * c + 1] * factor), __float_as_uint(v[4 * c + 2] * factor), __float_as_uint(v[4 * c + 3] * factor)));
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            put_chunk(out, lane, 4 * part + c,
                                      make_uint4(pair16<T>(v[8 * c] * factor, v[8 * c + 1] * factor), pair16<T>(v[8 * c + 2] * factor, v[8 * c + 3] * factor), pair16<T>(v[8 * c + 4] * factor, v[8 * c + 5] * factor),
                                                 pair16<T>(v[8 * c + 6] * factor, v[8 * c + 7] * factor)));
                    }
                    if (part == kPer - 1) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        const int x = col - 32 * (kPer - 1), y = row0 + tile.slice * p.slice_rows;
                        if (row0 < p.m && x < p.n && elect_one()) {
                            if (END == kWide && p.add) add_2d(&map_c, out, x, y);
                            else store_2d(&map_c, out, x, y);
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                        __syncwarp();
                    }
                }
                drained();
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves, or gives tensor memory back, while the other may still touch it
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace head
}  // namespace k
}  // namespace sage
