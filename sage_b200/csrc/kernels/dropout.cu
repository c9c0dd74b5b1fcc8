// Dropout whose mask is drawn from each element's position and never stored: y_i = x_i 65536 / (65536 - bar) where element i stays, else 0
// (counter_random.h says which stay).  Its gradient is the same map of the gradient that arrives.
//
// Bound by memory, nearly as much by instructions: an element is read and written once, a draw of 40 instructions (two products and two exclusive ors a round; the keys' sums are made
// once for a warp) serves eight of them (16384 x 4096 bf16 46-49 us, 5.5-5.8 TB/s, 69 % of the issue slots; one block to a thread 63).  A thread takes blocks of
// eight elements, whatever the layout: as vectors where rows keep blocks whole and on 32-byte (16 bits: 16-byte) boundaries, element by element elsewhere.
#include <algorithm>

#include "counter_random.h"
#include "eight.h"
#include "language.h"
#include "launch.h"

namespace sage {
namespace k {
namespace {

struct DropoutArgs {
    const void *x;
    void *y;
    long long n, cols, px, py;  // elements; of a row (n: one row)
    Dropout d;
};

constexpr int kThreads = 256, kBlocks = 2;  // of a CTA; blocks of eight elements to a thread

template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropoutArgs a) {
    grid_dependency_sync();
    const Key key = key_of(a.d);
    const long long block0 = (long long)blockIdx.x * (kThreads * kBlocks) + threadIdx.x;
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const auto row_of = [&](long long i) { return a.cols == a.n ? 0 : a.n <= 0xffffffffll ? (long long)((unsigned)i / (unsigned)a.cols) : i / a.cols; };
    if (WIDE && 8 * (block0 + (kBlocks - 1) * kThreads) + 8 <= a.n) {  // whole blocks, all of them asked for at once
        Eight<T> v[kBlocks];
        long long to[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const long long first = 8 * (block0 + b * kThreads), row = row_of(first), col = first - row * a.cols;
            v[b].load((const char *)(x + row * a.px + col));
            to[b] = row * a.py + col;
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            float2 f[4];
            v[b].open(f);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = mul2(f[i], both(a.d.factor));
            if (a.d.bar) drop8(f, philox(key, block0 + b * kThreads, a.d.site), a.d.bar);
            v[b].close(f);
            v[b].store((char *)(y + to[b]));
        }
        return;
    }
    for (int b = 0; b < kBlocks; ++b) {
        const long long block = block0 + b * kThreads, first = 8 * block;
        if (first >= a.n) return;
        const unsigned keep = a.d.bar ? keep8(a.d, key, block) : 0xffu;
        long long row = row_of(first), col = first - row * a.cols;
        const int count = (int)min(8ll, a.n - first);
        for (int e = 0; e < count; ++e) {
            y[row * a.py + col] = narrowed<T>(keep >> e & 1u ? widen(x[row * a.px + col]) * a.d.factor : 0.f);
            if (++col == a.cols) {
                col = 0;
                ++row;
            }
        }
    }
}

}  // namespace

sage_status dropout(Context &ctx, const RowsArg &x, const RowsArg &y, const Dropout &d) {
    if (!x.rows || !x.cols) return SAGE_OK;
    DropoutArgs a{x.ptr, y.ptr, x.rows * x.cols, x.cols, x.pitch, y.pitch, d};
    if (x.rows == 1 || (x.pitch == x.cols && y.pitch == x.cols)) a.cols = a.n;
    const long long size = x.dtype == SAGE_F32 ? 4 : 2, blocks = (a.n + 8 * kThreads * kBlocks - 1) / (8 * kThreads * kBlocks);
    if (blocks > 0x7fffffffll) return ctx.fail(SAGE_ERR_INVALID, "dropout: more than 2^43 elements");
    const bool one = a.cols == a.n;
    const bool wide = (uintptr_t)x.ptr % (8 * size) == 0 && (uintptr_t)y.ptr % (8 * size) == 0 && (one || (a.cols % 8 == 0 && x.pitch % 8 == 0 && y.pitch % 8 == 0));  // eight elements in one access
    ctx.note_launch("dropout");
    if (ctx.dry()) return SAGE_OK;
    return with_type(x.dtype, [&](auto t) {
        typedef decltype(t) T;
        return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? dropout_kernel<T, true> : dropout_kernel<T, false>, dim3((unsigned)blocks), dim3(kThreads), 0, a), "dropout");
    });
}

}  // namespace k
}  // namespace sage
