// Dropout whose mask is drawn from each element's position and never stored: y_i = x_i 65536 / (65536 - bar) where element i stays, else 0
// (counter_random.h says which stay).  Its gradient is the same map of the gradient that arrives.
//
// Bound by memory: an element is read and written once; a draw of 60 integer instructions serves eight of them.  A thread takes one block of
// eight elements, whatever the layout: as vectors where rows keep blocks whole and on 16-byte boundaries, element by element elsewhere.
#include <algorithm>

#include "counter_random.h"
#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {
namespace {

struct DropoutArgs {
    const void *x;
    void *y;
    long long n, cols, px, py;  // elements; of a row (n: one row)
    Dropout d;
};

constexpr int kThreads = 256;

template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropoutArgs a) {
    grid_dependency_sync();
    const Key key = key_of(a.d);
    const long long block = (long long)blockIdx.x * kThreads + threadIdx.x, first = 8 * block;
    if (first >= a.n) return;
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    if (WIDE && first + 8 <= a.n) {
        const long long row = a.cols == a.n ? 0 : a.n <= 0xffffffffll ? (unsigned)first / (unsigned)a.cols : first / a.cols, col = first - row * a.cols;
        constexpr int N = Pack<T>::N, P = 8 / N;
        Pack<T> p[P];
#pragma unroll
        for (int i = 0; i < P; ++i) p[i] = *(const Pack<T> *)(x + row * a.px + col + i * N);
        const unsigned keep = a.d.bar ? keep8(a.d, key, block) : 0xffu;
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int e = 0; e < N; ++e) p[i].v[e] = narrowed<T>(keep >> (i * N + e) & 1u ? widen(p[i].v[e]) * a.d.factor : 0.f);
            *(Pack<T> *)(y + row * a.py + col + i * N) = p[i];
        }
    } else {
        const unsigned keep = a.d.bar ? keep8(a.d, key, block) : 0xffu;
        long long row = first / a.cols, col = first - row * a.cols;
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
    const long long size = x.dtype == SAGE_F32 ? 4 : 2, blocks = (a.n + 8 * kThreads - 1) / (8 * kThreads);
    if (blocks > 0x7fffffffll) return ctx.fail(SAGE_ERR_INVALID, "dropout: more than 2^42 elements");
    const bool one = a.cols == a.n;
    const bool wide = (uintptr_t)x.ptr % 16 == 0 && (uintptr_t)y.ptr % 16 == 0 && (one || (a.cols % 8 == 0 && x.pitch * size % 16 == 0 && y.pitch * size % 16 == 0));
    ctx.note_launch("dropout");
    if (ctx.dry()) return SAGE_OK;
    return with_type(x.dtype, [&](auto t) {
        typedef decltype(t) T;
        return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), wide ? dropout_kernel<T, true> : dropout_kernel<T, false>, dim3((unsigned)blocks), dim3(kThreads), 0, a), "dropout");
    });
}

}  // namespace k
}  // namespace sage
