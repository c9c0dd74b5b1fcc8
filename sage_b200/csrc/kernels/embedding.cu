// Token embedding: y[t, :] = scale * table[ids[t], :], and its gradient by table rows.
#include <cuda_runtime.h>

#include "language.h"
#include "launch.h"
#include "narrow.h"

namespace sage {
namespace k {

namespace {

template <class T, class Y>
__global__ void __launch_bounds__(256) embedding_kernel(const T *__restrict__ table, long long vocab, long long ld, const int *__restrict__ ids, long long ids_stride, float scale, Y *__restrict__ y,
                                                        long long ldy, long long tokens, long long dim) {
    grid_dependency_sync();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < tokens * dim; i += (long long)gridDim.x * 256) {
        const long long t = i / dim, c = i - t * dim;
        const int id = ids[t * ids_stride];
        const bool some = id >= 0 && id < vocab;
        y[t * ldy + c] = narrowed<Y>(some ? widen(table[id * ld + c]) * scale : 0.f);
    }
}

// One block sums one row of the table, over the tokens in their order.
template <class T>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const T *__restrict__ g, long long ldg, const int *__restrict__ ids, long long ids_stride, float scale, int add, float *dtable, long long ld,
                                                             long long tokens, long long dim) {
    grid_dependency_sync();
    const long long v = blockIdx.x;
    for (long long c = threadIdx.x; c < dim; c += 256) {
        float s = 0.f;
        for (long long t = 0; t < tokens; ++t)
            if (ids[t * ids_stride] == v) s += widen(g[t * ldg + c]);
        s *= scale;
        dtable[v * ld + c] = add ? dtable[v * ld + c] + s : s;
    }
}

}  // namespace

sage_status embedding(Context &ctx, const RowsArg &table, const VectorArg &ids, float scale, const RowsArg &y) {
    const long long n = y.rows * y.cols;
    if (!n) return SAGE_OK;
    ctx.note_launch("embedding");
    if (ctx.dry()) return SAGE_OK;
    const long long blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < ctx.sm_count * 32ll ? blocks : ctx.sm_count * 32ll));
    return with_type(table.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_type(y.dtype, [&](auto o) {
            typedef decltype(o) Y;
            return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), embedding_kernel<T, Y>, grid, dim3(256), 0, (const T *)table.ptr, table.rows, table.pitch, (const int *)ids.ptr, ids.stride,
                                                   scale, (Y *)y.ptr, y.pitch, y.rows, y.cols),
                                  "embedding");
        });
    });
}

sage_status embedding_grad(Context &ctx, const RowsArg &g, const VectorArg &ids, float scale, bool add, const RowsArg &dtable) {
    if (!dtable.rows || !dtable.cols) return SAGE_OK;
    ctx.note_launch("embedding_grad");
    if (ctx.dry()) return SAGE_OK;
    return with_type(g.dtype, [&](auto t) {
        typedef decltype(t) T;
        return ctx.check_cuda(launch_dependent(ctx.pdl, ctx.stream(), embedding_grad_kernel<T>, dim3((unsigned)dtable.rows), dim3(256), 0, (const T *)g.ptr, g.pitch, (const int *)ids.ptr, ids.stride, scale,
                                               (int)add, (float *)dtable.ptr, dtable.pitch, g.rows, g.cols),
                              "embedding_grad");
    });
}

}  // namespace k
}  // namespace sage
