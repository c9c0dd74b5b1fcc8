// extern "C" surface of the language-model operators of include/sage_cuda.h: argument checks, then kernels/language.h.
#include <algorithm>
#include <cmath>
#include <exception>
#include <new>
#include <vector>

#include "../kernels/language.h"
#include "../runtime/runtime.h"

using namespace sage;

namespace {

struct Refused {
    std::string why;
};

size_t element_size(int dtype) { return dtype == SAGE_F16 || dtype == SAGE_BF16 ? 2 : dtype == SAGE_I8 || dtype == SAGE_U8 ? 1 : 4; }
bool is_real(int dtype) { return dtype == SAGE_F32 || dtype == SAGE_F16 || dtype == SAGE_BF16; }
bool is_index(int dtype) { return dtype == SAGE_I32 || dtype == SAGE_U32; }

// The checks of one call; each throws Refused with the call's and the operand's name.
struct Checks {
    Context &C;
    const char *call;

    [[noreturn]] void refuse(const char *operand, const char *why) const { throw Refused{std::string(call) + ": " + operand + " " + why}; }

    // The view lies in a buffer of this context.  Returns the address of its first element.
    void *view(const sage_tensor *t, const char *name) const {
        if (!t || !t->buf) refuse(name, "is missing");
        if (t->buf->owner != &C) refuse(name, "is another context's");
        if (t->dtype < SAGE_F32 || t->dtype > SAGE_U8) refuse(name, "has an unknown element type");
        if (t->ndim < 1 || t->ndim > SAGE_MAX_DIMS) refuse(name, "has no rank of 1 to 8");
        if (t->offset < 0) refuse(name, "starts in front of its buffer");
        bool empty = false;
        for (int i = 0; i < t->ndim; ++i) {
            if (t->extents[i] < 0 || t->strides[i] < 0) refuse(name, "has a negative extent or stride");
            empty |= t->extents[i] == 0;
        }
        const size_t size = element_size(t->dtype);
        const __int128 room = t->buf->size / size;
        __int128 last = t->offset;
        for (int i = 0; i < t->ndim && !empty; ++i) {  // a product has 126 bits at most
            last += (__int128)(t->extents[i] - 1) * t->strides[i];
            if (last >= room) refuse(name, "reaches behind the end of its buffer");
        }
        char *p = (char *)t->buf->ptr + (empty ? 0 : t->offset * (long long)size);
        if (!empty && (uintptr_t)p % size) refuse(name, "is not aligned to its elements");
        return p;
    }
    k::RowsArg rows(const sage_tensor *t, const char *name, bool output) const {
        k::RowsArg r;
        r.ptr = view(t, name);
        if (t->ndim != 2) refuse(name, "does not have rank 2");
        r.dtype = t->dtype;
        r.rows = t->extents[0];
        r.cols = t->extents[1];
        r.pitch = t->strides[0];
        if (r.cols > 1 && t->strides[1] != 1) refuse(name, "is not contiguous along its rows");
        if (output && r.rows > 1 && r.pitch < r.cols) refuse(name, "has rows that overlap");
        if (r.rows > k::kMaxRows || r.cols > k::kMaxRows) refuse(name, "has more than 2^31 - 2^16 rows or columns");
        return r;
    }
    k::RowsArg real_rows(const sage_tensor *t, const char *name, bool output) const {
        k::RowsArg r = rows(t, name, output);
        if (!is_real(r.dtype)) refuse(name, "is not f32, f16 or bf16");
        return r;
    }
    // A vector of n elements; `optional`: null gives a null argument.
    k::VectorArg vector(const sage_tensor *t, const char *name, long long n, bool index, bool output, bool optional) const {
        if (!t && optional) return k::VectorArg{};
        k::VectorArg v;
        v.ptr = view(t, name);
        if (t->ndim != 1 || t->extents[0] != n) refuse(name, "does not have one element for each row");
        if (index ? !is_index(t->dtype) : t->dtype != SAGE_F32) refuse(name, index ? "is not i32 or u32" : "is not f32");
        v.stride = t->strides[0];
        if (output && n > 1 && v.stride < 1) refuse(name, "has elements that overlap");
        return v;
    }
    // f32 [dim], or [groups, dim] whose groups divide `n` rows.
    k::RowsArg gate(const sage_tensor *t, const char *name, long long n, long long dim, bool output) const {
        k::RowsArg r;
        if (t->ndim == 1) {
            r.ptr = flat(t, name, dim);
            r.rows = 1;
            r.cols = r.pitch = dim;
            r.dtype = t->dtype;
        } else {
            r = rows(t, name, output);
            if (r.cols != dim) refuse(name, "does not have one element for each column");
            if (r.rows < 1 || n % r.rows) refuse(name, "has a number of rows that does not divide theirs");
        }
        if (r.dtype != SAGE_F32) refuse(name, "is not f32");
        return r;
    }
    // f32 [n, 4]
    k::RowsArg stats4(const sage_tensor *t, long long n, bool output, bool optional) const {
        if (!t && optional) return k::RowsArg{};
        const k::RowsArg r = rows(t, "stats", output);
        if (r.rows != n || r.cols != 4 || r.dtype != SAGE_F32) refuse("stats", "is not f32 [rows, 4]");
        return r;
    }
    // Contiguous memory of n elements (n < 0: as many as it has, left in *count).
    void *flat(const sage_tensor *t, const char *name, long long n, long long *count = nullptr) const {
        void *p = view(t, name);
        long long s = 1;
        for (int i = 0; i < t->ndim; ++i)
            if (!t->extents[i]) s = 0;
        for (int i = t->ndim - 1; i >= 0 && s; --i) {
            if (t->extents[i] > 1 && t->strides[i] != s) refuse(name, "is not contiguous");
            s *= t->extents[i];
        }
        if (n >= 0 && s != n) refuse(name, "does not have the number of elements that it should");
        if (count) *count = s;
        return p;
    }
};

template <class F>
sage_status guarded(sage_ctx *ctx, const char *call, F f) {
    if (!ctx || !ctx->impl) return SAGE_ERR_INVALID;
    Context &C = *ctx->impl;
    try {
        C.make_current();
        return f(Checks{C, call});
    } catch (const Refused &r) {
        return C.fail(SAGE_ERR_INVALID, r.why);
    } catch (const std::bad_alloc &) {
        return C.fail(SAGE_ERR_OOM, std::string(call) + ": out of host memory");
    } catch (const std::exception &e) {
        return C.fail(SAGE_ERR_INVALID, std::string(call) + ": " + e.what());
    }
}

float finite(const Checks &c, const char *name, double x) {
    if (!std::isfinite((float)x)) c.refuse(name, "is not finite");
    return (float)x;
}

float temperature_scale(const Checks &c, float scale) {
    if (!k::is_scale(scale)) c.refuse("scale", "is not positive and finite, also times log2(e)");
    return scale;
}

}  // namespace

extern "C" {

sage_status sage_embedding(sage_ctx *ctx, const sage_tensor *table, const sage_tensor *ids, float scale, const sage_tensor *y) {
    return guarded(ctx, "embedding", [&](const Checks &c) {
        const k::RowsArg t = c.real_rows(table, "table", false), o = c.real_rows(y, "y", true);
        const k::VectorArg i = c.vector(ids, "ids", o.rows, true, false, false);
        if (o.cols != t.cols) c.refuse("y", "does not have the table's width");
        if (o.dtype != SAGE_F32 && o.dtype != t.dtype) c.refuse("y", "is neither f32 nor of the table's type");
        return k::embedding(c.C, t, i, finite(c, "scale", scale), o);
    });
}

sage_status sage_embedding_grad(sage_ctx *ctx, const sage_tensor *g, const sage_tensor *ids, float scale, int32_t add, const sage_tensor *dtable) {
    return guarded(ctx, "embedding_grad", [&](const Checks &c) {
        const k::RowsArg in = c.real_rows(g, "g", false), o = c.rows(dtable, "dtable", true);
        const k::VectorArg i = c.vector(ids, "ids", in.rows, true, false, false);
        if (o.dtype != SAGE_F32) c.refuse("dtable", "is not f32");
        if (o.cols != in.cols) c.refuse("dtable", "does not have the width of g");
        return k::embedding_grad(c.C, in, i, finite(c, "scale", scale), add != 0, o);
    });
}

sage_status sage_token_log_probs(sage_ctx *ctx, const sage_tensor *logits, const sage_tensor *ids, float scale, const sage_tensor *log_probs,
                                 const sage_tensor *entropy, const sage_tensor *stats, const sage_tensor *top_ids, const sage_tensor *top_log_probs) {
    return guarded(ctx, "token_log_probs", [&](const Checks &c) {
        k::LogProbs a;
        a.logits = c.real_rows(logits, "logits", false);
        const long long n = a.logits.rows;
        if (n && !a.logits.cols) c.refuse("logits", "has rows without elements");
        a.scale = temperature_scale(c, scale);
        a.ids = c.vector(ids, "ids", n, true, false, false);
        a.log_probs = c.vector(log_probs, "log_probs", n, false, true, false);
        a.entropy = c.vector(entropy, "entropy", n, false, true, true);
        if (stats) {
            a.stats = c.rows(stats, "stats", true);
            if (a.stats.rows != n || a.stats.cols != 2 || a.stats.dtype != SAGE_F32) c.refuse("stats", "is not f32 [rows, 2]");
        }
        if (!top_ids != !top_log_probs) c.refuse(top_ids ? "top_log_probs" : "top_ids", "is missing");
        if (top_ids) {
            a.top_ids = c.rows(top_ids, "top_ids", true);
            a.top_log_probs = c.rows(top_log_probs, "top_log_probs", true);
            if (!is_index(a.top_ids.dtype)) c.refuse("top_ids", "is not i32 or u32");
            if (a.top_log_probs.dtype != SAGE_F32) c.refuse("top_log_probs", "is not f32");
            if (a.top_ids.rows != n || a.top_log_probs.rows != n || a.top_ids.cols != a.top_log_probs.cols) c.refuse("top_ids", "and top_log_probs do not have one row for each row of the logits and the same width");
            if (a.top_ids.cols > k::kMaxTop || (n && a.top_ids.cols > a.logits.cols)) c.refuse("top_ids", "asks for more than 32 alternatives, or more than there are tokens");
            a.top = (int)a.top_ids.cols;
        }
        return k::token_log_probs(c.C, a);
    });
}

static k::LogProbsGrad grad_args(const Checks &c, const sage_tensor *logits, const sage_tensor *ids, float scale, const sage_tensor *g_log_probs, const sage_tensor *g_entropy, const sage_tensor *dlogits) {
    k::LogProbsGrad a;
    a.logits = c.real_rows(logits, "logits", false);
    const long long n = a.logits.rows;
    if (n && !a.logits.cols) c.refuse("logits", "has rows without elements");
    a.scale = temperature_scale(c, scale);
    a.ids = c.vector(ids, "ids", n, true, false, false);
    a.g_log_probs = c.vector(g_log_probs, "g_log_probs", n, false, false, true);
    a.g_entropy = c.vector(g_entropy, "g_entropy", n, false, false, true);
    a.dlogits = c.real_rows(dlogits, "dlogits", true);
    if (a.dlogits.rows != n || a.dlogits.cols != a.logits.cols || a.dlogits.dtype != a.logits.dtype) c.refuse("dlogits", "does not have the logits' shape and type");
    return a;
}

sage_status sage_token_log_probs_grad(sage_ctx *ctx, const sage_tensor *logits, const sage_tensor *ids, float scale, const sage_tensor *stats,
                                      const sage_tensor *entropy, const sage_tensor *g_log_probs, const sage_tensor *g_entropy, const sage_tensor *dlogits) {
    return guarded(ctx, "token_log_probs_grad", [&](const Checks &c) {
        k::LogProbsGrad a = grad_args(c, logits, ids, scale, g_log_probs, g_entropy, dlogits);
        a.stats = c.rows(stats, "stats", false);
        if (a.stats.rows != a.logits.rows || a.stats.cols != 2 || a.stats.dtype != SAGE_F32) c.refuse("stats", "is not f32 [rows, 2]");
        if (g_entropy && !entropy) c.refuse("entropy", "is missing, which g_entropy needs");
        a.entropy = c.vector(entropy, "entropy", a.logits.rows, false, false, true);
        return k::token_log_probs_grad(c.C, a);
    });
}

sage_status sage_token_log_probs_and_grad(sage_ctx *ctx, const sage_tensor *logits, const sage_tensor *ids, float scale, const sage_tensor *g_log_probs,
                                          const sage_tensor *g_entropy, const sage_tensor *log_probs, const sage_tensor *entropy, const sage_tensor *dlogits) {
    return guarded(ctx, "token_log_probs_and_grad", [&](const Checks &c) {
        k::LogProbsGrad a = grad_args(c, logits, ids, scale, g_log_probs, g_entropy, dlogits);
        const k::VectorArg lp = c.vector(log_probs, "log_probs", a.logits.rows, false, true, false);
        const k::VectorArg h = c.vector(entropy, "entropy", a.logits.rows, false, true, true);
        return k::token_log_probs_and_grad(c.C, a, lp, h);
    });
}

static k::Head head_args(const Checks &c, const sage_tensor *hidden, const sage_tensor *weight, const sage_tensor *ids, float scale) {
    k::Head a;
    a.hidden = c.real_rows(hidden, "hidden", false);
    a.weight = c.real_rows(weight, "weight", false);
    if (a.weight.dtype != a.hidden.dtype) c.refuse("weight", "does not have the type of hidden");
    if (a.weight.cols != a.hidden.cols) c.refuse("weight", "does not have the width of hidden");
    if (!a.weight.cols) c.refuse("hidden", "has rows without elements");
    if (!a.weight.rows) c.refuse("weight", "has no rows");
    a.ids = c.vector(ids, "ids", a.hidden.rows, true, false, false);
    a.scale = temperature_scale(c, scale);
    return a;
}

sage_status sage_head_log_probs(sage_ctx *ctx, const sage_tensor *hidden, const sage_tensor *weight, const sage_tensor *ids, float scale, const sage_tensor *log_probs,
                                const sage_tensor *entropy, const sage_tensor *stats) {
    return guarded(ctx, "head_log_probs", [&](const Checks &c) {
        const k::Head a = head_args(c, hidden, weight, ids, scale);
        const long long n = a.hidden.rows;
        const k::VectorArg lp = c.vector(log_probs, "log_probs", n, false, true, false), h = c.vector(entropy, "entropy", n, false, true, true);
        k::RowsArg st;
        if (stats) {
            st = c.rows(stats, "stats", true);
            if (st.rows != n || st.cols != 2 || st.dtype != SAGE_F32) c.refuse("stats", "is not f32 [rows, 2]");
        }
        return k::head_log_probs(c.C, a, lp, h, st);
    });
}

sage_status sage_head_log_probs_grad(sage_ctx *ctx, const sage_tensor *hidden, const sage_tensor *weight, const sage_tensor *ids, float scale, const sage_tensor *stats,
                                     const sage_tensor *entropy, const sage_tensor *g_log_probs, const sage_tensor *g_entropy, const sage_tensor *dhidden, const sage_tensor *dweight) {
    return guarded(ctx, "head_log_probs_grad", [&](const Checks &c) {
        const k::Head a = head_args(c, hidden, weight, ids, scale);
        const long long n = a.hidden.rows;
        const k::RowsArg st = c.rows(stats, "stats", false);
        if (st.rows != n || st.cols != 2 || st.dtype != SAGE_F32) c.refuse("stats", "is not f32 [rows, 2]");
        if (g_entropy && !entropy) c.refuse("entropy", "is missing, which g_entropy needs");
        const k::VectorArg h = c.vector(entropy, "entropy", n, false, false, true), gl = c.vector(g_log_probs, "g_log_probs", n, false, false, true), ge = c.vector(g_entropy, "g_entropy", n, false, false, true);
        const auto like = [&](const sage_tensor *t, const char *name, const k::RowsArg &of) {
            k::RowsArg r;
            if (!t) return r;
            r = c.real_rows(t, name, true);
            if (r.rows != of.rows || r.cols != of.cols) c.refuse(name, "does not have its operand's shape");
            if (r.dtype != SAGE_F32 && r.dtype != of.dtype) c.refuse(name, "is neither f32 nor of its operand's type");
            return r;
        };
        const k::RowsArg dh = like(dhidden, "dhidden", a.hidden), dw = like(dweight, "dweight", a.weight);
        return k::head_log_probs_grad(c.C, a, st, h, gl, ge, dh, dw);
    });
}

static k::Dropout dropout_args(const Checks &c, const sage_tensor *seed, float p, uint64_t site) {
    k::Dropout d;
    if (!(p >= 0.f && p < 1.f)) c.refuse("p", "is not in [0, 1)");
    d.bar = (unsigned)std::min(65535.0, std::nearbyint((double)p * 65536.0));
    d.factor = (float)(65536.0 / (65536.0 - d.bar));
    d.site = site;
    if (p > 0.f || seed) {
        const k::VectorArg v = c.vector(seed, "seed", 2, true, false, false);
        d.seed = (const unsigned *)v.ptr;
        d.seed_stride = v.stride;
    }
    return d;
}

sage_status sage_dropout(sage_ctx *ctx, const sage_tensor *x, const sage_tensor *y, const sage_tensor *seed, float p, uint64_t site) {
    return guarded(ctx, "dropout", [&](const Checks &c) {
        const k::RowsArg in = c.real_rows(x, "x", false), o = c.real_rows(y, "y", true);
        if (o.rows != in.rows || o.cols != in.cols || o.dtype != in.dtype) c.refuse("y", "does not have the shape and type of x");
        return k::dropout(c.C, in, o, dropout_args(c, seed, p, site));
    });
}

static const sage_tensor *given(const sage_tensor &t) { return t.buf ? &t : nullptr; }

// The description of both directions, for rows of `dim` columns; `branch`: there is a y.
static k::BlockNorms norms_args(const Checks &c, const sage_block_norms_opts *o, long long rows, long long dim, bool branch) {
    if (!o) c.refuse("opts", "is missing");
    k::BlockNorms n;
    if (dim < 1 || dim > k::kMaxNormColumns) c.refuse("x", "does not have 1 to 16384 columns");
    n.dim = dim;
    for (int kind : {o->after, o->before})
        if (kind < SAGE_NORM_NONE || kind > SAGE_NORM_LAYER) c.refuse("after or before", "is no sage_norm");
    n.after = o->after;
    n.before = o->before;
    const auto row = [&](const sage_tensor &t, const char *name, int kind) -> const float * {
        if (!t.buf) return nullptr;
        if (kind == SAGE_NORM_NONE) c.refuse(name, "is given without its norm");
        if (t.dtype != SAGE_F32) c.refuse(name, "is not f32");
        if (t.ndim != 1) c.refuse(name, "does not have rank 1");
        return (const float *)c.flat(&t, name, dim);
    };
    n.after_weight = row(o->after_weight, "after_weight", n.after);
    n.after_bias = row(o->after_bias, "after_bias", n.after);
    n.before_weight = row(o->before_weight, "before_weight", n.before);
    n.before_bias = row(o->before_bias, "before_bias", n.before);
    n.eps = o->eps;
    if (!(n.eps > 0.f) || !std::isfinite(n.eps)) c.refuse("eps", "is not positive and finite");
    n.scale = finite(c, "residual_scale", o->residual_scale);
    n.drop = dropout_args(c, given(o->seed), o->p, o->site);
    if (o->gate.buf) n.gate = c.gate(&o->gate, "gate", rows, dim, false);
    if (!branch && (n.after != SAGE_NORM_NONE || o->gate.buf || o->p > 0.f)) c.refuse("y", "is missing, which the norm after, the gate and dropout need");
    return n;
}

sage_status sage_block_norms(sage_ctx *ctx, const sage_block_norms_opts *opts, const sage_tensor *x, const sage_tensor *y, const sage_tensor *out, const sage_tensor *h, const sage_tensor *stats) {
    return guarded(ctx, "block_norms", [&](const Checks &c) {
        const k::RowsArg xs = c.real_rows(x, "x", false);
        const auto like = [&](const sage_tensor *t, const char *name, bool output) {
            k::RowsArg r;
            if (!t) return r;
            r = c.real_rows(t, name, output);
            if (r.rows != xs.rows || r.cols != xs.cols) c.refuse(name, "does not have the shape of x");
            return r;
        };
        const k::RowsArg ys = like(y, "y", false), os = like(out, "out", true), hs = like(h, "h", true);
        k::BlockNorms n = norms_args(c, opts, xs.rows, xs.cols, y != nullptr);
        n.x_dtype = xs.dtype;
        n.dtype = y ? ys.dtype : h ? hs.dtype : xs.dtype;
        if (out && os.dtype != xs.dtype) c.refuse("out", "does not have the type of x");
        if (xs.dtype != SAGE_F32 && xs.dtype != n.dtype) c.refuse("x", "is neither f32 nor of the type of y and h");
        if (y && h && hs.dtype != ys.dtype) c.refuse("h", "does not have the type of y");
        if (!h != (n.before == SAGE_NORM_NONE)) c.refuse("h", h ? "is given without a norm before" : "is missing, which the norm before writes");
        if (!out && (y || n.scale != 1.f || !h)) c.refuse("out", "is missing");
        return k::block_norms(c.C, n, xs, ys, os, hs, c.stats4(stats, xs.rows, true, true));
    });
}

sage_status sage_block_norms_grad(sage_ctx *ctx, const sage_block_norms_opts *opts, const sage_tensor *out, const sage_tensor *y, const sage_tensor *stats, const sage_tensor *g_out,
                                  const sage_tensor *g_h, const sage_tensor *dx, const sage_tensor *dy, const sage_block_norms_sums *sums) {
    return guarded(ctx, "block_norms_grad", [&](const Checks &c) {
        const k::RowsArg os = c.real_rows(out, "out", false);
        const auto like = [&](const sage_tensor *t, const char *name, bool output) {
            k::RowsArg r;
            if (!t) return r;
            r = c.real_rows(t, name, output);
            if (r.rows != os.rows || r.cols != os.cols) c.refuse(name, "does not have the shape of out");
            return r;
        };
        const k::RowsArg ys = like(y, "y", false), go = like(g_out, "g_out", false), gh = like(g_h, "g_h", false), xs = like(dx, "dx", true), d = like(dy, "dy", true);
        k::BlockNorms n = norms_args(c, opts, os.rows, os.cols, y != nullptr);
        n.x_dtype = os.dtype;
        n.dtype = y ? ys.dtype : g_h ? gh.dtype : os.dtype;
        if (os.dtype != SAGE_F32 && os.dtype != n.dtype) c.refuse("out", "is neither f32 nor of the type of y and g_h");
        if (g_out && go.dtype != os.dtype) c.refuse("g_out", "does not have the type of out");
        if (dx && xs.dtype != os.dtype) c.refuse("dx", "does not have the type of out");
        if (y && g_h && gh.dtype != ys.dtype) c.refuse("g_h", "does not have the type of y");
        if (dy && (!y || d.dtype != n.dtype)) c.refuse("dy", y ? "does not have the type of y" : "is given without y");
        if (g_h && n.before == SAGE_NORM_NONE) c.refuse("g_h", "is given without a norm before");
        if (!g_out && !g_h) c.refuse("g_out", "and g_h are both missing");
        const k::RowsArg st = c.stats4(stats, os.rows, false, false);
        k::BlockNormsSums s;
        if (sums) {
            const auto row = [&](const sage_tensor &t, const char *name, int kind) -> float * {
                if (!t.buf) return nullptr;
                if (kind == SAGE_NORM_NONE) c.refuse(name, "is given without its norm");
                if (t.dtype != SAGE_F32) c.refuse(name, "is not f32");
                if (t.ndim != 1) c.refuse(name, "does not have rank 1");
                return (float *)c.flat(&t, name, os.cols);
            };
            s.after_weight = row(sums->after_weight, "sums of after_weight", n.after);
            s.after_bias = row(sums->after_bias, "sums of after_bias", n.after);
            s.before_weight = row(sums->before_weight, "sums of before_weight", n.before);
            s.before_bias = row(sums->before_bias, "sums of before_bias", n.before);
            if (sums->gate.buf) {
                if (!n.gate.ptr) c.refuse("sums of gate", "is given without a gate");
                s.gate = c.gate(&sums->gate, "sums of gate", os.rows, os.cols, true);
                if (s.gate.rows != n.gate.rows) c.refuse("sums of gate", "does not have the gate's shape");
            }
        }
        return k::block_norms_grad(c.C, n, os, ys, st, go, gh, xs, d, s);
    });
}

sage_status sage_adamw_step(sage_ctx *ctx, const sage_adamw_tensor *tensors, int32_t count, const sage_adamw_opts *o) {
    return guarded(ctx, "adamw_step", [&](const Checks &c) {
        if (!o) c.refuse("opts", "is missing");
        if (count < 0 || (count && !tensors)) c.refuse("tensors", "is missing");
        if (o->step < 1) c.refuse("step", "is less than 1");
        if (!(o->beta1 >= 0.0 && o->beta1 < 1.0) || !(o->beta2 >= 0.0 && o->beta2 < 1.0)) c.refuse("beta1 or beta2", "is not in [0, 1)");
        if (!(o->eps >= 1e-15)) c.refuse("eps", "is less than 1e-15");
        for (double x : {o->lr, o->weight_decay, o->lr * o->weight_decay, o->eps}) finite(c, "lr, weight_decay or eps", x);
        finite(c, "grad_scale", o->grad_scale);
        const k::AdamWRule rule = k::adamw_rule(o->lr, o->beta1, o->beta2, o->eps, o->weight_decay, o->grad_scale, o->step);
        std::vector<k::AdamWSlot> slots;
        slots.reserve((size_t)count);
        const bool states8 = count && tensors[0].m.dtype == SAGE_I8;
        for (int i = 0; i < count; ++i) {
            const sage_adamw_tensor &t = tensors[i];
            k::AdamWSlot s;
            if (t.param.dtype != SAGE_F32) c.refuse("param", "is not f32");
            s.p = (float *)c.flat(&t.param, "param", -1, &s.n);
            if (!is_real(t.grad.dtype)) c.refuse("grad", "is not f32, f16 or bf16");
            s.g = c.flat(&t.grad, "grad", s.n);
            s.g_dtype = (short)t.grad.dtype;
            if (t.m.dtype != (states8 ? SAGE_I8 : SAGE_F32) || t.v.dtype != (states8 ? SAGE_U8 : SAGE_F32)) c.refuse("m or v", "is not of the first tensor's kind: f32 both, or i8 and u8");
            s.m = c.flat(&t.m, "m", s.n);
            s.v = c.flat(&t.v, "v", s.n);
            if (states8) {
                if (t.m_scale.dtype != SAGE_F32 || t.v_scale.dtype != SAGE_F32) c.refuse("m_scale or v_scale", "is not f32");
                const long long blocks = (s.n + k::kAdamWBlock - 1) / k::kAdamWBlock;
                s.m_scale = (float *)c.flat(&t.m_scale, "m_scale", blocks);
                s.v_scale = (float *)c.flat(&t.v_scale, "v_scale", blocks);
            }
            if (t.copy.buf) {
                if (t.copy.dtype != SAGE_F16 && t.copy.dtype != SAGE_BF16) c.refuse("copy", "is not f16 or bf16");
                s.copy = c.flat(&t.copy, "copy", s.n);
                s.copy_dtype = (short)t.copy.dtype;
            }
            if (s.n) slots.push_back(s);
        }
        return k::adamw_step(c.C, slots.data(), (int)slots.size(), states8, rule);
    });
}

sage_status sage_adamw_states(sage_ctx *ctx, const sage_tensor *m, const sage_tensor *m_scale, const sage_tensor *v, const sage_tensor *v_scale,
                              const sage_tensor *m_out, const sage_tensor *v_out) {
    return guarded(ctx, "adamw_states", [&](const Checks &c) {
        long long n = 0;
        const void *mp = c.flat(m, "m", -1, &n), *vp = c.flat(v, "v", n);
        if (m->dtype != SAGE_I8 || v->dtype != SAGE_U8) c.refuse("m or v", "is not i8 and u8");
        const long long blocks = (n + k::kAdamWBlock - 1) / k::kAdamWBlock;
        const float *ms = (const float *)c.flat(m_scale, "m_scale", blocks), *vs = (const float *)c.flat(v_scale, "v_scale", blocks);
        float *mo = (float *)c.flat(m_out, "m_out", n), *vo = (float *)c.flat(v_out, "v_out", n);
        if (m_scale->dtype != SAGE_F32 || v_scale->dtype != SAGE_F32 || m_out->dtype != SAGE_F32 || v_out->dtype != SAGE_F32) c.refuse("a scale or an output", "is not f32");
        return k::adamw_states(c.C, mp, ms, vp, vs, n, mo, vo);
    });
}

}  // extern "C"
