// Language-model operators of the lazy graph: token embedding, log probabilities of given tokens with entropy, alternatives, the same from hidden
// states, dropout, norms around a block (kernels/language.h).  No counterpart in the reference, whose embedding is a gather (layers.rs:427-452) with a scatter as its
// gradient and whose loss is composed (nn.rs:70-82).
#include <algorithm>
#include <cmath>

#include "../kernels/language.h"
#include "graph.h"

namespace sage {
using namespace ops;

namespace {

// `t` as rows of its last axis, contiguous along them; a copy in *hold where its strides are others.
sage_status rows_of(Context &ctx, const Tensor &t, long long rows, long long cols, Tensor *hold, k::RowsArg *out) {
    *hold = t;
    const Shape &s = t.desc.shape;
    const bool plain = s.has_default_strides(), pitched = s.rank() == 2 && s.extents[0] == rows && s.extents[1] == cols && (cols <= 1 || s.strides[1] == 1);
    if (t.data->planes_only) return ctx.fail(SAGE_ERR_INVALID, "internal: an operand exists in the tensor cores' form only");
    if (!plain && !pitched) {
        sage_status st = Tensor::uninit(ctx, t.desc.pristine(), hold);
        if (st) return st;
        st = k::strided_copy(ctx, (const uint32_t *)t.ptr(), t.dims(), (uint32_t *)hold->ptr(), hold->desc.shape.strides.data());
        if (st) return st;
    }
    *out = k::RowsArg{hold->ptr(), SAGE_F32, rows, cols, !plain && pitched ? s.strides[0] : cols};
    return SAGE_OK;
}
// `t` as a vector of all of its elements.
sage_status vector_of(Context &ctx, const Tensor &t, Tensor *hold, k::VectorArg *out) {
    k::RowsArg r;
    sage_status st = rows_of(ctx, t, t.desc.shape.size(), 1, hold, &r);
    if (st) return st;
    *out = k::VectorArg{r.ptr, r.pitch};
    return SAGE_OK;
}

void check_ids(const Var &ids, const char *what) {
    if (ids.dtype() != SAGE_I32 && ids.dtype() != SAGE_U32) shape_fail(std::string(what) + ": token ids must be i32 or u32");
}

void check_rows(long long rows, long long cols, const char *what) {
    if (rows > k::kMaxRows || cols > k::kMaxRows) shape_fail(std::string(what) + ": more than 2^31 - 2^16 rows, tokens or columns");
}

struct EmbeddingGradOp : Operator {  // inputs gy [.., D], ids [..] -> [V, D]
    float scale;
    const char *name() const override { return "embedding_grad"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &, const Var &gy) override { return {embedding(gy, x[1], scale), Var()}; }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor g_hold, ids_hold;
        k::RowsArg g;
        k::VectorArg ids;
        const long long dim = out.shape.extents[1];
        sage_status st = rows_of(ctx, x[0], dim ? x[0].desc.shape.size() / dim : 0, dim, &g_hold, &g);
        if (!st) st = vector_of(ctx, x[1], &ids_hold, &ids);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        return k::embedding_grad(ctx, g, ids, scale, false, k::RowsArg{y->ptr(), SAGE_F32, out.shape.extents[0], dim, dim});
    }
};

struct EmbeddingOp : Operator {  // inputs table [V, D], ids [..] -> [.., D]
    float scale;
    const char *name() const override { return "embedding"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &, const Var &gy) override {
        auto op = std::make_shared<EmbeddingGradOp>();
        op->scale = scale;
        op->in = {gy.desc, x[1].desc};
        op->out = x[0].desc.pristine();
        return {Var::from_op(op, {gy, x[1]}), Var()};
    }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor table_hold, ids_hold;
        k::RowsArg table;
        k::VectorArg ids;
        const Shape &t = x[0].desc.shape;
        sage_status st = rows_of(ctx, x[0], t.extents[0], t.extents[1], &table_hold, &table);
        if (!st) st = vector_of(ctx, x[1], &ids_hold, &ids);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        return k::embedding(ctx, table, ids, scale, k::RowsArg{y->ptr(), SAGE_F32, x[1].desc.shape.size(), t.extents[1], t.extents[1]});
    }
};

// y [R, 4]: the token's log probability, the row's entropy, and what the gradient reads (the largest logit, the sum of exponentials).
k::VectorArg column(const Tensor &y, int c) { return k::VectorArg{(float *)y.ptr() + c * y.desc.shape.strides[1], y.desc.shape.strides[0]}; }

struct TokenLogProbsGradOp : Operator {  // inputs logits, ids, y, gy -> [R, V]
    float scale;
    const char *name() const override { return "token_log_probs_grad"; }
    std::vector<Var> grad(const std::vector<Var> &, const Var &, const Var &) override { shape_fail("token_log_probs is differentiated once"); }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor logits_hold, ids_hold, y_hold, gy_hold;
        k::LogProbsGrad a;
        k::RowsArg gy;
        const long long rows = out.shape.extents[0], vocab = out.shape.extents[1];
        sage_status st = rows_of(ctx, x[0], rows, vocab, &logits_hold, &a.logits);
        if (!st) st = vector_of(ctx, x[1], &ids_hold, &a.ids);
        if (!st) st = rows_of(ctx, x[2], rows, 4, &y_hold, &a.stats);
        if (!st) st = rows_of(ctx, x[3], rows, 4, &gy_hold, &gy);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        a.scale = scale;
        a.entropy = k::VectorArg{(float *)a.stats.ptr + 1, a.stats.pitch};
        a.stats.ptr = (float *)a.stats.ptr + 2;
        a.stats.cols = 2;
        a.g_log_probs = k::VectorArg{gy.ptr, gy.pitch};
        a.g_entropy = k::VectorArg{(float *)gy.ptr + 1, gy.pitch};
        a.dlogits = k::RowsArg{y->ptr(), SAGE_F32, rows, vocab, vocab};
        return k::token_log_probs_grad(ctx, a);
    }
};

struct TokenLogProbsOp : Operator {  // inputs logits [R, V], ids [R] or [R, 1] -> [R, 4]
    float scale;
    const char *name() const override { return "token_log_probs"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &y, const Var &gy) override {
        auto op = std::make_shared<TokenLogProbsGradOp>();
        op->scale = scale;
        op->in = {x[0].desc, x[1].desc, y.desc, gy.desc};
        op->out = x[0].desc.pristine();
        return {Var::from_op(op, {x[0], x[1], y, gy}), Var()};
    }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor logits_hold, ids_hold;
        k::LogProbs a;
        sage_status st = rows_of(ctx, x[0], in[0].shape.extents[0], in[0].shape.extents[1], &logits_hold, &a.logits);
        if (!st) st = vector_of(ctx, x[1], &ids_hold, &a.ids);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        a.scale = scale;
        a.log_probs = column(*y, 0);
        a.entropy = column(*y, 1);
        a.stats = k::RowsArg{(float *)y->ptr() + 2, SAGE_F32, a.logits.rows, 2, 4};
        return k::token_log_probs(ctx, a);
    }
};

struct TopTokensOp : Operator {  // logits [R, V] -> [R, k] u32
    const char *name() const override { return "top_tokens"; }
    std::vector<Var> grad(const std::vector<Var> &, const Var &, const Var &) override { return {Var()}; }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor hold;
        k::LogProbs a;
        sage_status st = rows_of(ctx, x[0], in[0].shape.extents[0], in[0].shape.extents[1], &hold, &a.logits);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        a.top = (int)out.shape.extents[1];
        a.top_ids = k::RowsArg{y->ptr(), SAGE_U32, a.logits.rows, a.top, a.top};
        return k::token_log_probs(ctx, a);
    }
};

// ------------------------------------------------------------------------------------------ results side by side
// An operator of the graph has one result: several lie behind one another in it, each from a multiple of 64 elements on, and their readers take views.
struct Parts {
    std::vector<long long> at, size;
    long long total = 0;
    int add(long long n) {
        at.push_back(total);
        size.push_back(n);
        total += (n + 63) / 64 * 64;
        return (int)at.size() - 1;
    }
    // What lies between parts is zero: a reader that takes the whole result to pieces (products do) scales groups of 64 elements by their largest.
    sage_status clear_gaps(Context &ctx, float *to) const {
        for (size_t i = 0; i < at.size(); ++i) {
            const long long gap = (64 - size[i] % 64) % 64;
            if (!gap) continue;
            ctx.note_memset();
            if (ctx.dry()) continue;
            sage_status st = ctx.check_cuda(cudaMemsetAsync(to + at[i] + size[i], 0, (size_t)gap * 4, ctx.stream()), "memset");
            if (st) return st;
        }
        return SAGE_OK;
    }
    Var view(const Var &all, int part, const Array &extents) const { return ops::view(slice(all, 0, at[part], at[part] + size[part]), extents); }
};
// Adds what arrives for the parts of such a result: the gradient of each view is an unslice, several are sums of them, whose inputs are taken as they are.
// False: something else.
bool arrivals(const Var &g, const Parts &parts, std::vector<Var> *found) {
    if (!g.is_op()) return false;
    const Origin &o = *g.origin;
    const long long start = unslice_start(*o.op);
    if (start >= 0) {
        for (size_t i = 0; i < parts.at.size(); ++i)
            if (parts.at[i] == start && parts.size[i] == o.inputs[0].size()) {
                (*found)[i] = (*found)[i].defined() ? add((*found)[i], o.inputs[0]) : o.inputs[0];
                return true;
            }
        return false;
    }
    const MapExpr *e = map_expr_of(*o.op);
    if (!e || e->kind != MapExpr::Bin || e->op != ops::Add || o.inputs.size() != 2) return false;
    for (const MapExpr &a : e->args)
        if (a.kind != MapExpr::Input) return false;
    return arrivals(o.inputs[e->args[0].input], parts, found) && arrivals(o.inputs[e->args[1].input], parts, found);
}

k::Dropout dropout_of(float p, unsigned long long site, const unsigned *seed, long long stride) {
    k::Dropout d;
    d.bar = (unsigned)std::min(65535.0, std::nearbyint((double)p * 65536.0));
    d.factor = (float)(65536.0 / (65536.0 - d.bar));
    d.site = site;
    d.seed = seed;
    d.seed_stride = stride;
    return d;
}
void check_dropout(const Var &seed, float p, const char *what) {
    if (!(p >= 0.f && p < 1.f)) shape_fail(std::string(what) + ": p must be in [0, 1)");
    if (seed.defined() ? (seed.dtype() != SAGE_U32 && seed.dtype() != SAGE_I32) || seed.size() != 2 || seed.rank() < 1 : p > 0.f) shape_fail(std::string(what) + ": the seed must be two i32 or u32");
}

struct DropoutOp : Operator {  // inputs x, seed -> the same extents
    float p;
    unsigned long long site;
    const char *name() const override { return "dropout"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &, const Var &gy) override { return {dropout(gy, x[1], p, site), Var()}; }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor x_hold, seed_hold;
        k::RowsArg in;
        k::VectorArg seed;
        const long long n = out.shape.size();
        sage_status st = rows_of(ctx, x[0], 1, n, &x_hold, &in);
        if (!st) st = vector_of(ctx, x[1], &seed_hold, &seed);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        return k::dropout(ctx, in, k::RowsArg{y->ptr(), SAGE_F32, 1, n, n}, dropout_of(p, site, (const unsigned *)seed.ptr, seed.stride));
    }
};

enum { kAfterWeight, kAfterBias, kBeforeWeight, kBeforeBias, kGate, kSeed, kNormOperands };
struct NormsGradOp;
struct NormsOp : Operator {  // inputs x, y, the operands (those that are there) -> out, h, statistics
    int after, before;
    float scale, eps, p;
    unsigned long long site;
    long long rows, dim;
    int y_at = -1, operand_at[kNormOperands];
    Parts parts;
    int out_part, h_part = -1, stats_part;
    const char *name() const override { return "block_norms"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &y, const Var &gy) override;
    // The kernels' description, with the operands' tensors.
    sage_status describe(const std::vector<Tensor> &x, Context &ctx, std::vector<Tensor> *hold, k::BlockNorms *n, k::RowsArg *y) const {
        n->after = after;
        n->before = before;
        n->scale = scale;
        n->eps = eps;
        n->dim = dim;
        hold->resize(kNormOperands + 1);
        sage_status st = SAGE_OK;
        const float **to[4] = {&n->after_weight, &n->after_bias, &n->before_weight, &n->before_bias};
        for (int i = 0; i < kNormOperands && !st; ++i) {
            if (operand_at[i] < 0) continue;
            const Tensor &t = x[operand_at[i]];
            k::RowsArg r;
            const long long groups = t.desc.shape.size() / dim;
            if (i == kSeed) {
                st = rows_of(ctx, t, 1, 2, &(*hold)[i], &r);
                n->drop = dropout_of(p, site, (const unsigned *)r.ptr, 1);
            } else if (i == kGate) {
                st = rows_of(ctx, t, groups, dim, &(*hold)[i], &n->gate);
            } else {
                st = rows_of(ctx, t, 1, dim, &(*hold)[i], &r);
                *to[i] = (const float *)r.ptr;
            }
        }
        if (!st && y_at >= 0) st = rows_of(ctx, x[y_at], rows, dim, &(*hold)[kNormOperands], y);
        return st;
    }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        std::vector<Tensor> hold;
        Tensor x_hold;
        k::BlockNorms n;
        k::RowsArg in, branch;
        sage_status st = describe(x, ctx, &hold, &n, &branch);
        if (!st) st = rows_of(ctx, x[0], rows, dim, &x_hold, &in);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (!st) st = parts.clear_gaps(ctx, (float *)y->ptr());
        if (st) return st;
        float *to = (float *)y->ptr();
        const auto part = [&](int i, long long cols) { return i < 0 ? k::RowsArg{} : k::RowsArg{to + parts.at[i], SAGE_F32, rows, cols, cols}; };
        return k::block_norms(ctx, n, in, branch, part(out_part, dim), part(h_part, dim), part(stats_part, 4));
    }
};
struct NormsGradOp : Operator {  // inputs the forward result, its inputs behind x, what arrives for out and h -> the gradients
    std::shared_ptr<NormsOp> forward;
    int go_at = -1, gh_at = -1;
    Parts parts;
    int dx_part = 0, dy_part = -1, sum_part[kNormOperands];
    const char *name() const override { return "block_norms_grad"; }
    std::vector<Var> grad(const std::vector<Var> &, const Var &, const Var &) override { shape_fail("block_norms is differentiated once"); }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        const NormsOp &f = *forward;
        std::vector<Tensor> hold;
        Tensor all_hold, go_hold, gh_hold;
        k::BlockNorms n;
        k::RowsArg all, branch, go, gh;
        sage_status st = f.describe(x, ctx, &hold, &n, &branch);  // (x[0] stands where the forward pass had the stream)
        if (!st) st = rows_of(ctx, x[0], 1, f.parts.total, &all_hold, &all);
        if (!st && go_at >= 0) st = rows_of(ctx, x[go_at], f.rows, f.dim, &go_hold, &go);
        if (!st && gh_at >= 0) st = rows_of(ctx, x[gh_at], f.rows, f.dim, &gh_hold, &gh);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (!st) st = parts.clear_gaps(ctx, (float *)y->ptr());
        if (st) return st;
        float *to = (float *)y->ptr(), *from = (float *)all.ptr;
        const auto rows = [&](float *p, long long at, long long cols) { return k::RowsArg{p + at, SAGE_F32, f.rows, cols, cols}; };
        const auto sum = [&](int i) { return sum_part[i] < 0 ? nullptr : to + parts.at[sum_part[i]]; };
        k::BlockNormsSums s;
        s.after_weight = sum(kAfterWeight);
        s.after_bias = sum(kAfterBias);
        s.before_weight = sum(kBeforeWeight);
        s.before_bias = sum(kBeforeBias);
        if (sum(kGate)) s.gate = k::RowsArg{sum(kGate), SAGE_F32, n.gate.rows, f.dim, f.dim};
        return k::block_norms_grad(ctx, n, rows(from, f.parts.at[f.out_part], f.dim), branch, rows(from, f.parts.at[f.stats_part], 4), go, gh, rows(to, parts.at[dx_part], f.dim),
                                   dy_part < 0 ? k::RowsArg{} : rows(to, parts.at[dy_part], f.dim), s);
    }
};
std::vector<Var> NormsOp::grad(const std::vector<Var> &x, const Var &y, const Var &gy) {
    std::vector<Var> arrived(parts.at.size());
    if (!arrivals(gy, parts, &arrived)) {
        arrived.assign(parts.at.size(), Var());
        for (int i : {out_part, h_part})
            if (i >= 0) arrived[i] = slice(gy, 0, parts.at[i], parts.at[i] + parts.size[i]);
    }
    auto op = std::make_shared<NormsGradOp>();
    op->forward = std::make_shared<NormsOp>(*this);
    std::vector<Var> in = x;
    in[0] = y;
    for (int i : {out_part, h_part}) {
        if (i < 0 || !arrived[i].defined()) continue;
        (i == out_part ? op->go_at : op->gh_at) = (int)in.size();
        in.push_back(arrived[i]);
    }
    op->dx_part = op->parts.add(rows * dim);
    if (y_at >= 0) op->dy_part = op->parts.add(rows * dim);
    for (int i = 0; i < kNormOperands; ++i) op->sum_part[i] = operand_at[i] < 0 || i == kSeed ? -1 : op->parts.add(x[operand_at[i]].size());
    for (const Var &v : in) op->in.push_back(v.desc);
    op->out = TensorDesc({op->parts.total}, SAGE_F32);
    const Var all = Var::from_op(op, in);
    std::vector<Var> found(x.size());
    found[0] = op->parts.view(all, op->dx_part, x[0].extents());
    if (y_at >= 0) found[y_at] = op->parts.view(all, op->dy_part, x[y_at].extents());
    for (int i = 0; i < kNormOperands; ++i)
        if (op->sum_part[i] >= 0) found[operand_at[i]] = op->parts.view(all, op->sum_part[i], x[operand_at[i]].extents());
    return found;
}

struct HeadGradOp : Operator {  // inputs hidden, weight, ids, the forward result, its gradient -> dhidden, dweight
    float scale;
    Parts parts;
    const char *name() const override { return "head_log_probs_grad"; }
    std::vector<Var> grad(const std::vector<Var> &, const Var &, const Var &) override { shape_fail("head_log_probs is differentiated once"); }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor hold[5];
        k::Head a;
        k::RowsArg kept, gy;
        const long long rows = in[0].shape.extents[0], width = in[0].shape.extents[1], vocab = in[1].shape.extents[0];
        sage_status st = rows_of(ctx, x[0], rows, width, &hold[0], &a.hidden);
        if (!st) st = rows_of(ctx, x[1], vocab, width, &hold[1], &a.weight);
        if (!st) st = vector_of(ctx, x[2], &hold[2], &a.ids);
        if (!st) st = rows_of(ctx, x[3], rows, 4, &hold[3], &kept);
        if (!st) st = rows_of(ctx, x[4], rows, 4, &hold[4], &gy);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (!st) st = parts.clear_gaps(ctx, (float *)y->ptr());
        if (st) return st;
        a.scale = scale;
        float *to = (float *)y->ptr(), *from = (float *)kept.ptr, *g = (float *)gy.ptr;
        return k::head_log_probs_grad(ctx, a, k::RowsArg{from + 2, SAGE_F32, rows, 2, kept.pitch}, k::VectorArg{from + 1, kept.pitch}, k::VectorArg{g, gy.pitch}, k::VectorArg{g + 1, gy.pitch},
                                      k::RowsArg{to + parts.at[0], SAGE_F32, rows, width, width}, k::RowsArg{to + parts.at[1], SAGE_F32, vocab, width, width});
    }
};
struct HeadOp : Operator {  // inputs hidden [R, D], weight [V, D], ids [R] or [R, 1] -> [R, 4]
    float scale;
    const char *name() const override { return "head_log_probs"; }
    std::vector<Var> grad(const std::vector<Var> &x, const Var &y, const Var &gy) override {
        auto op = std::make_shared<HeadGradOp>();
        op->scale = scale;
        op->parts.add(x[0].size());
        op->parts.add(x[1].size());
        op->in = {x[0].desc, x[1].desc, x[2].desc, y.desc, gy.desc};
        op->out = TensorDesc({op->parts.total}, SAGE_F32);
        const Var all = Var::from_op(op, {x[0], x[1], x[2], y, gy});
        return {op->parts.view(all, 0, x[0].extents()), op->parts.view(all, 1, x[1].extents()), Var()};
    }
    sage_status compute(const std::vector<Tensor> &x, Context &ctx, Tensor *y) override {
        Tensor hold[3];
        k::Head a;
        const Shape &h = in[0].shape, &w = in[1].shape;
        sage_status st = rows_of(ctx, x[0], h.extents[0], h.extents[1], &hold[0], &a.hidden);
        if (!st) st = rows_of(ctx, x[1], w.extents[0], w.extents[1], &hold[1], &a.weight);
        if (!st) st = vector_of(ctx, x[2], &hold[2], &a.ids);
        if (!st) st = Tensor::uninit(ctx, out, y);
        if (st) return st;
        a.scale = scale;
        return k::head_log_probs(ctx, a, column(*y, 0), column(*y, 1), k::RowsArg{(float *)y->ptr() + 2, SAGE_F32, h.extents[0], 2, 4});
    }
};

}  // namespace

Var ops::dropout(const Var &x, const Var &seed, float p, unsigned long long site) {
    if (x.dtype() != SAGE_F32 || x.rank() < 1) shape_fail("dropout: f32 with one axis at least is needed");
    if (!seed.defined()) shape_fail("dropout: a seed is needed");
    check_dropout(seed, p, "dropout");
    auto op = std::make_shared<DropoutOp>();
    op->p = p;
    op->site = site;
    op->in = {x.desc, seed.desc};
    op->out = x.desc.pristine();
    return Var::from_op(op, {x, seed});
}

void ops::block_norms(const Var &x, const Var &y, const BlockNorms &n, Var *out, Var *h) {
    const char *what = "block_norms";
    const auto fail = [&](const char *why) { shape_fail(std::string(what) + ": " + why); };
    if (x.dtype() != SAGE_F32 || x.rank() < 1) fail("the stream must be f32 [.., width]");
    const long long dim = x.extents().back(), rows = dim ? x.size() / dim : 0;
    if (dim < 1 || dim > k::kMaxNormColumns || rows < 1) fail("rows of 1 to 16384 columns are needed");
    check_rows(rows, dim, what);
    if (y.defined() && (y.dtype() != SAGE_F32 || y.extents() != x.extents())) fail("the block's output must be f32 with the stream's extents");
    for (int kind : {n.after, n.before})
        if (kind < SAGE_NORM_NONE || kind > SAGE_NORM_LAYER) fail("no such norm");
    if (!(n.eps > 0.f) || !std::isfinite(n.eps) || !std::isfinite(n.scale)) fail("eps must be positive and finite, the residual scale finite");
    check_dropout(n.seed, n.p, what);
    if (!y.defined() && (n.after != SAGE_NORM_NONE || n.gate.defined() || n.p > 0.f)) fail("the norm after, the gate and dropout need a block's output");
    auto op = std::make_shared<NormsOp>();
    op->after = n.after;
    op->before = n.before;
    op->scale = n.scale;
    op->eps = n.eps;
    op->p = n.p;
    op->site = n.site;
    op->rows = rows;
    op->dim = dim;
    std::vector<Var> in = {x};
    if (y.defined()) {
        op->y_at = 1;
        in.push_back(y);
    }
    const Var *operands[kNormOperands] = {&n.after_weight, &n.after_bias, &n.before_weight, &n.before_bias, &n.gate, &n.seed};
    for (int i = 0; i < kNormOperands; ++i) {
        const Var &v = *operands[i];
        op->operand_at[i] = -1;
        if (!v.defined() || (i == kSeed && !(n.p > 0.f))) continue;
        if (i != kSeed) {
            if (v.dtype() != SAGE_F32) fail("weights, biases and gates must be f32");
            if (i < kGate && (v.rank() != 1 || v.size() != dim)) fail("a weight or bias does not have one element for each column");
            if (i < kGate && (i < kBeforeWeight ? n.after : n.before) == SAGE_NORM_NONE) fail("a weight or bias is given without its norm");
            if (i == kGate && (v.rank() < 1 || v.rank() > 2 || v.extents().back() != dim || !v.size() || rows % (v.size() / dim))) fail("the gate must be [width], or [groups, width] whose groups divide the rows");
        }
        op->operand_at[i] = (int)in.size();
        in.push_back(v);
    }
    op->out_part = op->parts.add(rows * dim);
    if (n.before != SAGE_NORM_NONE) op->h_part = op->parts.add(rows * dim);
    op->stats_part = op->parts.add(rows * 4);
    for (const Var &v : in) op->in.push_back(v.desc);
    op->out = TensorDesc({op->parts.total}, SAGE_F32);
    const Var all = Var::from_op(op, in);
    *out = op->parts.view(all, op->out_part, x.extents());
    *h = op->h_part < 0 ? Var() : op->parts.view(all, op->h_part, x.extents());
}

Var ops::head_log_probs(const Var &hidden, const Var &weight, const Var &ids, float scale) {
    if (hidden.rank() != 2 || hidden.dtype() != SAGE_F32 || weight.rank() != 2 || weight.dtype() != SAGE_F32 || weight.extents()[1] != hidden.extents()[1])
        shape_fail("head_log_probs: hidden states f32 [rows, width] and a weight f32 [tokens, width] are needed");
    check_ids(ids, "head_log_probs");
    check_rows(hidden.extents()[0], hidden.extents()[1], "head_log_probs");
    check_rows(weight.extents()[0], 0, "head_log_probs");
    if (ids.rank() < 1 || ids.size() != hidden.extents()[0] || ids.extents()[0] != hidden.extents()[0]) shape_fail("head_log_probs: one token id for each row is needed");
    if (!k::is_scale(scale)) shape_fail("head_log_probs: the scale must be positive and finite, also times log2(e)");
    if (!weight.size() || !hidden.size()) shape_fail("head_log_probs: rows without tokens or columns");
    auto op = std::make_shared<HeadOp>();
    op->scale = scale;
    op->in = {hidden.desc, weight.desc, ids.desc};
    op->out = TensorDesc({hidden.extents()[0], 4}, SAGE_F32);
    return Var::from_op(op, {hidden, weight, ids});
}

Var ops::embedding(const Var &table, const Var &ids, float scale) {
    if (table.rank() != 2 || table.dtype() != SAGE_F32) shape_fail("embedding: the table must be f32 [tokens, width]");
    check_ids(ids, "embedding");
    check_rows(table.extents()[0], table.extents()[1], "embedding");
    check_rows(ids.size(), 0, "embedding");
    if (!std::isfinite(scale)) shape_fail("embedding: the scale must be finite");
    auto op = std::make_shared<EmbeddingOp>();
    op->scale = scale;
    Array e = ids.extents();
    e.push_back(table.extents()[1]);
    if (e.size() > SAGE_MAX_DIMS) shape_fail("embedding: too many axes");
    op->in = {table.desc, ids.desc};
    op->out = TensorDesc(e, SAGE_F32);
    return Var::from_op(op, {table, ids});
}

Var ops::token_log_probs(const Var &logits, const Var &ids, float scale) {
    if (logits.rank() != 2 || logits.dtype() != SAGE_F32) shape_fail("token_log_probs: logits must be f32 [rows, tokens]");
    check_ids(ids, "token_log_probs");
    check_rows(logits.extents()[0], logits.extents()[1], "token_log_probs");
    if (ids.rank() < 1 || ids.size() != logits.extents()[0] || ids.extents()[0] != logits.extents()[0]) shape_fail("token_log_probs: one token id for each row is needed");
    if (!k::is_scale(scale)) shape_fail("token_log_probs: the scale must be positive and finite, also times log2(e)");
    if (!logits.extents()[1]) shape_fail("token_log_probs: rows without tokens");
    auto op = std::make_shared<TokenLogProbsOp>();
    op->scale = scale;
    op->in = {logits.desc, ids.desc};
    op->out = TensorDesc({logits.extents()[0], 4}, SAGE_F32);
    return Var::from_op(op, {logits, ids});
}

Var ops::top_tokens(const Var &logits, long long k) {
    if (logits.rank() != 2 || logits.dtype() != SAGE_F32) shape_fail("top_tokens: logits must be f32 [rows, tokens]");
    check_rows(logits.extents()[0], logits.extents()[1], "top_tokens");
    if (k < 1 || k > k::kMaxTop || k > logits.extents()[1]) shape_fail("top_tokens: 1 to 32 tokens of a row, and no more than it has");
    auto op = std::make_shared<TopTokensOp>();
    op->in = {logits.desc};
    op->out = TensorDesc({logits.extents()[0], k}, SAGE_U32);
    return Var::from_op(op, {logits});
}

}  // namespace sage
