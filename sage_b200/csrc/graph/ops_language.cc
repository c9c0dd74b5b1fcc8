// Language-model operators of the lazy graph: token embedding, log probabilities of given tokens with entropy, alternatives
// (kernels/language.h).  No counterpart in the reference, whose embedding is a gather (layers.rs:427-452) with a scatter as its
// gradient and whose loss is composed (nn.rs:70-82).
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

}  // namespace

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
