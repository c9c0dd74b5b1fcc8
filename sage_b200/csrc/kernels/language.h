// Host launchers of the language-model operators: token embedding and its gradient (embedding.cu), log probabilities of given
// tokens with entropy, alternatives and gradient (log_probs.cu), AdamW over many tensors (adamw.cu).  Pointers are raw device
// addresses with the offset applied, strides in elements; the caller (abi/language_abi.cc, graph/ops_language.cc) has checked
// types, extents and that views lie in their buffers.
#pragma once
#include "kernels.h"

namespace sage {
namespace k {

// Rows, tokens or columns: the kernels number them in 32 bits, with room for a last round's.
constexpr long long kMaxRows = 0x7fff0000;

struct RowsArg {  // [rows, cols], contiguous along a row
    void *ptr = nullptr;
    int dtype = SAGE_F32;
    long long rows = 0, cols = 0, pitch = 0;
};
struct VectorArg {  // ptr[i * stride]; null = not given
    void *ptr = nullptr;
    long long stride = 0;
};

// y[t, :] = scale * table[ids[t], :], zeros where ids[t] is outside [0, table.rows)
sage_status embedding(Context &ctx, const RowsArg &table, const VectorArg &ids, float scale, const RowsArg &y);
// dtable[v, :] = (add ? dtable[v, :] : 0) + scale * sum of g[t, :] over ids[t] = v
sage_status embedding_grad(Context &ctx, const RowsArg &g, const VectorArg &ids, float scale, bool add, const RowsArg &dtable);

constexpr int kMaxTop = 32;
constexpr float kLog2E = 1.4426950408889634f;
// Scales of logits: positive, and finite in base 2 too, in which exponentials are taken.
inline bool is_scale(float scale) { return scale > 0.f && scale <= 3.4028235e38f / kLog2E; }
struct LogProbs {  // what has no ptr is not wanted, or (ids) not given
    RowsArg logits;
    VectorArg ids;
    float scale = 1.f;
    VectorArg log_probs, entropy;  // f32
    RowsArg stats;                 // [rows, 2] f32 {max of the logits, sum of exp(scale * (logit - max))}
    int top = 0;
    RowsArg top_ids, top_log_probs;
};
sage_status token_log_probs(Context &ctx, const LogProbs &a);
struct LogProbsGrad {
    RowsArg logits;
    VectorArg ids;
    float scale = 1.f;
    RowsArg stats;
    VectorArg entropy, g_log_probs, g_entropy;
    RowsArg dlogits;
};
sage_status token_log_probs_grad(Context &ctx, const LogProbsGrad &a);
// Both at once: `a.stats` and `a.entropy` are not read; log_probs and entropy (null = not wanted) are written.
sage_status token_log_probs_and_grad(Context &ctx, const LogProbsGrad &a, const VectorArg &log_probs, const VectorArg &entropy);

constexpr int kAdamWBlock = 256;  // elements of an 8-bit state that share a scale
struct AdamWSlot {
    float *p = nullptr;
    const void *g = nullptr;
    void *m = nullptr, *v = nullptr;
    float *m_scale = nullptr, *v_scale = nullptr;
    void *copy = nullptr;
    long long n = 0;
    short g_dtype = SAGE_F32, copy_dtype = SAGE_F32;
    int wide = 0;  // filled in by the launcher: whole blocks lie on vector boundaries
};
struct AdamWRule {
    float beta1, one_minus_beta1, beta2, one_minus_beta2;
    float keep;         // 1 - lr * weight_decay
    float step_size;    // lr / (1 - beta1^t)
    float root_factor;  // 1 / sqrt(1 - beta2^t)
    float eps, grad_scale;
    float minus_zero = -0.f;
};
AdamWRule adamw_rule(double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale, long long step);
sage_status adamw_step(Context &ctx, const AdamWSlot *slots, int count, bool states8, const AdamWRule &rule);
sage_status adamw_states(Context &ctx, const void *m, const float *m_scale, const void *v, const float *v_scale, long long n, float *m_out, float *v_out);

}  // namespace k
}  // namespace sage
