"""Operators at the two ends of a language model and of its training step, on device tensors (include/sage_cuda.h, "language
models"): token embedding and its gradient, log probabilities of given tokens with entropy, alternatives and gradient, AdamW
over many tensors.

Every operand is a DeviceTensor of one context: `Context.tensor` / `Context.empty`, or `Context.borrow` of another package's
memory.  Results go into tensors that the caller gives; calls enqueue work on the context's stream and return.  The lazy-graph
forms of the same operators are `sage_b200.embedding`, `token_log_probs`, `top_tokens` and `AdamW`.
"""
import ctypes

from . import CTensor, SageError, lib

_F = ctypes.c_float


def _ref(t):
    return None if t is None else t.ref()


def embedding(table, ids, y, scale=1.0):
    """y[t, :] = scale * table[ids[t], :]; an id outside the table gives zeros."""
    y.ctx._ck(lib.sage_embedding(y.ctx.h, table.ref(), ids.ref(), _F(scale), y.ref()))


def embedding_grad(g, ids, dtable, scale=1.0, add=False):
    """dtable[v, :] = scale * the sum of g[t, :] over the tokens with ids[t] = v, or that added to dtable.  The order of the
    sums is fixed: the same inputs give the same bits."""
    g.ctx._ck(lib.sage_embedding_grad(g.ctx.h, g.ref(), ids.ref(), _F(scale), 1 if add else 0, dtable.ref()))


def token_log_probs(logits, ids, log_probs, entropy=None, stats=None, top_ids=None, top_log_probs=None, scale=1.0):
    """Log probabilities of ids[r] under softmax(scale * logits[r, :]), with the rows' entropies, what the gradient reads
    (`stats`, [rows, 2]) and the largest alternatives (ids and log probabilities, [rows, k]) where they are asked for."""
    logits.ctx._ck(lib.sage_token_log_probs(logits.ctx.h, logits.ref(), ids.ref(), _F(scale), log_probs.ref(), _ref(entropy), _ref(stats), _ref(top_ids), _ref(top_log_probs)))


def token_log_probs_grad(logits, ids, stats, entropy, g_log_probs, g_entropy, dlogits, scale=1.0):
    """The gradient of g_log_probs . log_probs + g_entropy . entropy with respect to the logits; dlogits may be the logits."""
    logits.ctx._ck(lib.sage_token_log_probs_grad(logits.ctx.h, logits.ref(), ids.ref(), _F(scale), stats.ref(), _ref(entropy), _ref(g_log_probs), _ref(g_entropy), dlogits.ref()))


def token_log_probs_and_grad(logits, ids, g_log_probs, g_entropy, log_probs, entropy, dlogits, scale=1.0):
    """Values and gradient in one call, for weights g_log_probs and g_entropy that are known before the values."""
    logits.ctx._ck(lib.sage_token_log_probs_and_grad(logits.ctx.h, logits.ref(), ids.ref(), _F(scale), _ref(g_log_probs), _ref(g_entropy), log_probs.ref(), _ref(entropy), dlogits.ref()))


_OPERANDS = ("param", "grad", "m", "v", "m_scale", "v_scale", "copy")


class _AdamWTensor(ctypes.Structure):
    _fields_ = [(n, CTensor) for n in _OPERANDS]


class _AdamWOpts(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "grad_scale")] + [("step", ctypes.c_int64)]


def adamw_tensor(param, grad, m, v, m_scale=None, v_scale=None, copy=None):
    """One tensor of an update: parameters (f32), gradient, states (f32, or i8 / u8 codes with f32 scales for each 256 elements,
    zeroed before the first step) and, if wanted, a 16-bit copy of the parameters."""
    return (param, grad, m, v, m_scale, v_scale, copy)


class AdamWTensors:
    """The tensors of an update as the library takes them; made once, used for every step until one of them is released."""

    def __init__(self, ctx, tensors):
        self.ctx, self.tensors = ctx, list(tensors)  # keeps the operands alive
        self.array = (_AdamWTensor * max(len(self.tensors), 1))()
        for slot, operands in zip(self.array, self.tensors):
            for name, t in zip(_OPERANDS, operands):
                if t is not None:
                    t.fill(getattr(slot, name))
        self.handles = [t.buf for operands in self.tensors for t in operands if t is not None]
        self.released = ctx.released

    def ready(self):
        """The array, behind a look at the operands if any tensor was released since the last one."""
        if self.released != self.ctx.released:
            if not all(self.handles):
                raise SageError(1, "adamw_step: an operand was released")
            self.released = self.ctx.released
        return self.array


def adamw_step(tensors, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=1.0):
    """One AdamW update of all tensors in place; `step` counts from 1."""
    o = _AdamWOpts(lr, beta1, beta2, eps, weight_decay, grad_scale, step)
    tensors.ctx._ck(lib.sage_adamw_step(tensors.ctx.h, tensors.ready(), len(tensors.tensors), ctypes.byref(o)))


def adamw_states(m, m_scale, v, v_scale, m_out, v_out):
    """The f32 values that 8-bit states stand for."""
    m.ctx._ck(lib.sage_adamw_states(m.ctx.h, m.ref(), m_scale.ref(), v.ref(), v_scale.ref(), m_out.ref(), v_out.ref()))
