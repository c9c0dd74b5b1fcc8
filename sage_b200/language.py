"""Operators of a language model's training step beside its products and attention, on device tensors (include/sage_cuda.h, "language
models"): token embedding and its gradient, log probabilities of given tokens with entropy, alternatives and gradient, the same from
hidden states, dropout, the norms around a block with gate and residual scale and their gradient, AdamW over many tensors.

Every operand is a DeviceTensor of one context: `Context.tensor` / `Context.empty`, or `Context.borrow` of another package's
memory.  Results go into tensors that the caller gives; calls enqueue work on the context's stream and return.  The lazy-graph
forms of the same operators are `sage_b200.embedding`, `token_log_probs`, `top_tokens`, `head_log_probs`, `dropout`, `block_norms`
and `AdamW`.
"""
import ctypes

from . import CTensor, SageError, lib

_F = ctypes.c_float
_U64 = ctypes.c_uint64


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


def head_log_probs(hidden, weight, ids, log_probs, entropy=None, stats=None, scale=1.0):
    """token_log_probs of the logits hidden weight^T [rows, vocab], which are made in pieces and not kept: hidden [rows, D], weight [vocab, D]."""
    hidden.ctx._ck(lib.sage_head_log_probs(hidden.ctx.h, hidden.ref(), weight.ref(), ids.ref(), _F(scale), log_probs.ref(), _ref(entropy), _ref(stats)))


def head_log_probs_grad(hidden, weight, ids, stats, entropy, g_log_probs, g_entropy, dhidden=None, dweight=None, scale=1.0):
    """The gradient of g_log_probs . log_probs + g_entropy . entropy with respect to the hidden states and the weight, from what head_log_probs left in
    `stats` and `entropy`."""
    hidden.ctx._ck(lib.sage_head_log_probs_grad(hidden.ctx.h, hidden.ref(), weight.ref(), ids.ref(), _F(scale), stats.ref(), _ref(entropy), _ref(g_log_probs), _ref(g_entropy),
                                                _ref(dhidden), _ref(dweight)))


def dropout(x, y, seed, p, site=0):
    """y = x / (1 - p) where an element stays, else 0; the same call makes the gradient of it.  Which elements stay follows from their places, `site`
    and what `seed` (u32 or i32 [2]) holds when the call is run; shares are multiples of 2^-16.  y may be x."""
    x.ctx._ck(lib.sage_dropout(x.ctx.h, x.ref(), y.ref(), _ref(seed), _F(p), _U64(site)))


_NORMS = {None: 0, "none": 0, "rms": 1, "layer": 2}
_NORM_OPERANDS = ("after_weight", "after_bias", "before_weight", "before_bias", "gate", "seed")


class _BlockNormsOpts(ctypes.Structure):
    _fields_ = [(n, CTensor) for n in _NORM_OPERANDS] + [("after", ctypes.c_int32), ("before", ctypes.c_int32)] + \
               [(n, _F) for n in ("residual_scale", "eps", "p")] + [("site", _U64)]


class _BlockNormsSums(ctypes.Structure):
    _fields_ = [(n, CTensor) for n in _NORM_OPERANDS[:-1]]


def _filled(struct, names, operands):
    """The struct with those operands that are there, and their handles, which it needs alive."""
    held = [t for t in operands if t is not None]
    for name, t in zip(names, operands):
        if t is not None:
            if not t.buf:
                raise SageError(1, "block_norms: %s was released" % name)
            t.fill(getattr(struct, name))
    return [t.buf for t in held], held


class BlockNorms:
    """How a block of a model is joined to its residual stream, made once and used for every call until one of its tensors is released:
    out = residual_scale * x + gate * dropout(A(y)), h = B(out), with A = `after` and B = `before` one of "rms", "layer" and None.  Weights and
    biases are f32 [D], the gate f32 [D] or [G, D], `seed` and `site` dropout's."""

    def __init__(self, ctx, after=None, after_weight=None, after_bias=None, before=None, before_weight=None, before_bias=None, gate=None, residual_scale=1.0, eps=1e-5,
                 p=0.0, seed=None, site=0):
        for name in (after, before):
            if name not in _NORMS:
                raise SageError(1, "block_norms: no norm is called %r" % (name,))
        self.ctx, self.opts = ctx, _BlockNormsOpts(after=_NORMS[after], before=_NORMS[before], residual_scale=residual_scale, eps=eps, p=p, site=site)
        self.handles, self.held = _filled(self.opts, _NORM_OPERANDS, (after_weight, after_bias, before_weight, before_bias, gate, seed))
        self.released = ctx.released

    def ready(self):
        """The struct, behind a look at the operands if any tensor was released since the last one."""
        if self.released != self.ctx.released:
            if not all(self.handles):
                raise SageError(1, "block_norms: an operand was released")
            self.released = self.ctx.released
        return ctypes.byref(self.opts)


def block_norms(norms, x, y, out, h=None, stats=None):
    """One call for all rows [R, D]: the stream x and the block's output y give the stream behind the block, the next block's input, and what the gradient
    reads (stats, [R, 4]).  y None: just h = B(x).  out may be x, h may be y."""
    norms.ctx._ck(lib.sage_block_norms(norms.ctx.h, norms.ready(), x.ref(), _ref(y), _ref(out), _ref(h), _ref(stats)))


def block_norms_grad(norms, out, y, stats, g_out, g_h, dx=None, dy=None, dgate=None, dafter_weight=None, dafter_bias=None, dbefore_weight=None, dbefore_bias=None):
    """From what block_norms left in out and stats, y, and the gradients of out and h (either may be None): those of x, of y, and the sums over rows that
    are those of the gate, the weights and the biases (f32), each where it is asked for."""
    sums = _BlockNormsSums()
    _filled(sums, _NORM_OPERANDS, (dafter_weight, dafter_bias, dbefore_weight, dbefore_bias, dgate))
    norms.ctx._ck(lib.sage_block_norms_grad(norms.ctx.h, norms.ready(), out.ref(), _ref(y), stats.ref(), _ref(g_out), _ref(g_h), _ref(dx), _ref(dy), ctypes.byref(sums)))


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
