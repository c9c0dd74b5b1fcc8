"""A plain implementation in 64 bits of log probabilities from hidden states and their gradient, and how far a correct kernel may be from it.

Products of 16-bit operands are summed in f32 on the tensor cores, which add 16 products at a time and cut what lies below the last place: a sum over
K is off by (K / 8 + 32) 2U of the sum of its terms' sizes at most.  Products of f32 operands (two pieces of 11 bits each): the same bound holds."""
import numpy as np

from language_oracle import ROUND, U, LogProbs

TINY = 2.0 ** -149


def product_tol(a, b, k):
    return (k / 8 + 32) * 2 * U * (np.abs(a) @ np.abs(b))


class Head(LogProbs):
    def __init__(self, hidden, weight, ids, scale, kind):
        self.h, self.w, self.kind = np.asarray(hidden, np.float64), np.asarray(weight, np.float64), kind
        x = self.h @ self.w.T
        super().__init__(x, ids, scale)
        off = self.scale * product_tol(self.h, self.w.T, self.h.shape[1])  # of a scaled logit
        mean = (self.p * off).sum(1, keepdims=True)
        self.tol_log_p = self.tol_log_p + off + mean
        self.rel_p = self.rel_p + 1.1 * (off + mean)  # (small against 1)
        spread = np.abs(np.where(self.p > 0, self.log_p, 0.0) + self.entropy[:, None])
        self.tol_entropy = self.tol_entropy + (self.p * spread * (off + mean)).sum(1)

    def gradients(self, gl, ge, out):
        """{name: (gradient, its bound before it is stored)}"""
        r, v = self.x.shape
        gl = np.zeros(r) if gl is None else np.asarray(gl, np.float64)
        ge = np.zeros(r) if ge is None else np.asarray(ge, np.float64)
        gl = np.where(self.scored, gl, 0.0)[:, None]
        ge = ge[:, None]
        h = self.entropy[:, None]
        ln_p = np.where(self.p > 0, self.log_p, 0.0)
        delta = np.zeros((r, v))
        delta[np.arange(r)[self.scored], self.ids[self.scored]] = 1.0
        q = gl * (delta - self.p) - ge * self.p * (ln_p + h)
        size = np.abs(gl) * (delta + self.p) + np.abs(ge) * self.p * (np.abs(ln_p) + np.abs(h))
        t = self.rel_p * (np.abs(gl) * self.p + np.abs(ge) * self.p * (np.abs(ln_p) + np.abs(h) + 1)) + np.abs(ge) * self.p * (self.tol_log_p + self.tol_entropy[:, None]) + 8 * U * size
        rel, absolute = ROUND[self.kind]
        if self.kind == "f16":  # stored by a power of two that leaves 2^13 at least for the largest possible
            absolute = absolute * float((np.abs(gl) + np.abs(ge) * (h + 0.5)).max()) / 2.0 ** 13
        t = t + rel * (np.abs(q) + t) + absolute + TINY
        c = self.scale
        found = {"dhidden": (c * (q @ self.w), c * (t @ np.abs(self.w) + product_tol(q, self.w, v))),
                 "dweight": (c * (q.T @ self.h), c * (t.T @ np.abs(self.h) + product_tol(q.T, self.h, r)))}
        return {n: (g, tol + ROUND[out][0] * (np.abs(g) + tol) + ROUND[out][1] + 4 * U * np.abs(g)) for n, (g, tol) in found.items()}
