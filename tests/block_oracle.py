"""Plain implementations in 64 bits of dropout and of the norms around a block, and how far a correct kernel that works in 32 bits may be from them:
U = 2^-24 is one rounding of f32; a row's sum has at most 53 steps in a chain (32 columns of a thread, 5 exchanges, 16 warps)."""
import numpy as np

from language_oracle import ROUND, U

CHAIN = 53
RSQRT = 4 * U  # the reciprocal root's own error, 2 units of the last place


def bar_of(p):
    return min(65535, int(np.rint(float(np.float32(p)) * 65536.0)))


def keep(seed, site, n, p):
    """Which of n elements stay: 16 bits of Philox4x32-10 each."""
    u, low = np.uint64, np.uint64(0xffffffff)
    block = np.arange((n + 7) // 8, dtype=u)
    x = [block & low, block >> u(32), np.full_like(block, site & 0xffffffff), np.full_like(block, site >> 32)]
    key = [u(int(s) & 0xffffffff) for s in seed]
    for _ in range(10):
        p0, p1 = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(p1 >> u(32)) ^ x[1] ^ key[0], p1 & low, (p0 >> u(32)) ^ x[3] ^ key[1], p0 & low]
        key = [(key[0] + u(0x9E3779B9)) & low, (key[1] + u(0xBB67AE85)) & low]
    words = np.stack([h for w in x for h in (w & u(0xffff), w >> u(16))], 1).reshape(-1)[:n]
    return words >= bar_of(p)


def factors(seed, site, shape, p):
    if bar_of(p) == 0:
        return np.ones(shape)
    return keep(seed, site, int(np.prod(shape)), p).reshape(shape) * (65536.0 / (65536 - bar_of(p)))


def stored_tol(value, tol, kind):
    """The bound behind a rounding to `kind`."""
    rel, absolute = ROUND[kind]
    return tol + rel * (np.abs(value) + tol) + absolute


def statistics(x, kind, eps):
    """(mean, 1 / deviation) of rows, and their bounds."""
    x = np.asarray(x, np.float64)
    n = x.shape[1]
    if kind == "none":
        return np.zeros((len(x), 1)), np.ones((len(x), 1)), np.zeros((len(x), 1)), np.zeros((len(x), 1))
    mean = x.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(x), 1))
    t_mean = (CHAIN + 2) * U * np.abs(x).mean(1, keepdims=True) if kind == "layer" else 0.0 * mean
    c = x - mean
    var = (c * c).mean(1, keepdims=True)
    # each c is off by t_mean and a rounding; their squares' sum by what that makes, and the chain
    t_var = (2 * np.abs(c) * (t_mean + U * np.abs(c))).mean(1, keepdims=True) + 2 * t_mean ** 2 + (CHAIN + 4) * U * var
    rstd = 1.0 / np.sqrt(var + eps)
    t_rstd = rstd * (np.minimum(1.0, 0.5 * t_var / (var + eps) * 1.01) + RSQRT + U)
    return mean, rstd, t_mean, t_rstd


def unit(x, mean, rstd, t_mean=0.0, t_rstd=0.0):
    c = np.asarray(x, np.float64) - mean
    v = c * rstd
    return v, rstd * t_mean + np.abs(c) * t_rstd + 2 * U * np.abs(v) + rstd * U * (np.abs(x) + np.abs(mean))


class Norms:
    """after, before: "none", "rms", "layer"; weights, biases, gate: f32 or None."""

    def __init__(self, after, before, aw=None, ab=None, bw=None, bb=None, gate=None, scale=1.0, eps=1e-5, p=0.0, seed=(0, 0), site=0):
        self.after, self.before, self.scale, self.eps = after, before, float(np.float32(scale)), float(np.float32(eps))
        f = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
        self.aw, self.ab, self.bw, self.bb, self.gate = f(aw), f(ab), f(bw), f(bb), f(gate)
        self.p, self.seed, self.site = p, seed, site

    def gates(self, rows, dim):
        if self.gate is None:
            return np.ones((1, dim))
        return self.gate[None] if self.gate.ndim == 1 else np.repeat(self.gate, rows // len(self.gate), 0)

    @staticmethod
    def affine(v, t, w, b):
        n = v * (1.0 if w is None else w)
        t = t * (1.0 if w is None else np.abs(w)) + U * np.abs(n)
        if b is not None:
            n = n + b
            t = t + U * (np.abs(n) + np.abs(b))
        return n, t

    def out(self, x, y):
        """(out, its bound before it is stored)"""
        x = np.asarray(x, np.float64)
        out, tol = self.scale * x, 2 * U * np.abs(self.scale * x)
        if y is not None:
            v, t = unit(y, *statistics(y, self.after, self.eps)) if self.after != "none" else (np.asarray(y, np.float64), 0.0)
            n, t = self.affine(v, t, self.aw, self.ab)
            f = np.abs(factors(self.seed, self.site, x.shape, self.p) * self.gates(*x.shape))
            b = n * factors(self.seed, self.site, x.shape, self.p) * self.gates(*x.shape)
            out, tol = out + b, tol + t * f + 4 * U * np.abs(b)
        return out, tol + 2 * U * np.abs(out)

    def h(self, out):
        v, t = unit(out, *statistics(out, self.before, self.eps))
        return self.affine(v, t, self.bw, self.bb)

    @staticmethod
    def through(q, t_q, u, t_u, rstd, kind):
        if kind == "none":
            return q, t_q
        along, mean = (q * u).mean(1, keepdims=True), q.mean(1, keepdims=True) if kind == "layer" else 0.0
        t_along = (t_q * np.abs(u) + np.abs(q) * t_u).mean(1, keepdims=True) + (CHAIN + 3) * U * np.abs(q * u).mean(1, keepdims=True)
        t_mean = (t_q.mean(1, keepdims=True) + (CHAIN + 3) * U * np.abs(q).mean(1, keepdims=True)) if kind == "layer" else 0.0
        g = rstd * (q - mean - u * along)
        return g, rstd * (t_q + t_mean + t_u * np.abs(along) + np.abs(u) * t_along + 4 * U * (np.abs(q) + np.abs(mean) + np.abs(u * along))) + 2 * U * np.abs(g)

    def grad(self, out, y, stats, go, gh):
        """{name: (gradient, its bound)} from the statistics that the forward pass left."""
        out = np.asarray(out, np.float64)
        rows, dim = out.shape
        ma, ra, mb, rb = (np.asarray(stats, np.float64)[:, i:i + 1] for i in range(4))
        G = np.zeros(out.shape) if go is None else np.asarray(go, np.float64)
        t_G, found = np.zeros(out.shape), {}

        def rows_sum(terms, t_terms, groups=1):  # any order: (n - 1) U of the terms' sizes
            n = rows // groups if groups else 1
            cut = lambda a: a.reshape(groups, n, dim).sum(1)  # noqa: E731
            s, t = cut(terms), cut(t_terms) + (n + 2) * U * cut(np.abs(terms))
            return (s, t) if groups > 1 else (s[0], t[0])

        if gh is not None:
            gh = np.asarray(gh, np.float64)
            u, t_u = unit(out, mb, rb)
            found["dbefore_weight"] = rows_sum(gh * u, np.abs(gh) * t_u + U * np.abs(gh * u))
            found["dbefore_bias"] = rows_sum(gh, 0 * gh)
            q = gh * (1.0 if self.bw is None else self.bw)
            g, t = self.through(q, U * np.abs(q), u, t_u, rb, self.before)
            G, t_G = G + g, t + 2 * U * (np.abs(g) + np.abs(G))
        found["dx"] = G * self.scale, abs(self.scale) * t_G + U * np.abs(G * self.scale)
        if y is None:
            return found
        v, t_v = unit(y, ma, ra) if self.after != "none" else (np.asarray(y, np.float64), 0.0 * G)
        n, t_n = self.affine(v, t_v, self.aw, self.ab)
        f, gate = factors(self.seed, self.site, out.shape, self.p), self.gates(rows, dim)
        K, t_K = G * f, t_G * f + U * np.abs(G * f)
        if self.gate is not None:
            found["dgate"] = rows_sum(K * n, t_K * np.abs(n) + np.abs(K) * t_n + 2 * U * np.abs(K * n), 1 if self.gate.ndim == 1 else len(self.gate))
            if self.gate.ndim == 2 and len(self.gate) == 1:
                found["dgate"] = tuple(a[None] for a in found["dgate"])
        t, t_t = K * gate, t_K * np.abs(gate) + U * np.abs(K * gate)
        found["dafter_weight"] = rows_sum(t * v, t_t * np.abs(v) + np.abs(t) * t_v + U * np.abs(t * v))
        found["dafter_bias"] = rows_sum(t, t_t)
        q = t * (1.0 if self.aw is None else self.aw)
        found["dy"] = self.through(q, t_t * (1.0 if self.aw is None else np.abs(self.aw)) + U * np.abs(q), v, t_v, ra, self.after)
        return found
