"""Plain implementations in 64 bits of the language-model operators, and how far a correct kernel that holds its sums in 32 bits may
be from them: u = 2^-24 is one rounding of f32."""
import numpy as np

U = 2.0 ** -24
ROUND = {"f32": (U, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}  # relative; absolute among the subnormals


def bf16_bits(x):
    """f32 -> bf16 bits, to nearest even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def bf16_values(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def stored(x, kind):
    """(what is uploaded, the f32 values it stands for)"""
    x = np.asarray(x, np.float32)
    if kind == "bf16":
        bits = bf16_bits(x)
        return bits, bf16_values(bits)
    if kind == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float32)
    return x, x


def values(raw, kind):
    return bf16_values(raw) if kind == "bf16" else np.asarray(raw).astype(np.float32)


def embedding_grad(g, ids, vocab, scale, start=None):
    """The gradient, and the bound: a sum of n terms in any order is off by (n - 1) u sum |g| at most, then come the scale, the
    last addition and what that holds."""
    out = np.zeros((vocab, g.shape[1])) if start is None else start.astype(np.float64)
    big, count = np.zeros((vocab, g.shape[1])), np.zeros((vocab, 1))
    ok = (ids >= 0) & (ids < vocab)
    np.add.at(out, ids[ok], scale * g[ok].astype(np.float64))
    np.add.at(big, ids[ok], abs(scale) * np.abs(g[ok].astype(np.float64)))
    np.add.at(count, ids[ok], 1.0)
    return out, (count + 2) * U * big + 2 * U * (np.abs(out) + (0 if start is None else np.abs(start)))


class LogProbs:
    """Of rows x (f32 values), tokens ids, a scale: log probabilities, entropy, alternatives, gradient, and their bounds.

    d = scale (x - max x) carries two roundings, exp(d) then |d| 2u and the function's own 4u; a thread's sum has at most
    vocab / 128 terms and a tree above it (16 levels at most)."""

    def __init__(self, x, ids, scale):
        x = np.asarray(x, np.float64)
        self.ids, self.scale, self.x = np.asarray(ids), float(np.float32(scale)), x
        r, v = x.shape
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            m = x.max(1, keepdims=True)
            self.none = np.isneginf(m)
            d = self.scale * (x - np.where(self.none, 0.0, m))
            e = np.exp(d)
            s = e.sum(1, keepdims=True)
            ln_s = np.log(s)
            self.log_p = np.where(self.none | (d - ln_s < -float(np.finfo(np.float32).max)), -np.inf, d - ln_s)  # f32 holds no less
            self.p = np.where(self.none, 0.0, e / np.where(s == 0, 1, s))
            dz = np.where(e > 0, np.abs(d), 0.0)  # |d| where it counts
            p_ln_p = np.where(self.p > 0, self.p * self.log_p, np.where(np.isnan(self.p), np.nan, 0.0))
            self.entropy = np.where(self.none[:, 0], 0.0, -p_ln_p.sum(1))
            terms = v / 128 + 16
            self.rel_s = (2 * U * (self.p * (dz + 4)).sum(1, keepdims=True) + terms * U)
            self.tol_log_p = 4 * U * np.where(np.isfinite(d), np.abs(d), 0.0) + self.rel_s + 4 * U * np.abs(ln_s)
            weighted = (self.p * dz).sum(1, keepdims=True)
            self.tol_entropy = (2 * U * (self.p * dz * (dz + 6)).sum(1, keepdims=True) + 2 * terms * U * weighted + self.rel_s * (1 + weighted)
                                + 4 * U * (np.abs(ln_s) + weighted))[:, 0]
            self.rel_p = 2 * U * (dz + 6) + self.rel_s
        self.m, self.s = m[:, 0], s[:, 0]
        ok = (self.ids >= 0) & (self.ids < v)
        self.scored = ok
        at = np.where(ok, self.ids, 0).astype(np.int64)
        self.log_probs = np.where(ok, self.log_p[np.arange(r), at], 0.0)
        self.tol_log_probs = self.tol_log_p[np.arange(r), at]

    def top(self, k):
        x = np.where(np.isnan(self.x), -np.inf, self.x)
        order = np.argsort(-x, axis=1, kind="stable")[:, :k]
        return order, np.take_along_axis(self.log_p, order, 1), np.take_along_axis(self.tol_log_p, order, 1)

    def grad(self, gl, ge, kind):
        r, v = self.x.shape
        gl = np.where(self.scored, np.broadcast_to(np.asarray(gl, np.float64), (r,)), 0.0)[:, None]
        ge = np.broadcast_to(np.asarray(ge, np.float64), (r,))[:, None]
        delta = np.zeros((r, v))
        delta[np.arange(r)[self.scored], self.ids[self.scored].astype(np.int64)] = 1.0
        h = self.entropy[:, None]
        with np.errstate(invalid="ignore"):
            inner = np.where(self.p > 0, self.log_p + h, np.where(np.isnan(self.p), np.nan, 0.0))
            g = self.scale * (gl * (delta - self.p) - ge * self.p * inner)
            g = np.where(self.none, 0.0, g)
            off = self.scale * (np.abs(gl) * (self.p * self.rel_p + 2 * U * (delta + self.p))
                                + np.abs(ge) * self.p * (np.abs(inner) * (self.rel_p + 4 * U) + self.tol_log_p + self.tol_entropy[:, None]))
            off = np.where(self.none, 0.0, off)  # nothing to round where there is no distribution
        rel, small = ROUND[kind]
        return g, off + rel * np.abs(g) + rel * off + small + 1e-37


def adamw_encode(x, top):
    """Codes and scales of 8-bit states, operation for operation in f32."""
    f = np.float32
    n = x.size
    pad = np.zeros(-(-n // 256) * 256, f)
    pad[:n] = x
    b = pad.reshape(-1, 256)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        big = np.abs(b).max(1, keepdims=True)
        fine, some = np.isfinite(big), big >= f(2.0 ** -100)
        factor = np.where(fine & some, f(1) / np.where(some & fine, big, f(1)) * f(top * top), f(0)).astype(f)
        c = np.rint(np.sqrt(np.where(fine, np.abs(b), f(0)) * factor)).astype(f)
        c = np.minimum(c, f(top))
        if top == 255:
            c = np.where((b > 0) & some & fine, np.maximum(c, f(1)), c)
        c = np.where(fine & (b < 0), -c, c)
        scale = np.where(fine, np.where(some, big * (f(1) / f(top * top)), f(0)), f("nan")).astype(f)
    return c.reshape(-1)[:n].astype(np.int8 if top == 127 else np.uint8), scale[:, 0]


def adamw_decode(c, scale):
    i = c.astype(np.float32)
    return np.repeat(scale, 256)[: c.size] * (i * np.abs(i))


def adamw_f32(m, v, g, beta1, beta2, grad_scale):
    """Moments as the kernel rounds them."""
    f = np.float32
    with np.errstate(invalid="ignore", over="ignore"):
        g = g * f(grad_scale)
        m = m * f(beta1) + g * f(1.0 - beta1)
        v = v * f(beta2) + (g * g) * f(1.0 - beta2)
    return m, v


def adamw_64(p, m, v, g, o):
    """Parameters and moments in 64 bits, and the parameters' bound: about ten roundings of the update, two of the parameter."""
    g = g.astype(np.float64) * o["grad_scale"]
    m = o["beta1"] * m.astype(np.float64) + (1 - o["beta1"]) * g
    v = o["beta2"] * v.astype(np.float64) + (1 - o["beta2"]) * g * g
    step = o["lr"] * (m / (1 - o["beta1"] ** o["step"])) / (np.sqrt(v / (1 - o["beta2"] ** o["step"])) + o["eps"])
    big = o["lr"] * ((o["beta1"] * np.abs(m) + np.abs(g)) / (1 - o["beta1"] ** o["step"])) / (np.sqrt(v / (1 - o["beta2"] ** o["step"])) + o["eps"])
    return p.astype(np.float64) * (1 - o["lr"] * o["weight_decay"]) - step, m, v, 12 * U * (np.abs(step) + big) + 3 * U * np.abs(p)
