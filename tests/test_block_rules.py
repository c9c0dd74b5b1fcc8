"""What dropout and the norms around a block refuse and launch (a planning context sees all of it), and their oracle's gradients against differences."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import block_oracle as B
from test_language_arguments import refused


@pytest.fixture()
def ctx():
    c = S.Context(-1)
    yield c
    c.close()


def test_dropout_refusals(ctx):
    x, y, s = ctx.empty((4, 8)), ctx.empty((4, 8)), ctx.empty((2,), S.U32)
    L.dropout(x, y, s, 0.1)
    L.dropout(x, x, None, 0.0)
    for p in (-0.1, 1.0, float("nan"), float("inf")):
        refused(L.dropout, x, y, s, p, match="p is not")
    refused(L.dropout, x, y, None, 0.1, match="seed")
    refused(L.dropout, x, y, ctx.empty((3,), S.U32), 0.1, match="seed")
    refused(L.dropout, x, y, ctx.empty((2,)), 0.1, match="i32")
    refused(L.dropout, x, ctx.empty((4, 8), S.BF16), s, 0.1, match="type")
    refused(L.dropout, x, ctx.empty((8, 4)), s, 0.1, match="shape")
    refused(L.dropout, ctx.empty((4, 8), S.I32), y, s, 0.1, match="f32")
    refused(L.dropout, x, y.view((4, 8), (4, 1)), s, 0.1, match="overlap")
    refused(L.dropout, x.view((32,), (1,)), y, s, 0.1, match="rank 2")
    s.release()
    refused(L.dropout, x, y, s, 0.1, match="missing")


def test_block_norms_refusals(ctx):
    f = lambda *s, d=S.F32: ctx.empty(s, d)  # noqa: E731
    x, y, out, h, w = f(6, 8), f(6, 8), f(6, 8), f(6, 8), f(8)
    N = lambda **k: L.BlockNorms(ctx, **k)  # noqa: E731
    go = lambda n, *a, **k: refused(L.block_norms, n, *a, **k)  # noqa: E731
    L.block_norms(N(after="rms", before="layer", gate=f(3, 8), after_weight=w, before_weight=w, before_bias=w), x, y, out, h, f(6, 4))
    L.block_norms(N(before="rms"), x, None, None, h)
    refused(N, after="batch", match="batch")
    go(N(), x, y, out, h, match="without a norm before")
    go(N(before="rms"), x, y, out, match="h is missing")
    go(N(), x, y, None, match="out is missing")
    go(N(before="rms", residual_scale=0.5), x, None, None, h, match="out is missing")
    for k in (dict(after="rms"), dict(gate=w), dict(p=0.1, seed=f(2, d=S.U32))):
        go(N(**k), x, None, out, match="y is missing")
    go(N(p=0.1), x, y, out, match="seed")
    go(N(p=1.0, seed=f(2, d=S.U32)), x, y, out, match="p is not")
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        go(N(eps=eps), x, y, out, match="eps")
    go(N(residual_scale=float("nan")), x, y, out, match="residual_scale")
    go(N(after_weight=w), x, y, out, match="without its norm")
    go(N(after="rms", after_weight=f(7)), x, y, out, match="after_weight")
    go(N(after="rms", after_weight=f(8, d=S.BF16)), x, y, out, match="f32")
    go(N(after="rms", after_weight=f(16).view((8,), (2,))), x, y, out, match="contiguous")
    go(N(gate=f(4, 8)), x, y, out, match="divide")
    go(N(gate=f(3, 7)), x, y, out, match="column")
    go(N(gate=f(3, 8, d=S.F16)), x, y, out, match="f32")
    go(N(), x, f(6, 8, d=S.BF16), f(6, 8, d=S.BF16), match="type of x")
    go(N(), f(6, 8, d=S.F16), f(6, 8, d=S.BF16), f(6, 8, d=S.F16), match="neither f32")
    go(N(before="rms"), x, y, out, f(6, 8, d=S.BF16), match="type of y")
    go(N(), x, f(5, 8), out, match="shape")
    go(N(), x, y, out.view((6, 8), (4, 1)), match="overlap")
    go(N(), x, y, out, stats=f(6, 3), match="stats")
    go(N(), f(2, 16385), f(2, 16385), f(2, 16385), match="16384")
    go(N(), f(2, 0), f(2, 0), f(2, 0), match="16384")
    n = N(after="rms", after_weight=w)
    w.release()
    go(n, x, y, out, match="released")
    refused(N, after="rms", after_weight=w, match="released")


def test_block_norms_grad_refusals(ctx):
    f = lambda *s, d=S.F32: ctx.empty(s, d)  # noqa: E731
    out, y, st, g, dx, dy, w = f(6, 8), f(6, 8), f(6, 4), f(6, 8), f(6, 8), f(6, 8), f(8)
    n, plain = L.BlockNorms(ctx, after="rms", before="rms", gate=f(2, 8)), L.BlockNorms(ctx)
    L.block_norms_grad(n, out, y, st, g, g, dx, dy, dgate=f(2, 8), dafter_weight=w, dbefore_bias=f(8))
    L.block_norms_grad(plain, out, None, st, g, None, dx)
    go = lambda n, *a, **k: refused(L.block_norms_grad, n, *a, **k)  # noqa: E731
    go(n, out, y, st, None, None, dx, dy, match="both missing")
    go(plain, out, y, st, g, g, dx, match="without a norm before")
    go(n, out, y, f(6, 2), g, g, dx, match="stats")
    go(n, out, y, st, g, g, dx, dy, dgate=f(3, 8), match="gate's shape")
    go(n, out, y, st, g, g, dx, dy, dgate=w, match="gate's shape")
    go(plain, out, y, st, g, None, dx, dgate=w, match="without a gate")
    go(plain, out, y, st, g, None, dx, dafter_weight=w, match="without its norm")
    go(n, out, y, st, g, g, dx, dy, dbefore_weight=f(8, d=S.F16), match="f32")
    go(plain, out, None, st, g, None, dx, dy, match="without y")
    go(n, out, y, st, f(6, 8, d=S.BF16), g, dx, match="type of out")
    go(n, out, y, st, g, f(6, 8, d=S.BF16), dx, match="type of y")
    go(n, out, y, st, g, g, f(6, 8, d=S.BF16), match="dx")
    w.release()
    go(n, out, y, st, g, g, dx, dafter_weight=w, match="released")


def test_launches(ctx):
    f = lambda *s, d=S.F32: ctx.empty(s, d)  # noqa: E731
    n = L.BlockNorms(ctx, after="rms", before="rms", gate=f(8))
    ctx.trace_begin()
    L.block_norms(n, f(6, 8), f(6, 8), f(6, 8), f(6, 8))
    L.block_norms_grad(n, f(6, 8), f(6, 8), f(6, 4), f(6, 8), f(6, 8), f(6, 8), f(6, 8))
    L.block_norms_grad(n, f(6, 8), f(6, 8), f(6, 4), f(6, 8), f(6, 8), f(6, 8), f(6, 8), dgate=f(8))
    L.block_norms(n, f(0, 8), f(0, 8), f(0, 8), f(0, 8))
    assert ctx.trace() == ["block_norms", "block_norms_grad", "block_norms_grad", "block_norms_join"]


def test_counter_matches_published_blocks():
    """Philox4x32-10's known answers: counter and key of zeros, and of ones throughout."""
    words = lambda seed, site, block: [h for h in _block(seed, site, block)]  # noqa: E731
    assert words((0, 0), 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert words((0xffffffff, 0xffffffff), (1 << 64) - 1, (1 << 64) - 1) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def _block(seed, site, block):
    x, key = [block & 0xffffffff, block >> 32, site & 0xffffffff, site >> 32], [int(seed[0]), int(seed[1])]
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(p1 >> 32) ^ x[1] ^ key[0], p1 & 0xffffffff, (p0 >> 32) ^ x[3] ^ key[1], p0 & 0xffffffff]
        key = [(key[0] + 0x9E3779B9) & 0xffffffff, (key[1] + 0xBB67AE85) & 0xffffffff]
    if block < 1 << 20:  # the vectorised form draws the same
        n = 8 * block + 8
        halves = np.array([h for w in x for h in (w & 0xffff, w >> 16)])
        for p in (0.1, 0.5, 0.9):
            assert np.array_equal(B.keep(seed, site, n, p)[-8:], halves >= B.bar_of(p))
    return x


@pytest.mark.parametrize("after,before,gate", [("none", "layer", 0), ("rms", "rms", 1), ("layer", "layer", 2), ("layer", "none", 1), ("rms", "layer", 4)])
def test_the_oracles_gradient_against_differences(after, before, gate):
    rng = np.random.default_rng(3)
    rows, dim, eps = 4, 6, 1e-6
    p = dict(aw=rng.standard_normal(dim), ab=rng.standard_normal(dim), bw=rng.standard_normal(dim), bb=rng.standard_normal(dim))
    p = {k: v if (after if k[0] == "a" else before) != "none" else None for k, v in p.items()}
    p["gate"] = None if not gate else rng.standard_normal((dim,) if gate == 1 else (gate, dim))
    x, y, go, gh = (rng.standard_normal((rows, dim)) for _ in range(4))
    gh = gh if before != "none" else None

    def value(x, y, **p):
        o = B.Norms(after, before, scale=0.5, p=0.4, seed=(1, 2), site=3, **p)
        out = o.out(x, y)[0]
        return (out * go).sum() + ((o.h(out)[0] * gh).sum() if gh is not None else 0.0)

    o = B.Norms(after, before, scale=0.5, p=0.4, seed=(1, 2), site=3, **p)
    out = o.out(x, y)[0]
    stats = np.concatenate([s for rows_, kind in ((y, after), (out, before)) for s in B.statistics(rows_, kind, o.eps)[:2]], 1)
    found = o.grad(out, y, stats, go, gh)
    for name, arg in (("dx", "x"), ("dy", "y"), ("dafter_weight", "aw"), ("dafter_bias", "ab"), ("dbefore_weight", "bw"), ("dbefore_bias", "bb"), ("dgate", "gate")):
        a = dict(x=x, y=y, **p)
        if a[arg] is None:
            continue
        want = np.zeros(a[arg].shape)
        for i in np.ndindex(*a[arg].shape):
            ends = []
            for s in (eps, -eps):
                moved = a[arg].copy()
                moved[i] += s
                ends.append(value(**{**a, arg: moved}))
            want[i] = (ends[0] - ends[1]) / (2 * eps)
        assert np.allclose(found[name][0], want, rtol=1e-6, atol=1e-6), name


# ------------------------------------------------------------------------------------------ log probabilities from hidden states
def test_head_refusals(ctx):
    f = lambda *s, d=S.BF16: ctx.empty(s, d)  # noqa: E731
    h, w, i, lp, st = f(6, 8), f(50, 8), f(6, d=S.I32), f(6, d=S.F32), f(6, 2, d=S.F32)
    L.head_log_probs(h, w, i, lp, lp, st)
    go = lambda *a, **k: refused(L.head_log_probs, *a, **k)  # noqa: E731
    go(h, f(50, 8, d=S.F16), i, lp, match="type of hidden")
    go(h, f(50, 9), i, lp, match="width")
    go(f(6, 0), f(50, 0), i, lp, match="without elements")
    go(h, f(0, 8), i, lp, match="no rows")
    go(f(6, 8, d=S.I8), w, i, lp, match="hidden")
    go(h, w, f(5, d=S.I32), lp, match="ids")
    go(h, w, lp, lp, match="i32")
    go(h, w, i, f(6), match="log_probs")
    go(h, w, i, lp, f(5, d=S.F32), match="entropy")
    go(h, w, i, lp, stats=f(6, 3, d=S.F32), match="stats")
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        go(h, w, i, lp, scale=scale, match="scale")
    go(h.view((6, 8), (1, 6)), w, i, lp, match="contiguous")
    L.head_log_probs_grad(h, w, i, st, lp, lp, lp, f(6, 8), f(50, 8))
    L.head_log_probs_grad(h, w, i, st, None, lp, None, f(6, 8, d=S.F32), None)
    go = lambda *a, **k: refused(L.head_log_probs_grad, *a, **k)  # noqa: E731
    go(h, w, i, st, None, lp, lp, h, match="entropy")
    go(h, w, i, f(6, 4, d=S.F32), lp, lp, lp, h, match="stats")
    go(h, w, i, st, lp, f(5, d=S.F32), None, h, match="g_log_probs")
    go(h, w, i, st, lp, lp, lp, f(6, 8, d=S.F16), match="dhidden")
    go(h, w, i, st, lp, lp, lp, f(6, 7), match="dhidden")
    go(h, w, i, st, lp, lp, lp, None, f(50, 9), match="dweight")
    go(h, w, i, st, lp, lp, lp, None, w.view((50, 8), (0, 1)), match="overlap")


def test_head_launches(ctx):
    f = lambda *s, d=S.BF16: ctx.empty(s, d)  # noqa: E731
    h, w, i, v, st = f(300, 64), f(1000, 64), f(300, d=S.I32), f(300, d=S.F32), f(300, 2, d=S.F32)
    ctx.trace_begin()
    L.head_log_probs(h, w, i, v, v, st)
    assert ctx.trace() == ["head_log_probs", "head_join"]
    ctx.trace_begin()
    L.head_log_probs_grad(h, w, i, st, v, v, v, f(300, 64), f(1000, 64))
    assert ctx.trace() == ["head_rows", "head_probs", "head_dhidden", "head_rows_copy", "head_dweight"], ctx.trace()
