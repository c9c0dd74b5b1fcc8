"""Gradients of tokens that a model is nearly sure of, on a B200 against 64 bits: what is left of 1 - p must be that, not what two roundings of a logit differ by."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import language_oracle as O
from test_gpu_language import Held, close

pytestmark = pytest.mark.gpu
U = O.U


@pytest.fixture(scope="module")
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


def confident(ctx, kind, rows, vocab, dim, logit):
    """Hidden states whose tokens' weights have their signs (every term of such a logit is positive, every addition cut the same way); other weights are small.

    With the values' own logits x and sum S, p = exp(x - m) / S of such a token (x = m) is off by the roundings of S, 25 at most (8 of a thread's columns, 3 and 4
    to join them, 5 and 5 in the join of a row's parts), 4 U of the exponential, and 2 U of q's own additions: 31 U, taken as 32 U, of |gl|; the entropy's part has the same
    factor p (the factor ln p + H beside it is small and exact to its own size).  Whatever else the logits are off by changes all p alike in proportion: (dim / 8 + 32) 2U of the sum of
    a logit's terms' sizes at most, times two for the sum's own.  Then q is rounded to 16 bits and multiplied."""
    rng = np.random.default_rng(rows + dim)
    h = rng.choice([-1.0, 1.0], (rows, dim)) * (0.5 + rng.random((rows, dim)))
    w = 0.1 * rng.standard_normal((vocab, dim)) / np.sqrt(dim)
    ids = rng.permutation(vocab)[:rows].astype(np.int32)
    for r, t in enumerate(ids):
        w[t] = h[r] * (logit / (h[r] ** 2).sum())
    gl, ge = -(0.5 + rng.random(rows)).astype(np.float32), -(0.01 * rng.random(rows)).astype(np.float32)
    with Held(ctx) as d:
        hd, hv = d.rows(h, kind)
        wd, wv = d.rows(w, kind)
        hv, wv = hv.astype(np.float64), wv.astype(np.float64)
        lp, en, st, dh, dw, i = d.empty((rows,)), d.empty((rows,)), d.empty((rows, 2)), d.empty((rows, dim)), d.empty((vocab, dim)), d.vec(ids)
        L.head_log_probs(hd, wd, i, lp, en, st)
        L.head_log_probs_grad(hd, wd, i, st, en, d.vec(gl), d.vec(ge), dh, dw)
        x = hv @ wv.T
        m = x.max(1, keepdims=True)
        ln_p = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
        p = np.exp(ln_p)
        entropy = -(p * ln_p).sum(1, keepdims=True)
        g, e, at = gl.astype(np.float64)[:, None], ge.astype(np.float64)[:, None], np.arange(rows)
        q = -g * p - e * p * (ln_p + entropy)
        q[at, ids] = -g[:, 0] * np.expm1(ln_p[at, ids]) - (e * p * (ln_p + entropy))[at, ids]
        off = 2 * (dim / 8 + 32) * 2 * U * (np.abs(hv) @ np.abs(wv).T).max(1, keepdims=True)
        # what the tokens other than the asked one have, in proportion; the asked one by its own roundings and by what the others' change adds up to
        others = p.copy()
        others[at, ids] = 0.0
        rest = others.sum(1, keepdims=True)
        t = others * (np.abs(g) + np.abs(e) * (np.abs(ln_p + entropy) + 1)) * (off + 64 * U)
        t[at, ids] += (np.abs(g) * (32 * U + rest * off) + np.abs(e) * (32 * U + (rest * (np.abs(np.log(rest)) + 2)) * off))[:, 0]
        rel, absolute = O.ROUND[kind]
        absolute = absolute * 4.0 / 2.0 ** 13 if kind == "f16" else absolute
        t = t + (rel * (np.abs(q) + t) + absolute if kind != "f32" else U * np.abs(q))
        product = lambda a, b, k: (k / 8 + 32) * 2 * U * (np.abs(a) @ np.abs(b))  # noqa: E731
        assert 2e-7 < rest.min() and rest.max() < 3e-6
        close(lp.numpy(), ln_p[at, ids], 32 * U + rest[:, 0] * off[:, 0])
        close(dh.numpy(), q @ wv, t @ np.abs(wv) + product(q, wv, vocab), "dhidden")
        close(dw.numpy(), q.T @ hv, t.T @ np.abs(hv) + product(q.T, hv, rows), "dweight")


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,dim,logit", [(300, 20000, 4096, 24.0), (64, 8192, 1000, 23.0)])
def test_gradients_of_confident_tokens(ctx, kind, rows, vocab, dim, logit):
    confident(ctx, kind, rows, vocab, dim, logit)


@pytest.mark.parametrize("kind,rows", [("bf16", 1), ("bf16", 3), ("f16", 4), ("f32", 2), ("f32", 20)])
def test_gradients_of_confident_tokens_in_few_rows(ctx, kind, rows):
    """Their values come from dot products."""
    confident(ctx, kind, rows, 20000, 4096, 24.0)
