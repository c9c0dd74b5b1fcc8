"""Log probabilities from hidden states on a B200: how accurate the sums are, and rows and tokens without a chance, in values and gradients."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import head_accuracy as A
import head_oracle as H
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


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_f32_operands_have_the_accuracy_of_f32(ctx, seed):
    """Within a limit that no five of the six products of pieces reach (tests/test_head_accuracy.py)."""
    h, w, ids = A.random_signs(seed)
    with Held(ctx) as d:
        lp = d.empty((256,))
        L.head_log_probs(d.put(h), d.put(w), d.vec(ids), lp)
        off = lp.numpy() - A.log_p(h.astype(np.float64) @ w.astype(np.float64).T, ids)
        assert np.sqrt((off ** 2).mean()) <= A.rms_limit(h, w, ids)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [4096, 1000])
def test_long_sums_of_one_sign(ctx, kind, dim):
    """Every cut makes them smaller: the bound counts them.  One token of each row has an exact logit above the one that is asked for, whose error then shows whole."""
    rng = np.random.default_rng(dim)
    rows, vocab = 100, 300
    h = rng.choice([-1.0, 1.0], (rows, dim)) * (0.5 + rng.random((rows, dim)))
    h[:, 0] = 1.0
    w = 0.1 * rng.standard_normal((vocab, dim)) / np.sqrt(dim)
    ids = rng.permutation(vocab - 1)[:rows].astype(np.int32)
    for r, t in enumerate(ids):
        w[t] = h[r] * (20.0 / (h[r, 1:] ** 2).sum())
    w[:, 0] = 0.0
    w[vocab - 1] = 0.0
    w[vocab - 1, 0] = 24.0
    with Held(ctx) as d:
        hd, hv = d.rows(h, kind)
        wd, wv = d.rows(w, kind)
        hv, wv = hv.astype(np.float64), wv.astype(np.float64)
        lp, i = d.empty((rows,)), d.vec(ids)
        L.head_log_probs(hd, wd, i, lp)
        want = A.log_p(hv @ wv.T, ids)
        # (4 for the exact token's distance, 25 for the sum of exponentials: a few dozen roundings of numbers near 4 and 1)
        close(lp.numpy(), want, A.positive_sums(hv * wv[ids], kind) + 64 * U)


def both(ctx, d, hv, wv, h, w, ids, kind):
    """Values and the gradient in f32, [lp, entropy, stats, dhidden, dweight], and the arrivals."""
    rng = np.random.default_rng(9)
    rows = len(ids)
    gl, ge = -(0.5 + rng.random(rows)).astype(np.float32), -(0.1 * rng.random(rows)).astype(np.float32)
    lp, en, st, dh, dw, i = d.empty((rows,)), d.empty((rows,)), d.empty((rows, 2)), d.empty(hv.shape), d.empty(wv.shape), d.vec(ids)
    L.head_log_probs(h, w, i, lp, en, st)
    L.head_log_probs_grad(h, w, i, st, en, d.vec(gl), d.vec(ge), dh, dw)
    return [t.numpy() for t in (lp, en, st, dh, dw)], gl, ge


@pytest.mark.parametrize("kind,rows", [("bf16", 3), ("bf16", 40), ("f16", 4), ("f16", 300), ("f32", 6)])
def test_a_row_without_a_chance(ctx, kind, rows):
    """All of its logits are -inf: log p is that, its entropy zero, and it takes no part in the gradient but where its own infinity is a factor."""
    rng = np.random.default_rng(rows)
    vocab, dim, none = 530, 24, 1
    w = rng.standard_normal((vocab, dim)) / 4
    w[:, 0] = 0.25 + rng.random(vocab)
    h = rng.standard_normal((rows, dim))
    h[none, 0] = -np.inf
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    with Held(ctx) as d:
        (hd, hv), (wd, wv) = d.rows(h, kind), d.rows(w, kind)
        (lp, en, st, dh, dw), gl, ge = both(ctx, d, hv, wv, hd, wd, ids, kind)
        fine = np.arange(rows) != none
        o = H.Head(hv[fine], wv, ids[fine], 1.0, kind)
        at = np.arange(rows - 1), ids[fine]
        close(lp[fine], o.log_p[at], o.tol_log_p[at])
        close(en[fine], o.entropy, o.tol_entropy)
        assert np.isneginf(lp[none]) and en[none] == 0.0 and np.isneginf(st[none, 0]) and st[none, 1] == 0.0
        found = o.gradients(gl[fine], ge[fine], "f32")
        close(dh[fine], *found["dhidden"])
        close(dw[:, 1:], found["dweight"][0][:, 1:], found["dweight"][1][:, 1:])
        assert (dh[none] == 0.0).all() and np.isnan(dw[:, 0]).all()  # (zero times infinity)


@pytest.mark.parametrize("kind,rows", [("bf16", 2), ("bf16", 50), ("f16", 4), ("f16", 50)])
def test_tokens_without_a_chance(ctx, kind, rows):
    """Logits of -inf beside others: as if those tokens were not there, and zeros as their gradient."""
    rng = np.random.default_rng(rows)
    vocab, dim = 700, 40
    w = rng.standard_normal((vocab, dim)) / 5
    masked = np.arange(vocab) % 3 == 0
    w[masked, 0] = -np.inf
    h = rng.standard_normal((rows, dim))
    h[:, 0] = 0.1 + rng.random(rows)
    ids = (3 * rng.integers(0, vocab // 3, rows) + 1).astype(np.int32)
    with Held(ctx) as d:
        (hd, hv), (wd, wv) = d.rows(h, kind), d.rows(w, kind)
        (lp, en, _, dh, dw), gl, ge = both(ctx, d, hv, wv, hd, wd, ids, kind)
        place = np.cumsum(~masked) - 1
        o = H.Head(hv, wv[~masked], place[ids], 1.0, kind)
        at = np.arange(rows), place[ids]
        close(lp, o.log_p[at], o.tol_log_p[at])
        close(en, o.entropy, o.tol_entropy)
        found = o.gradients(gl, ge, "f32")
        close(dh[:, 1:], found["dhidden"][0][:, 1:], found["dhidden"][1][:, 1:])
        close(dw[~masked], *found["dweight"])
        assert (dw[masked] == 0.0).all() and np.isnan(dh[:, 0]).all()


@pytest.mark.parametrize("kind,rows", [("bf16", 4), ("bf16", 70), ("f16", 70), ("f32", 8), ("f32", 70)])
def test_rows_that_are_not_numbers(ctx, kind, rows):
    """Their values and gradients are not numbers either; the other rows' are what they are without them (f16's common scale too)."""
    rng = np.random.default_rng(rows)
    vocab, dim = 530, 24
    w, h = rng.standard_normal((vocab, dim)) / 4, rng.standard_normal((rows, dim))
    h[2, 3] = np.nan
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    with Held(ctx) as d:
        (hd, hv), (wd, wv) = d.rows(h, kind), d.rows(w, kind)
        (lp, en, _, dh, dw), gl, ge = both(ctx, d, hv, wv, hd, wd, ids, kind)
        fine = np.arange(rows) != 2
        o = H.Head(hv[fine], wv, ids[fine], 1.0, kind)
        at = np.arange(rows - 1), ids[fine]
        close(lp[fine], o.log_p[at], o.tol_log_p[at])
        close(en[fine], o.entropy, o.tol_entropy)
        found = o.gradients(gl[fine], ge[fine], "f32")
        close(dh[fine], *found["dhidden"])
        assert np.isnan(lp[2]) and np.isnan(en[2]) and np.isnan(dh[2]).all() and np.isnan(dw).all()
