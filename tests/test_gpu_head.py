"""Log probabilities from hidden states and their gradient on a B200 against a plain implementation in 64 bits (head_oracle.py, which derives the
bounds), through the public package."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import head_oracle as H
import language_oracle as O
from test_gpu_language import KIND, Held, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


def operands(d, rng, rows, vocab, dim, kind, pitch=0, lead=0):
    w = rng.standard_normal((vocab, dim)) / np.sqrt(dim)
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    h = 2 * rng.standard_normal((rows, dim)) + 4 * w[ids]
    if rows > 4:
        ids[2], ids[3] = -1, vocab
    h, hv = d.rows(h, kind, dim + pitch, lead)
    w, wv = d.rows(w, kind, dim + pitch, lead)
    return h, hv, w, wv, ids


def check(ctx, d, rng, rows, vocab, dim, kind, scale=1.0, pitch=0, lead=0, out=None, entropy=True, parts=(True, True), stride=1):
    h, hv, w, wv, ids = operands(d, rng, rows, vocab, dim, kind, pitch, lead)
    o = H.Head(hv, wv, ids, scale, kind)
    i, lp, en, st = d.vec(ids, stride), d.empty((rows * stride,)).view((rows,), (stride,)), d.empty((rows,)), d.empty((rows, 2))
    L.head_log_probs(h, w, i, lp, en if entropy else None, st, scale=scale)
    want = np.where(o.scored, np.take_along_axis(o.log_p, np.clip(ids, 0, vocab - 1)[:, None], 1)[:, 0], 0.0)
    close(lp.numpy(), want, np.where(o.scored, np.take_along_axis(o.tol_log_p, np.clip(ids, 0, vocab - 1)[:, None], 1)[:, 0], 0.0), "log probabilities")
    if entropy:
        close(en.numpy(), o.entropy, o.tol_entropy, "entropy")
    gl = -rng.random(rows).astype(np.float32) / rows
    ge = -rng.random(rows).astype(np.float32) * np.float32(0.1 / rows) if entropy else None
    dh, dw = (d.empty((rows, dim + pitch), KIND[out or kind]).view((rows, dim), (dim + pitch, 1)) if parts[0] else None,
              d.empty((vocab, dim + pitch), KIND[out or kind]).view((vocab, dim), (dim + pitch, 1)) if parts[1] else None)
    L.head_log_probs_grad(h, w, i, st, en if entropy else None, d.vec(gl), d.vec(ge) if entropy else None, dh, dw, scale=scale)
    found = o.gradients(gl, ge, out or kind)
    for name, t in (("dhidden", dh), ("dweight", dw)):
        if t is not None:
            close(O.values(t.numpy(), out or kind), *found[name], name)
    assert ctx.status_word() == 0


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 1, 1), (1, 8, 8), (1, 100, 64), (3, 257, 40), (32, 128, 128), (130, 1000, 264), (300, 2049, 64), (257, 515, 1000), (64, 4096, 256),
                                            (5, 50021, 72), (513, 300, 520), (1000, 130, 48), (128, 256, 2048)])
def test_head_sizes(ctx, kind, rows, vocab, dim):
    with Held(ctx) as d:
        check(ctx, d, np.random.default_rng(rows + vocab + dim), rows, vocab, dim, kind)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,dim,pitch,lead", [(7, 300, 33, 0, 0), (40, 130, 64, 8, 0), (40, 130, 64, 3, 1), (40, 130, 65, 7, 8), (2, 33, 3, 1, 2)])
def test_head_layouts(ctx, kind, rows, vocab, dim, pitch, lead):
    with Held(ctx) as d:
        check(ctx, d, np.random.default_rng(dim), rows, vocab, dim, kind, pitch=pitch, lead=lead, scale=0.7, stride=3)


@pytest.mark.parametrize("kind,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("entropy,parts", [(False, (True, True)), (True, (True, False)), (True, (False, True)), (False, (False, False))])
def test_head_parts(ctx, kind, out, entropy, parts):
    with Held(ctx) as d:
        check(ctx, d, np.random.default_rng(1), 140, 700, 72, kind, out=out, entropy=entropy, parts=parts, scale=1.3)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_head_in_pieces_of_the_vocabulary(ctx, kind):
    """More than 256 MB of q: two pieces and more, the last one shorter."""
    rows, vocab = (4100, 40001) if kind == "bf16" else (2100, 40001)
    for out in {kind, "f32"}:
        with Held(ctx) as d:
            check(ctx, d, np.random.default_rng(2), rows, vocab, 40, kind, out=out)


def test_head_rows_in_runs(ctx):
    """More rows than one launch's sums are kept for: the rows on both sides of the cut."""
    rng, rows, vocab, dim = np.random.default_rng(3), 33100, 131072, 8
    with Held(ctx) as d:
        h, hv, w, wv, ids = operands(d, rng, rows, vocab, dim, "bf16")
        lp, en, st = d.empty((rows,)), d.empty((rows,)), d.empty((rows, 2))
        L.head_log_probs(h, w, d.vec(ids), lp, en, st)
        for at in (0, 32640, 32760, 33092):
            some = slice(at, at + 8)
            o = H.Head(hv[some], wv, ids[some], 1.0, "bf16")
            col = np.clip(ids[some], 0, vocab - 1)[:, None]
            close(lp.numpy()[some], np.where(o.scored, np.take_along_axis(o.log_p, col, 1)[:, 0], 0.0), np.take_along_axis(o.tol_log_p, col, 1)[:, 0])
            close(en.numpy()[some], o.entropy, o.tol_entropy)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_head_repeats_its_bits(ctx, kind):
    rng = np.random.default_rng(4)
    with Held(ctx) as d:
        h, _, w, _, ids = operands(d, rng, 300, 3001, 264, kind)
        i, g = d.vec(ids), d.vec(-rng.random(300).astype(np.float32))
        seen = []
        for _ in range(3):
            lp, en, st, dh, dw = d.empty((300,)), d.empty((300,)), d.empty((300, 2)), d.empty((300, 264), KIND[kind]), d.empty((3001, 264), KIND[kind])
            L.head_log_probs(h, w, i, lp, en, st)
            L.head_log_probs_grad(h, w, i, st, en, g, g, dh, dw)
            seen.append([t.numpy() for t in (lp, en, st, dh, dw)])
        for other in seen[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_head_strange_rows(ctx, kind):
    rng = np.random.default_rng(5)
    with Held(ctx) as d:
        w = (rng.standard_normal((300, 24)) / 5).astype(np.float32)
        h = rng.standard_normal((6, 24)).astype(np.float32)
        h[1], h[2, 3], h[4] = 0.0, np.nan, 1000 * h[4]
        h, hv = d.rows(h, kind)
        w, wv = d.rows(w, kind)
        ids = np.array([0, 1, 2, 299, 4, -7], np.int32)
        lp, en, st = d.empty((6,)), d.empty((6,)), d.empty((6, 2))
        L.head_log_probs(h, w, d.vec(ids), lp, en, st)
        o = H.Head(hv, wv, ids, 1.0, kind)
        fine = [0, 1, 3, 4]
        close(lp.numpy()[fine], o.log_p[fine, ids[fine]], o.tol_log_p[fine, ids[fine]])
        close(en.numpy()[fine], o.entropy[fine], o.tol_entropy[fine])
        assert np.isnan(lp.numpy()[2]) and np.isnan(en.numpy()[2]) and lp.numpy()[5] == 0.0
        if kind == "f32":  # (pieces of infinities: their product is not a number)
            return
        masked, mv = d.rows(np.where(np.arange(300)[:, None] % 3 == 0, -np.inf, wv), kind)  # tokens that no positive state reaches
        h, hv = d.rows(np.abs(rng.standard_normal((6, 24))) + 0.1, kind)
        L.head_log_probs(h, masked, d.vec(ids), lp, en, st)
        close(en.numpy(), O.LogProbs(hv.astype(np.float64) @ mv.T.astype(np.float64), ids, 1.0).entropy, H.Head(hv, np.where(np.isinf(mv), -50, mv), ids, 1.0, kind).tol_entropy)
        assert np.isneginf(lp.numpy()[0]) and np.isneginf(lp.numpy()[[3]]) .sum() == (299 % 3 == 0)


def test_head_of_no_rows_and_broadcast_operands(ctx):
    with Held(ctx) as d:
        for kind in ("bf16", "f32"):
            h, w = d.empty((0, 16), KIND[kind]), d.put(np.ones((5, 16), S._NP[KIND[kind]]), KIND[kind])
            dw, e = d.empty((5, 16), KIND[kind]), d.empty((0,))
            L.head_log_probs(h, w, d.empty((0,), S.I32), e, e, d.empty((0, 2)))
            L.head_log_probs_grad(h, w, d.empty((0,), S.I32), d.empty((0, 2)), e, e, e, d.empty((0, 16), KIND[kind]), dw)
            assert (dw.numpy() == 0).all()
            one, ov = d.rows(np.linspace(-1, 1, 16)[None], kind)
            ids, lp, en, st = np.arange(4).astype(np.int32), d.empty((4,)), d.empty((4,)), d.empty((4, 2))
            table, tv = d.rows(np.random.default_rng(0).standard_normal((9, 16)), kind)
            L.head_log_probs(one.view((4, 16), (0, 1)), table, d.vec(ids), lp, en, st)
            o = H.Head(np.repeat(ov, 4, 0), tv, ids, 1.0, kind)
            close(lp.numpy(), o.log_p[np.arange(4), ids], o.tol_log_p[np.arange(4), ids])
            close(en.numpy(), o.entropy, o.tol_entropy)
