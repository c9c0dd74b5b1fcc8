"""The language-model operators on a B200 against plain implementations in 64 bits (language_oracle.py, which derives the bounds),
through the public package, at sizes, layouts, masks and values where they can go wrong."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import language_oracle as O

pytestmark = pytest.mark.gpu
KIND = {"f32": S.F32, "f16": S.F16, "bf16": S.BF16}


@pytest.fixture(scope="module")
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


class Held:
    def __init__(self, ctx):
        self.ctx, self.items = ctx, []

    def keep(self, t):
        self.items.append(t)
        return t

    def put(self, a, dtype=None):
        return self.keep(self.ctx.tensor(a, dtype))

    def empty(self, shape, dtype=S.F32):
        t = self.keep(self.ctx.empty(shape, dtype))
        if np.prod(shape):  # a value that no result has by accident
            self.ctx._ck(S.lib.sage_memset(self.ctx.h, t.buf, S.ctypes.c_size_t(0), 0x5a, S.ctypes.c_size_t(int(np.prod(shape)) * S._NP[dtype]().itemsize)))
        return t

    def rows(self, x, kind, pitch=None, lead=0):
        """x [r, c] stored as `kind` with `pitch` elements between rows, `lead` elements into its buffer; the f32 values too."""
        raw, val = O.stored(x, kind)
        r, c = raw.shape
        pitch = c if pitch is None else pitch
        flat = np.zeros(lead + max(r - 1, 0) * pitch + c if r else lead + 1, raw.dtype)
        for i in range(r):
            flat[lead + i * pitch: lead + i * pitch + c] = raw[i]
        return self.put(flat, KIND[kind]).view((r, c), (pitch, 1), lead), val

    def vec(self, x, stride=1, dtype=None):
        x = np.asarray(x)
        if stride == 0:
            return self.put(x[:1], dtype).view((x.size,), (0,))
        flat = np.zeros(x.size * stride + 1, x.dtype)
        flat[: x.size * stride: stride] = x
        return self.put(flat, dtype).view((x.size,), (stride,))

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for t in self.items:
            t.release()


def close(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    off = np.abs(got - want)[fine] - np.broadcast_to(bound, want.shape)[fine]
    assert off.size == 0 or off.max() <= 0, (what, off.max(), np.abs(got - want)[fine].max())


# ------------------------------------------------------------------------------------------ embedding
@pytest.mark.parametrize("table,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("tokens,vocab,dim,pitch,lead,stride", [
    (1, 1, 1, None, 0, 1), (1, 997, 768, None, 0, 1), (8, 30522, 768, None, 0, 2), (33, 50, 1000, 1008, 8, 1), (257, 100, 129, 131, 3, 1),
    (5, 7, 8, 24, 0, 3), (64, 33, 4096, None, 0, 1), (3, 9, 12, 16, 4, 1), (4099, 61, 40, None, 0, 1)])
def test_embedding(ctx, table, out, tokens, vocab, dim, pitch, lead, stride):
    rng = np.random.default_rng(tokens + dim)
    with Held(ctx) as h:
        t, val = h.rows(rng.standard_normal((vocab, dim)), table, pitch, lead)
        ids = rng.integers(-2, vocab + 2, tokens).astype(np.int32)
        scale = 1.7
        y = h.empty((tokens, dim), KIND[out])
        L.embedding(t, h.vec(ids, stride), y, scale=scale)
        want = np.where(((ids >= 0) & (ids < vocab))[:, None], val[np.clip(ids, 0, vocab - 1)] * np.float32(scale), np.float32(0))
        raw, _ = O.stored(want, out)
        assert np.array_equal(y.numpy(), raw)  # one product, rounded once


def test_embedding_into_a_view_leaves_the_rest(ctx):
    with Held(ctx) as h:
        t, val = h.rows(np.arange(40.0).reshape(10, 4), "f32")
        buf = h.put(np.full(100, 7.0, np.float32))
        L.embedding(t, h.vec(np.array([3, 9, 0], np.int32)), buf.view((3, 4), (10, 1), 5))
        got = buf.numpy()
        want = np.full(100, 7.0, np.float32)
        for i, v in enumerate((3, 9, 0)):
            want[5 + 10 * i: 9 + 10 * i] = val[v]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("tokens,vocab,dim,how", [
    (1, 1, 1, "any"), (1, 300, 768, "any"), (7, 5, 3, "any"), (64, 64, 130, "all"), (1000, 97, 72, "any"), (4096, 3001, 96, "often"),
    (5000, 11, 40, "one"), (3001, 2, 33, "any"), (20000, 7001, 16, "often"), (33, 10, 1030, "none"), (2049, 1500, 257, "often")])
def test_embedding_grad(ctx, kind, add, tokens, vocab, dim, how):
    rng = np.random.default_rng(tokens * 3 + dim)
    ids = {"any": lambda: rng.integers(-1, vocab + 1, tokens), "all": lambda: rng.permutation(vocab)[:tokens], "one": lambda: np.full(tokens, vocab // 2),
           "none": lambda: np.full(tokens, -1), "often": lambda: np.minimum(np.exp(rng.uniform(0, np.log(vocab + 1), tokens)).astype(np.int64) - 1, vocab - 1)}[how]().astype(np.int32)
    with Held(ctx) as h:
        g, val = h.rows(rng.standard_normal((tokens, dim)), kind)
        start = rng.standard_normal((vocab, dim)).astype(np.float32)
        d = h.put(start)
        L.embedding_grad(g, h.vec(ids), d, scale=0.5, add=add)
        want, bound = O.embedding_grad(val, ids, vocab, 0.5, start if add else None)
        first = d.numpy()
        close(first, want, bound)
        d2 = h.put(start)
        L.embedding_grad(g, h.vec(ids), d2, scale=0.5, add=add)
        assert np.array_equal(first.view(np.uint32), d2.numpy().view(np.uint32))  # the same bits every time


@pytest.mark.parametrize("tokens,vocab,dim,how,stride", [
    (40000, 11, 8, "any", 1), (40000, 5, 8, "one", 1), (17001, 200003, 4, "often", 1), (20000, 700001, 4, "any", 1), (70001, 3001, 20, "often", 2), (16384, 129, 12, "any", 1),
    (16385, 128, 12, "often", 1), (9000, 40, 2052, "often", 1), (300000, 1000, 4, "often", 1)])
def test_embedding_grad_of_long_batches(ctx, tokens, vocab, dim, how, stride):
    """Sorting by one launch and by two, lists that overflow, rows that many blocks share, tables of more rows than a block counts."""
    rng = np.random.default_rng(tokens)
    ids = {"any": lambda: rng.integers(-1, vocab + 1, tokens), "one": lambda: np.full(tokens, vocab // 2),
           "often": lambda: np.minimum(np.exp(rng.uniform(0, np.log(vocab + 1), tokens)).astype(np.int64) - 1, vocab - 1)}[how]().astype(np.int32)
    with Held(ctx) as h:
        g, val = h.rows(rng.standard_normal((tokens, dim)), "f32")
        for add in (False, True):
            start = np.full((vocab, dim), 0.25, np.float32)
            d, i = h.put(start), h.vec(ids, stride)
            L.embedding_grad(g, i, d, add=add)
            want, bound = O.embedding_grad(val, ids, vocab, 1.0, start if add else None)
            got = d.numpy()
            close(got, want, bound)
            d2 = h.put(start)
            L.embedding_grad(g, i, d2, add=add)
            assert np.array_equal(got.view(np.uint32), d2.numpy().view(np.uint32))


@pytest.mark.parametrize("vocab,dim", [(1, 1), (7, 12), (9000, 768)])
def test_no_tokens(ctx, vocab, dim):
    """A gradient of nothing is zeros, or leaves what is there; calls without rows do nothing."""
    with Held(ctx) as h:
        g, ids, d = h.empty((0, dim), S.BF16), h.empty((0,), S.I32), h.put(np.full((vocab, dim), 2.0, np.float32))
        L.embedding_grad(g, ids, d, add=True)
        assert (d.numpy() == 2.0).all()
        L.embedding_grad(g, ids, d)
        assert (d.numpy() == 0.0).all()
        L.embedding(d, ids, h.empty((0, dim)))
        L.embedding(h.empty((0, dim)), h.put(np.array([0, 1], np.int32)), y := h.empty((2, dim)))
        assert (y.numpy() == 0.0).all()
        x, f = h.empty((0, dim), S.F16), h.empty((0,))
        L.token_log_probs(x, ids, f, f, stats=h.empty((0, 2)), top_ids=h.empty((0, 1), S.I32), top_log_probs=h.empty((0, 1)))
        L.token_log_probs_grad(x, ids, h.empty((0, 2)), f, f, f, x)
        L.token_log_probs_and_grad(x, ids, f, f, f, f, x)


@pytest.mark.parametrize("dim,pitch,lead,ld", [(64, 72, 8, 64), (50, 53, 1, 57), (129, 129, 0, 130), (8, 8, 4, 8)])
def test_embedding_grad_of_views(ctx, dim, pitch, lead, ld):
    rng = np.random.default_rng(dim)
    tokens, vocab = 300, 41
    ids = rng.integers(0, vocab, tokens).astype(np.uint32)
    with Held(ctx) as h:
        for kind in ("f32", "bf16"):
            g, val = h.rows(rng.standard_normal((tokens, dim)), kind, pitch, lead)
            buf = h.put(np.full(vocab * ld + 2, 3.0, np.float32))
            L.embedding_grad(g, h.vec(ids, 3), buf.view((vocab, dim), (ld, 1), 1))
            want, bound = O.embedding_grad(val, ids.astype(np.int64), vocab, 1.0)
            raw = buf.numpy()
            got = np.stack([raw[1 + ld * i: 1 + ld * i + dim] for i in range(vocab)])
            close(got, want, bound)
            left = np.ones(raw.size, bool)
            for i in range(vocab):
                left[1 + ld * i: 1 + ld * i + dim] = False
            assert (raw[left] == 3.0).all()


def test_embedding_grad_with_values_that_are_not_finite(ctx):
    """They stay in their rows and columns."""
    rng = np.random.default_rng(0)
    g = rng.standard_normal((100, 24)).astype(np.float32)
    ids = (np.arange(100) % 10).astype(np.int32)
    g[3, 5], g[14, 6], g[27, 7], g[37, 7] = np.nan, np.inf, np.inf, -np.inf
    ids[50] = -1
    g[50] = np.nan
    with Held(ctx) as h:
        d = h.empty((12, 24))
        L.embedding_grad(h.put(g), h.put(ids), d)
        want, bound = O.embedding_grad(g, ids, 12, 1.0)
        got = d.numpy()
        assert np.isnan(got[3, 5]) and np.isposinf(got[4, 6]) and np.isnan(got[7, 7])
        close(got, want, np.where(np.isfinite(bound), bound, 0))


def test_embedding_gradient_is_the_gradient(ctx):
    """Sum of w * embedding(table), by differences in one entry of the table at a time; the sum is linear, so they are exact but for rounding."""
    rng = np.random.default_rng(4)
    vocab, dim, tokens = 6, 5, 9
    table, w = rng.standard_normal((vocab, dim)), rng.standard_normal((tokens, dim)).astype(np.float32)
    ids = rng.integers(0, vocab, tokens).astype(np.int32)
    with Held(ctx) as h:
        d = h.empty((vocab, dim))
        L.embedding_grad(h.put(w), h.put(ids), d, scale=2.0)

        def value(t):
            y = h.empty((tokens, dim))
            L.embedding(h.put(t.astype(np.float32)), h.put(ids), y, scale=2.0)
            return float((y.numpy().astype(np.float64) * w).sum())
        got = d.numpy()
        for i in range(vocab):
            for j in range(dim):
                hi, lo = table.copy(), table.copy()
                hi[i, j] += 0.5
                lo[i, j] -= 0.5
                assert abs(value(hi) - value(lo) - got[i, j]) < 1e-4


# ------------------------------------------------------------------------------------------ log probabilities
def logits_for(rng, rows, vocab, mask):
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    if mask == "inf":
        x[rng.random((rows, vocab)) < 0.5] = -np.inf
        x[:, vocab // 2] = 1.0
    elif mask == "lowest":
        x[rng.random((rows, vocab)) < 0.9] = np.finfo(np.float32).min
        x[:, vocab // 2] = 1.0
    elif mask == "empty":
        x[::2] = -np.inf
    elif mask == "ties":
        x = np.round(x)
    elif mask == "equal":
        x[:] = -4.25
    elif mask == "few":
        x[:] = -np.inf
        x[:, vocab // 3] = 2.0
        x[:, vocab - 1] = -0.0
    elif mask == "far":
        x = x + np.float32(3e4)
    elif mask == "sorted":
        x = -np.sort(-x, axis=1)
    elif mask == "rising":
        x = np.sort(x, axis=1)
    return x


SHAPES = [(1, 1), (1, 30522), (3, 2), (2, 31), (5, 100), (17, 997), (4, 4096), (3, 8191), (2, 16385), (2, 50021), (1, 131072), (300, 130), (1, 262147), (600, 1025)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["", "inf", "lowest", "empty", "ties", "equal", "few", "far", "sorted", "rising"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_token_log_probs(ctx, kind, mask, rows, vocab):
    if kind == "f16" and mask in ("far", "lowest"):
        pytest.skip("not a range of f16")
    rng = np.random.default_rng(rows * 7 + vocab)
    scale = 1.0 if vocab % 2 else 0.75
    with Held(ctx) as h:
        with np.errstate(over="ignore"):
            x, val = h.rows(logits_for(rng, rows, vocab, mask), kind)
        ids = rng.integers(-1, vocab + 1, rows).astype(np.int32)
        ids[0] = vocab // 2
        top = min(vocab, (0, 1, 5, 20, 32)[(rows + vocab) % 5])
        lp, en, st, ti, tl = h.empty((rows,)), h.empty((rows,)), h.empty((rows, 2)), h.empty((rows, top), S.I32), h.empty((rows, top))
        L.token_log_probs(x, h.vec(ids), lp, en, stats=st, top_ids=ti, top_log_probs=tl, scale=scale)
        want = O.LogProbs(val, ids, scale)
        close(lp.numpy(), want.log_probs, want.tol_log_probs, "log probabilities")
        close(en.numpy(), want.entropy, want.tol_entropy, "entropy")
        assert np.array_equal(st.numpy()[:, 0], val.max(1))
        close(st.numpy()[:, 1], want.s, want.s * want.rel_s[:, 0], "sums")
        if top:
            tops, probs, bound = want.top(top)
            assert np.array_equal(ti.numpy(), tops)
            close(tl.numpy(), probs, bound, "alternatives")
        # without what is not asked for, and twice: the same bits
        lp2 = h.empty((rows,))
        L.token_log_probs(x, h.vec(ids), lp2, scale=scale)
        assert np.array_equal(lp.numpy().view(np.uint32), lp2.numpy().view(np.uint32))


@pytest.mark.parametrize("kind,rows,vocab,top", [("f32", 2400, 5003, 5), ("bf16", 2500, 20000, 32), ("bf16", 2400, 40001, 3), ("f32", 100, 40003, 20), ("f16", 90, 70000, 0), ("f32", 700, 9001, 7),
                                                 ("bf16", 74, 20001, 9), ("bf16", 20, 262144, 32)])
@pytest.mark.parametrize("mask", ["", "inf", "ties", "few", "empty", "equal"])
def test_token_log_probs_of_many_rows(ctx, kind, rows, vocab, top, mask):
    """Blocks of every size, a row to each or several to a row; on top of the values of a few rows, all rows' tops and sums."""
    rng = np.random.default_rng(rows)
    base = logits_for(rng, 8, vocab, mask)
    at = rng.integers(0, 8, rows)
    with Held(ctx) as h:
        raw, val = O.stored(base, kind)
        x = h.put(raw[at], KIND[kind])
        ids = rng.integers(-1, vocab + 1, rows).astype(np.int32)
        lp, en, ti, tl = h.empty((rows,)), h.empty((rows,)), h.empty((rows, top), S.I32), h.empty((rows, top))
        L.token_log_probs(x, h.vec(ids), lp, en, top_ids=ti, top_log_probs=tl)
        eight = O.LogProbs(val, np.zeros(8, np.int64), 1.0)
        ok = (ids >= 0) & (ids < vocab)
        close(lp.numpy(), np.where(ok, eight.log_p[at, np.where(ok, ids, 0)], 0.0), eight.tol_log_p[at, np.where(ok, ids, 0)])
        close(en.numpy(), eight.entropy[at], eight.tol_entropy[at])
        if top:
            tops, probs, bound = eight.top(top)
            assert np.array_equal(ti.numpy(), tops[at])
            close(tl.numpy(), probs[at], bound[at])


@pytest.mark.parametrize("kind,rows,vocab", [("f32", 300, 5000), ("bf16", 1200, 9001), ("f16", 40, 50021), ("bf16", 300, 131072), ("f32", 9, 131075), ("bf16", 9, 262137), ("f32", 9, 140000), ("bf16", 700, 16400)])
def test_gradient_of_many_rows(ctx, kind, rows, vocab):
    """Rows in the registers of clusters of every size, and rows that no cluster holds."""
    rng = np.random.default_rng(rows + vocab)
    base = logits_for(rng, 4, vocab, "inf")
    at = rng.integers(0, 4, rows)
    with Held(ctx) as h:
        raw, val = O.stored(base, kind)
        x = h.put(raw[at], KIND[kind])
        own = rng.integers(0, vocab, 4).astype(np.int32)
        ids, gl, ge = own[at], np.array([0.5, -1.0, 0.25, 2.0], np.float32), np.array([0.1, 0.0, -0.3, 1.0], np.float32)
        lp, en, dx = h.empty((rows,)), h.empty((rows,)), h.empty((rows, vocab), KIND[kind])
        L.token_log_probs_and_grad(x, h.put(ids), h.put(gl[at]), h.put(ge[at]), lp, en, dx)
        want = O.LogProbs(val, own, 1.0)
        g, bound = want.grad(gl, ge, kind)
        close(lp.numpy(), want.log_probs[at], want.tol_log_probs[at])
        close(en.numpy(), want.entropy[at], want.tol_entropy[at])
        got = O.values(dx.numpy(), kind)
        for i in range(rows):  # rows of an odd length start at different places of a vector, so equal rows may differ in their last bits
            close(got[i], g[at[i]], bound[at[i]])


@pytest.mark.parametrize("top", range(1, 33))
def test_every_number_of_alternatives(ctx, top):
    rng = np.random.default_rng(top)
    for rows, vocab in ((3, 32 + top), (2, 20011)):
        with Held(ctx) as h:
            x, val = h.rows(np.round(rng.standard_normal((rows, vocab)) * 4), "bf16")
            ids = np.zeros(rows, np.int32)
            lp, ti, tl = h.empty((rows,)), h.empty((rows, top), S.U32), h.empty((rows, top))
            L.token_log_probs(x, h.put(ids), lp, top_ids=ti, top_log_probs=tl)
            tops, probs, bound = O.LogProbs(val, ids, 1.0).top(top)
            assert np.array_equal(ti.numpy(), tops)
            close(tl.numpy(), probs, bound)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bad", ["nan", "inf", "both"])
def test_log_probs_of_rows_that_are_not_finite(ctx, kind, bad):
    """Such a row's values are NaN, its alternatives take NaN for -inf, and the other rows are as ever."""
    rng = np.random.default_rng(1)
    for vocab in (40, 5000, 70001):
        x = rng.standard_normal((4, vocab)).astype(np.float32)
        if bad in ("nan", "both"):
            x[1, 7] = np.nan
        if bad in ("inf", "both"):
            x[1, 9] = np.inf
        x[3, :] = np.nan if bad == "nan" else x[3, :]
        with Held(ctx) as h:
            xs, val = h.rows(x, kind)
            ids = np.array([3, 3, 3, 3], np.int32)
            lp, en, ti, tl = h.empty((4,)), h.empty((4,)), h.empty((4, 6), S.I32), h.empty((4, 6))
            L.token_log_probs(xs, h.put(ids), lp, en, top_ids=ti, top_log_probs=tl)
            broken = [1, 3] if bad == "nan" else [1]
            whole = [i for i in range(4) if i not in broken]
            want = O.LogProbs(val[whole], ids[whole], 1.0)
            close(lp.numpy()[whole], want.log_probs, want.tol_log_probs)
            close(en.numpy()[whole], want.entropy, want.tol_entropy)
            assert np.isnan(lp.numpy()[broken]).all() and np.isnan(en.numpy()[broken]).all()
            order = np.argsort(-np.where(np.isnan(val), -np.inf, val), axis=1, kind="stable")[:, :6]
            assert np.array_equal(ti.numpy(), order)
            gl = h.put(np.ones(4, np.float32))
            dx = h.empty((4, vocab), KIND[kind])
            L.token_log_probs_and_grad(xs, h.put(ids), gl, None, lp, en, dx)
            got = O.values(dx.numpy(), kind)
            assert np.isnan(got[broken]).all() and np.isfinite(got[whole]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["", "inf", "lowest", "empty", "equal", "far"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_log_probs_gradient(ctx, kind, mask, rows, vocab):
    if kind == "f16" and mask in ("far", "lowest"):
        pytest.skip("not a range of f16")
    rng = np.random.default_rng(rows * 5 + vocab)
    scale = 1.0 if vocab % 2 else 1.5
    with Held(ctx) as h:
        x, val = h.rows(logits_for(rng, rows, vocab, mask), kind)
        ids = rng.integers(-1, vocab, rows).astype(np.int32)
        gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
        want = O.LogProbs(val, ids, scale)
        lp, en, st = h.empty((rows,)), h.empty((rows,)), h.empty((rows, 2))
        i, gls, ges = h.vec(ids), h.vec(gl), h.vec(ge)
        L.token_log_probs(x, i, lp, en, stats=st, scale=scale)
        for a, b in ((gls, ges), (gls, None), (None, ges)):
            g, bound = want.grad(gl if a else 0.0, ge if b else 0.0, kind)
            dx = h.empty((rows, vocab), KIND[kind])
            L.token_log_probs_grad(x, i, st, en, a, b, dx, scale=scale)
            close(O.values(dx.numpy(), kind), g, bound, "from stats")
            lp2, en2, dx2 = h.empty((rows,)), h.empty((rows,)), h.empty((rows, vocab), KIND[kind])
            L.token_log_probs_and_grad(x, i, a, b, lp2, en2, dx2, scale=scale)
            close(O.values(dx2.numpy(), kind), g, bound, "at once")
            close(lp2.numpy(), want.log_probs, want.tol_log_probs)
            close(en2.numpy(), want.entropy, want.tol_entropy)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,pitch,lead,pitch2,lead2", [(7, 1001, 1003, 1, 1001, 0), (5, 4096, 4104, 8, 4096, 0), (3, 30522, 30528, 2, 30522, 6), (4, 513, 513, 0, 515, 3),
                                                              (3, 70000, 70008, 8, 70001, 1)])
def test_log_probs_of_views(ctx, kind, rows, vocab, pitch, lead, pitch2, lead2):
    """Any distance between rows, any start; vectors with strides and broadcast gradients; nothing is written beside the results."""
    rng = np.random.default_rng(vocab)
    with Held(ctx) as h:
        x, val = h.rows(rng.standard_normal((rows, vocab)) * 2, kind, pitch, lead)
        ids = rng.integers(0, vocab, rows).astype(np.uint32)
        want = O.LogProbs(val, ids.astype(np.int64), 1.0)
        g, bound = want.grad(np.full(rows, -0.25), np.full(rows, 0.125), kind)
        lp_buf, st, en = h.put(np.full(3 * rows + 4, 9.0, np.float32)), h.put(np.full((rows, 5), 9.0, np.float32)), h.empty((rows,))
        lp = lp_buf.view((rows,), (3,), 1)
        top = h.put(np.full((rows, 8), 77, np.int32))
        topl = h.put(np.full((rows, 6), 77.0, np.float32))
        gl, ge, i = h.vec(np.full(rows, -0.25, np.float32), 0), h.vec(np.full(rows, 0.125, np.float32), 0), h.vec(ids, 2)
        L.token_log_probs(x, i, lp, en, stats=st.view((rows, 2), (5, 1), 2), top_ids=top.view((rows, 4), (8, 1), 3), top_log_probs=topl.view((rows, 4), (6, 1), 0))
        raw = lp_buf.numpy()
        close(raw[1: 3 * rows: 3], want.log_probs, want.tol_log_probs)
        assert (np.delete(raw, np.arange(1, 3 * rows, 3)) == 9.0).all() and (st.numpy()[:, [0, 1, 4]] == 9.0).all()
        tops, probs, tol = want.top(4)
        assert np.array_equal(top.numpy()[:, 3:7], tops) and (np.delete(top.numpy(), range(3, 7), 1) == 77).all()
        close(topl.numpy()[:, :4], probs, tol)
        for at_once in (False, True):
            size = lead2 + rows * pitch2 + 5
            buf = h.put(np.full(size, 3, np.float32) if kind == "f32" else np.full(size, 0x4040, np.uint16), KIND[kind])
            dx = buf.view((rows, vocab), (pitch2, 1), lead2)
            if at_once:
                L.token_log_probs_and_grad(x, i, gl, ge, lp, en, dx)
            else:
                L.token_log_probs_grad(x, i, st.view((rows, 2), (5, 1), 2), en, gl, ge, dx)
            raw = O.values(buf.numpy(), kind)
            inside = np.zeros(size, bool)
            for r in range(rows):
                inside[lead2 + r * pitch2: lead2 + r * pitch2 + vocab] = True
            close(raw[inside].reshape(rows, vocab), g, bound)
            assert (raw[~inside] == 3.0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(5, 1000), (3, 30522), (2, 131073), (2, 300001)])
def test_gradient_over_the_logits(ctx, kind, rows, vocab):
    """dlogits may be the logits' own memory, in both forms."""
    rng = np.random.default_rng(vocab)
    x0 = rng.standard_normal((rows, vocab)) * 2
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    gl = np.full(rows, -0.5, np.float32)
    for at_once in (False, True):
        with Held(ctx) as h:
            x, val = h.rows(x0, kind)
            want = O.LogProbs(val, ids, 1.0)
            g, bound = want.grad(gl, 0.0, kind)
            lp, en, st, i, gls = h.empty((rows,)), h.empty((rows,)), h.empty((rows, 2)), h.put(ids), h.put(gl)
            if at_once:
                L.token_log_probs_and_grad(x, i, gls, None, lp, en, x)
            else:
                L.token_log_probs(x, i, lp, en, stats=st)
                L.token_log_probs_grad(x, i, st, None, gls, None, x)
            close(O.values(x.numpy(), kind), g, bound)
            close(lp.numpy(), want.log_probs, want.tol_log_probs)


def test_log_probs_gradient_is_the_gradient(ctx):
    """By central differences of the values themselves: step 2^-6, third derivatives at most 8 in size here, values good to 2e-6."""
    rng = np.random.default_rng(8)
    rows, vocab, scale, step = 3, 9, 1.25, 2.0 ** -6
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    ids = np.array([2, 8, 0], np.int32)
    gl, ge = np.array([0.5, -1.0, 0.25], np.float32), np.array([1.0, 0.5, -0.75], np.float32)
    with Held(ctx) as h:
        def value(x):
            lp, en = h.empty((rows,)), h.empty((rows,))
            L.token_log_probs(h.put(x), h.put(ids), lp, en, scale=scale)
            return gl.astype(np.float64) * lp.numpy() + ge.astype(np.float64) * en.numpy()
        dx, lp, en = h.empty((rows, vocab)), h.empty((rows,)), h.empty((rows,))
        L.token_log_probs_and_grad(h.put(x), h.put(ids), h.put(gl), h.put(ge), lp, en, dx, scale=scale)
        got = dx.numpy()
        for j in range(vocab):
            hi, lo = x.copy(), x.copy()
            hi[:, j] += np.float32(step)
            lo[:, j] -= np.float32(step)
            num = (value(hi) - value(lo)) / (hi[:, j].astype(np.float64) - lo[:, j])
            assert np.abs(num - got[:, j]).max() < 8 * 3 * step ** 2 / 6 + 4 * 2e-6 / step


def test_offsets_beyond_32_bits(ctx):
    """Rows 2^30 elements apart: the last ones start behind 2^31 elements and 2^32 bytes."""
    pitch, rows, vocab, dim = 1 << 30, 4, 1000, 64
    rng = np.random.default_rng(3)
    with Held(ctx) as h:
        big = h.keep(ctx.empty((rows * pitch - pitch + 4096,), S.BF16))
        raw, val = O.stored(rng.standard_normal((rows, vocab)), "bf16")
        for r in range(rows):
            ctx.upload(big.buf, raw[r], offset=2 * r * pitch)
        x = big.view((rows, vocab), (pitch, 1))
        ids = np.array([1, 999, 0, 500], np.int32)
        want = O.LogProbs(val, ids, 1.0)
        lp, en, i, gl = h.empty((rows,)), h.empty((rows,)), h.put(ids), h.put(np.ones(rows, np.float32))
        L.token_log_probs(x, i, lp, en)
        close(lp.numpy(), want.log_probs, want.tol_log_probs)
        L.token_log_probs_and_grad(x, i, gl, None, lp, en, x)
        g, bound = want.grad(np.ones(rows), 0.0, "bf16")
        got = np.stack([ctx.download(big.buf, (vocab,), np.uint16, offset=2 * r * pitch) for r in range(rows)])
        close(O.values(got, "bf16"), g, bound)
        # the same memory as a table, and as its gradient
        for r in range(rows):
            ctx.upload(big.buf, raw[r], offset=2 * r * pitch)
        y = h.empty((rows, dim), S.BF16)
        t = np.array([3, 0, 2, 1], np.int32)
        L.embedding(big.view((rows, dim), (pitch, 1)), h.put(t), y)
        assert np.array_equal(y.numpy(), raw[t][:, :dim])
        d = h.empty((5, dim))
        L.embedding_grad(big.view((rows, dim), (pitch, 1)), h.put(t), d)
        assert np.array_equal(d.numpy()[t], val[:, :dim]) and (d.numpy()[4] == 0).all()


# ------------------------------------------------------------------------------------------ AdamW
RULE = dict(step=3, lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, grad_scale=0.25)
SIZES = [(1,), (255,), (256,), (257,), (3, 100), (0,), (1000, 17), (4096,), (7,), (70001,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("copy", [None, "bf16", "f16"])
@pytest.mark.parametrize("lead", [0, 1])
def test_adamw(ctx, bits, grad, copy, lead):
    rng = np.random.default_rng(bits + lead)
    with Held(ctx) as h:
        slots, all_ = [], []
        for shape in SIZES:
            n = int(np.prod(shape))

            def put(a, dtype=None):  # `lead` elements into its buffer
                flat = np.zeros(n + lead + 1, a.dtype)
                flat[lead: lead + n] = a.reshape(-1)
                strides = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
                return h.put(flat, dtype).view(shape, strides, lead)
            p = rng.standard_normal(n).astype(np.float32)
            raw, g = O.stored(rng.standard_normal(n) * 10.0 ** rng.uniform(-4, 0, n), grad)
            m = (rng.standard_normal(n) * 10.0 ** rng.uniform(-4, 0, n)).astype(np.float32)
            root = np.abs(rng.standard_normal(n) * 10.0 ** rng.uniform(-3, 0, n)).astype(np.float32)
            e = dict(n=n, p=p, g=g)
            if bits == 8:
                (mc, ms), (vc, vs) = O.adamw_encode(m, 127), O.adamw_encode(root, 255)
                e["m"], q = O.adamw_decode(mc, ms), O.adamw_decode(vc, vs)
                e["v"] = q * q
                states = [put(mc, S.I8), put(vc, S.U8), h.put(ms if n else np.zeros(1, np.float32)).view((len(ms),), (1,)), h.put(vs if n else np.zeros(1, np.float32)).view((len(vs),), (1,))]
            else:
                e["m"], e["v"] = m, root * root
                states = [put(m), put(root * root), None, None]
            c = put(np.zeros(n, np.uint16) if copy == "bf16" else np.zeros(n, np.float16), KIND[copy]) if copy else None
            e["t"] = [put(p), put(raw, KIND[grad])] + states + [c]
            slots.append(L.adamw_tensor(*e["t"]))
            all_.append(e)
        tensors = L.AdamWTensors(ctx, slots)
        L.adamw_step(tensors, **RULE)
        for e in all_:
            if not e["n"]:
                continue
            want, m64, v64, bound = O.adamw_64(e["p"], e["m"], e["v"], e["g"], RULE)
            got = e["t"][0].numpy().reshape(-1)
            close(got, want, bound, "parameters")
            m, v = O.adamw_f32(e["m"], e["v"], e["g"], RULE["beta1"], RULE["beta2"], RULE["grad_scale"])
            if bits == 8:
                (mc, ms), (vc, vs) = O.adamw_encode(m, 127), O.adamw_encode(np.sqrt(v), 255)
                assert np.array_equal(e["t"][2].numpy().reshape(-1), mc) and np.array_equal(e["t"][3].numpy().reshape(-1), vc)
                assert np.array_equal(e["t"][4].numpy(), ms) and np.array_equal(e["t"][5].numpy(), vs)
                # stored values: half a step of the square law, code +- 1/2 of top at the most
                close(O.adamw_decode(mc, ms), m64, (np.sqrt(np.abs(m64) * np.repeat(ms, 256)[: e["n"]]) + np.repeat(ms, 256)[: e["n"]]) * 1.001 + 1e-30)
            else:
                assert np.array_equal(e["t"][2].numpy().reshape(-1), m) and np.array_equal(e["t"][3].numpy().reshape(-1), v)
                close(m, m64, 4 * O.U * (np.abs(m64) + np.abs(e["m"]) + np.abs(e["g"])))
                close(v, v64, 6 * O.U * np.abs(v64))
            if copy:
                raw, _ = O.stored(got, copy)
                assert np.array_equal(e["t"][6].numpy().reshape(-1), raw)


def test_adamw_of_many_tensors(ctx):
    """More tensors than one launch's list holds, empty ones among them."""
    rng = np.random.default_rng(0)
    sizes = [int(s) for s in rng.integers(0, 700, 1003)]
    with Held(ctx) as h:
        p, g = [rng.standard_normal(s).astype(np.float32) for s in sizes], [rng.standard_normal(s).astype(np.float32) for s in sizes]
        flat = {k: h.put(np.concatenate([np.pad(a, (0, 1024 - a.size)) for a in v])) for k, v in (("p", p), ("g", g))}
        m, v = h.put(np.zeros(1024 * len(sizes), np.float32)), h.put(np.zeros(1024 * len(sizes), np.float32))
        part = lambda t, i: t.view((sizes[i],), (1,), 1024 * i)  # noqa: E731
        L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(part(flat["p"], i), part(flat["g"], i), part(m, i), part(v, i)) for i in range(len(sizes))]), **RULE)
        got = flat["p"].numpy().reshape(-1, 1024)
        for i, s in enumerate(sizes):
            want, _, _, bound = O.adamw_64(p[i], np.zeros(s), np.zeros(s), g[i], RULE)
            close(got[i, :s], want, bound)
            assert (got[i, s:] == 0).all()


def test_adamw_first_steps_from_zeroed_states(ctx):
    """Zeroed codes and scales are zero states: the first step moves every parameter by lr against its gradient's sign; ten steps of
    8-bit states stay near the 64-bit ones."""
    rng = np.random.default_rng(6)
    n = 5000
    p0, o = rng.standard_normal(n).astype(np.float32), dict(RULE, weight_decay=0.0, grad_scale=1.0, lr=1e-3)
    with Held(ctx) as h:
        p, m, v = h.put(p0), h.put(np.zeros(n, np.int8), S.I8), h.put(np.zeros(n, np.uint8), S.U8)
        ms, vs = h.put(np.zeros(20, np.float32)), h.put(np.zeros(20, np.float32))
        want, wm, wv = p0.astype(np.float64), np.zeros(n), np.zeros(n)
        for step in range(1, 11):
            g = (rng.standard_normal(n) + 2.0).astype(np.float32)
            o["step"] = step
            L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(p, h.put(g), m, v, ms, vs)]), **o)
            want, wm, wv, _ = O.adamw_64(want, wm, wv, g, o)
            if step == 1:
                assert np.abs(p.numpy() - (p0 - 1e-3 * np.sign(g))).max() < 1e-5
        assert np.abs(p.numpy() - want).max() < 0.05 * 10 * 1e-3  # codes of both moments: a few per cent of the way gone


def test_adamw_states_that_are_not_finite(ctx):
    """A block with an infinite or undefined moment has scales that are NaN; other blocks and the parameters of the block's other
    elements are as ever.  Blocks that vanish are zero."""
    n = 1024
    rng = np.random.default_rng(2)
    g = rng.standard_normal(n).astype(np.float32)
    g[5], g[300] = np.nan, np.inf
    g[512:768] = 0.0
    g[768:] *= np.float32(1e-25)  # v underflows, m does not
    p0 = rng.standard_normal(n).astype(np.float32)
    with Held(ctx) as h:
        p, m, v = h.put(p0), h.put(np.zeros(n, np.int8), S.I8), h.put(np.zeros(n, np.uint8), S.U8)
        ms, vs, mo, vo = h.put(np.zeros(4, np.float32)), h.put(np.zeros(4, np.float32)), h.empty((n,)), h.empty((n,))
        L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(p, h.put(g), m, v, ms, vs)]), **RULE)
        L.adamw_states(m, ms, v, vs, mo, vo)
        assert np.isnan(ms.numpy()[:2]).all() and np.isnan(vs.numpy()[:2]).all() and (ms.numpy()[2], vs.numpy()[2]) == (0, 0)
        assert np.isnan(mo.numpy()[:512]).all() and np.isnan(vo.numpy()[:512]).all() and (mo.numpy()[512:768] == 0).all() and (vo.numpy()[512:768] == 0).all()
        got = p.numpy()
        fine = np.setdiff1d(np.arange(n), [5, 300])
        want, _, _, bound = O.adamw_64(p0, np.zeros(n), np.zeros(n), g, RULE)
        close(got[fine][:700], want[fine][:700], bound[fine][:700])
        assert np.isnan(got[5]) and np.isnan(got[300]) and np.isfinite(got[fine]).all()
        mm, _ = O.adamw_f32(np.zeros(n, np.float32), np.zeros(n, np.float32), g, RULE["beta1"], RULE["beta2"], RULE["grad_scale"])
        assert np.array_equal(m.numpy()[768:], O.adamw_encode(mm, 127)[0][768:])


def test_second_moments_do_not_become_zero(ctx):
    """One large second moment beside small ones: their codes would round to nothing, and their steps be divided by eps."""
    n = 256
    g = np.full(n, 1e-7, np.float32)
    g[0] = 1.0
    with Held(ctx) as h:
        p, m, v, ms, vs = h.put(np.zeros(n, np.float32)), h.put(np.zeros(n, np.int8), S.I8), h.put(np.zeros(n, np.uint8), S.U8), h.put(np.zeros(1, np.float32)), h.put(np.zeros(1, np.float32))
        L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(p, h.put(g), m, v, ms, vs)]), **RULE)
        assert (v.numpy()[1:] == 1).all() and v.numpy()[0] == 255


# ------------------------------------------------------------------------------------------ streams and foreign memory
def test_on_another_runtimes_stream_and_memory(ctx):
    """Operands that torch fills on its own stream just before, results that it reads right after, without a synchronisation."""
    import torch
    other = S.Context(0)
    side = torch.cuda.Stream()
    other.use_stream(side.cuda_stream)
    with torch.cuda.stream(side):
        for i in range(5):
            x = torch.randn(64, 20000, device="cuda") * 2
            ids = torch.randint(0, 20000, (64,), device="cuda", dtype=torch.int32)
            lp, dx, gl = torch.empty(64, device="cuda"), torch.empty_like(x), torch.ones(64, device="cuda")
            h = [other.borrow(t) for t in (x, ids, gl, lp, dx)]
            L.token_log_probs_and_grad(h[0], h[1], h[2], None, h[3], None, h[4])
            want = torch.log_softmax(x.double(), 1).gather(1, ids.long()[:, None])[:, 0]
            assert (lp.double() - want).abs().max().item() < 1e-4
            assert dx.double().sum(1).abs().max().item() < 1e-4
            for t in h:
                t.release()
    # what the context does on its own stream afterwards is behind that
    other.use_own_stream()
    y = other.empty((64,))
    other._ck(S.lib.sage_map(other.h, b"(x0 * 2.0f)", other.borrow(lp).ref(), 1, y.ref()))
    assert np.array_equal(y.numpy(), 2 * lp.cpu().numpy())
    other.close()


def test_host_memory_is_refused(ctx):
    a = np.zeros(64, np.float32)
    with pytest.raises(S.SageError) as e:
        ctx.wrap(a.ctypes.data, (64,))
    assert e.value.code == 1
