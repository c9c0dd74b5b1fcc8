"""The lazy-graph forms of the language-model operators on a B200: values, gradients through the graph, the AdamW optimizer, and the
example that runs them together."""
import importlib.util
import os

import numpy as np
import pytest

import sage_b200 as S

import language_oracle as O

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


def close(got, want, bound):
    off = np.abs(np.asarray(got, np.float64) - want) - bound
    assert off.shape == np.asarray(want).shape and (off.size == 0 or off.max() <= 0), off.max()


@pytest.mark.parametrize("extents", [(7,), (3, 5), (2, 1, 4)])
@pytest.mark.parametrize("turned", [False, True])
def test_embedding_and_its_gradient(ctx, extents, turned):
    rng = np.random.default_rng(len(extents))
    vocab, dim, scale = 11, 20, 1.5
    table = rng.standard_normal((dim, vocab) if turned else (vocab, dim)).astype(np.float32)
    ids = rng.integers(-1, vocab + 1, extents).astype(np.int32)
    w = rng.standard_normal(extents + (dim,)).astype(np.float32)
    tv, iv, wv = ctx.var(table), ctx.var(ids), ctx.var(w)
    rows = table.T if turned else table
    y = S.embedding(tv.tr() if turned else tv, iv, scale)
    assert y.extents == extents + (dim,)
    g = tv.grad((y * wv).sum(None))
    want = np.where(((ids >= 0) & (ids < vocab))[..., None], rows[np.clip(ids, 0, vocab - 1)] * np.float32(scale), np.float32(0))
    assert np.array_equal(y.eval(ctx), want)
    grad, bound = O.embedding_grad(w.reshape(-1, dim), ids.reshape(-1), vocab, scale)
    got = g.eval(ctx)
    close(got.T if turned else got, grad, bound + 4 * O.U * np.abs(grad))


def test_embedding_takes_slices_and_broadcast_gradients(ctx):
    """Ids that are a slice, a gradient that is one broadcast number, a table used twice."""
    rng = np.random.default_rng(2)
    vocab, dim = 9, 12
    table, ids = rng.standard_normal((vocab, dim)).astype(np.float32), rng.integers(0, vocab, (4, 6)).astype(np.uint32)
    tv, iv = ctx.var(table), ctx.var(ids)
    y = S.embedding(tv, iv.slice(1, 1, 4)).sum(None) + S.embedding(tv, iv.index(1, 0), 3.0).sum(None)
    part, first = ids[:, 1:4].reshape(-1), ids[:, 0]
    want = np.zeros((vocab, dim))
    np.add.at(want, part, 1.0)
    np.add.at(want, first, 3.0)
    close(tv.grad(y).eval(ctx), want, 1e-5)
    total = table[part].astype(np.float64).sum() + 3.0 * table[first].astype(np.float64).sum()
    close(y.eval(ctx).reshape(-1), np.array([total]), 1e-3)


@pytest.mark.parametrize("rows,vocab", [(1, 5), (37, 1000), (8, 30522)])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_token_log_probs_and_their_gradient(ctx, rows, vocab, scale):
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[:, 1] = -np.inf
    ids = rng.integers(-1, vocab, rows).astype(np.int32)
    gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    xv = ctx.var(x)
    lp, h = S.token_log_probs(xv, ctx.var(ids.reshape(rows, 1)), scale)
    loss = (lp * ctx.var(gl)).sum(None) + (h * ctx.var(ge)).sum(None)
    dx = xv.grad(loss)
    ctx.eval(lp, h, dx)
    want = O.LogProbs(x, ids, scale)
    with np.errstate(invalid="ignore"):
        fine = np.isfinite(want.log_probs)
        close(ctx.read(lp)[fine], want.log_probs[fine], want.tol_log_probs[fine])
    close(ctx.read(h), want.entropy, want.tol_entropy)
    g, bound = want.grad(gl, ge, "f32")
    close(ctx.read(dx), g, bound)
    top = S.top_tokens(xv, min(vocab, 4)).eval(ctx)
    assert top.dtype == np.uint32 and np.array_equal(top, want.top(min(vocab, 4))[0])


def test_only_one_of_the_values_is_used(ctx):
    """The other's gradient is zero, and logits that are a transposed product."""
    rng = np.random.default_rng(5)
    a, b = rng.standard_normal((6, 16)).astype(np.float32), rng.standard_normal((50, 16)).astype(np.float32)
    ids = rng.integers(0, 50, 6).astype(np.uint32)
    av, bv = ctx.var(a), ctx.var(b)
    _, h = S.token_log_probs(av.matmul(bv.tr()), ctx.var(ids))
    ga = av.grad(h.sum(None)).eval(ctx)
    want = O.LogProbs(a.astype(np.float64) @ b.T.astype(np.float64), ids.astype(np.int64), 1.0)
    g, _ = want.grad(0.0, 1.0, "f32")
    assert np.abs(ga - g @ b).max() < 1e-4


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_over_parameters(ctx, bits):
    rng = np.random.default_rng(bits)
    shapes = [(300, 40), (40,), (1,), (64, 64)]
    values = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    params = [ctx.var(v) for v in values]
    o = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
    opt = S.AdamW(state_bits=bits, **o)
    opt.init(ctx)
    m, v = [np.zeros(s) for s in shapes], [np.zeros(s) for s in shapes]
    want = [x.astype(np.float64) for x in values]
    for step in range(1, 5):
        grads = [(rng.standard_normal(s) + 1.0).astype(np.float32) for s in shapes]
        opt.update(dict(zip(params, [ctx.var(g) for g in grads])), ctx)
        for i, g in enumerate(grads):
            want[i], m[i], v[i], _ = O.adamw_64(want[i], m[i], v[i], g, dict(o, step=step, grad_scale=1.0))
            # 32 bits: a dozen roundings a step; 8 bits: codes are off by 1 % of the largest of a block, a few per cent of lr a step
            close(ctx.read(params[i]), want[i], step * (2e-6 if bits == 32 else 0.1 * o["lr"]))
    opt.init(ctx)  # from the start again
    before = [ctx.read(p) for p in params]
    g = [np.full(s, 0.5, np.float32) for s in shapes]
    opt.update(dict(zip(params, [ctx.var(x) for x in g])), ctx)
    for p, b in zip(params, before):
        close(ctx.read(p), b * (1 - o["lr"] * o["weight_decay"]) - o["lr"], 1e-5)


@pytest.mark.parametrize("bits", [32, 8])
def test_products_read_updated_parameters(ctx, bits):
    """What the tensor cores keep of a parameter (pieces, planes) is of its new values after an update: forward products and training ones."""
    rng = np.random.default_rng(9)
    x, w = rng.standard_normal((256, 128)).astype(np.float32), rng.standard_normal((128, 256)).astype(np.float32)
    xv, wv = ctx.var(x), ctx.var(w)
    y = xv.matmul(wv)
    loss = (y * y).sum(None)
    gw, gx = S.grad(loss, [wv, xv])
    opt = S.AdamW(0.5, weight_decay=0.0, state_bits=bits)
    opt.init(ctx)
    for _ in range(3):
        ctx.clear()
        ctx.eval(y, gw, gx, loss)
        now = ctx.read(wv).astype(np.float64)
        product = x.astype(np.float64) @ now
        assert np.abs(ctx.read(y) - product).max() < 1e-3 * np.abs(product).max()
        back = 2 * product @ now.T
        assert np.abs(ctx.read(gx) - back).max() < 1e-3 * np.abs(back).max()
        opt.update({wv: gw}, ctx)
        assert np.abs(ctx.read(wv) - now).max() > 0.1


def test_the_example_learns():
    spec = importlib.util.spec_from_file_location("language_model_example", os.path.join(ROOT, "examples", "language_model.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    losses, found = M.main(["--steps", "150", "--tokens", "300", "--width", "32"])
    assert losses[0] > 4.0 and losses[-1] < 1.5 and sum(found) >= 3
