"""The lazy-graph forms of dropout, the norms around a block and the log probabilities from hidden states on a B200, alone and together as a training step
uses them."""
import importlib.util
import os

import numpy as np
import pytest

import sage_b200 as S

import block_oracle as B
import head_oracle as H
import language_oracle as O
from test_gpu_language import close

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SEED = np.array([7, 0xfffffff0], np.uint32)


@pytest.fixture()
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


@pytest.mark.parametrize("extents", [(5,), (3, 4, 5), (64, 96)])
def test_dropout_and_its_gradient(ctx, extents):
    rng = np.random.default_rng(1)
    x, w = (rng.standard_normal(extents).astype(np.float32) for _ in range(2))
    xv, sv = ctx.var(x), ctx.var(SEED)
    y = S.dropout(xv, sv, 0.3, site=5)
    g = xv.grad((y * ctx.var(w)).sum(None))
    for seed in (SEED, SEED + np.uint32(9)):  # the mask follows the variable
        ctx.set(sv, seed)
        ctx.clear()
        ctx.eval(y, g)
        f = B.factors(seed, 5, extents, 0.3)
        close(ctx.read(y), x * f, 2 * O.U * np.abs(x * f))
        close(ctx.read(g), w * f, 2 * O.U * np.abs(w * f))
    turned = S.dropout(xv.permute(range(len(extents))[::-1]), sv, 0.3)
    f = B.factors(SEED + np.uint32(9), 0, extents[::-1], 0.3)
    close(turned.eval(ctx), x.T * f, 2 * O.U * np.abs(x.T * f))


@pytest.mark.parametrize("used", ["both", "out", "h"])
@pytest.mark.parametrize("after,before,gate,p,extents", [("none", "layer", 0, 0.1, (4, 6, 40)), ("rms", "rms", 1, 0.0, (7, 33)), ("layer", "layer", 3, 0.25, (3, 5, 64)), ("rms", "none", 1, 0.5, (9, 768))])
def test_block_norms_and_their_gradients(ctx, used, after, before, gate, p, extents):
    if used == "h" and before == "none":
        return
    rng = np.random.default_rng(len(after) + gate)
    dim, rows = extents[-1], int(np.prod(extents[:-1]))
    draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    host = dict(aw=1 + draw(dim) if after != "none" else None, ab=draw(dim) if after == "layer" else None, bw=1 + draw(dim) if before != "none" else None,
                bb=draw(dim) if before == "layer" else None, gate=None if not gate else draw(dim) if gate == 1 else draw(gate, dim))
    o = B.Norms(after, before, scale=0.5, p=p, seed=SEED, site=2, **host)
    x, y, wo, wh = (draw(*extents) for _ in range(4))
    v = {k: None if a is None else ctx.var(a) for k, a in host.items()}
    xv, yv = ctx.var(x), ctx.var(y)
    out, h = S.block_norms(xv, yv, after, v["aw"], v["ab"], before, v["bw"], v["bb"], v["gate"], residual_scale=0.5, p=p, seed=ctx.var(SEED) if p else None, site=2)
    assert out.extents == extents and (h is None) == (before == "none")
    loss = ([(out * ctx.var(wo)).sum(None)] if used != "h" else []) + ([(h * ctx.var(wh)).sum(None)] if used != "out" and h is not None else [])
    loss = loss[0] + loss[1] if len(loss) > 1 else loss[0]
    names = {"dx": xv, "dy": yv, "dafter_weight": v["aw"], "dafter_bias": v["ab"], "dgate": v["gate"]}
    if used != "out":
        names.update(dbefore_weight=v["bw"], dbefore_bias=v["bb"])
    names = {k: t for k, t in names.items() if t is not None}
    grads = dict(zip(names, S.grad(loss, list(names.values()))))
    ctx.eval(out, *([h] if h is not None else []), *grads.values())
    flat = lambda a: a.reshape(rows, dim)  # noqa: E731
    want, tol = o.out(flat(x), flat(y))
    got = flat(ctx.read(out))
    close(got, want, tol)
    if h is not None:
        want, tol = o.h(got)
        close(flat(ctx.read(h)), want, tol + O.U * np.abs(want))
    sa, sb = B.statistics(flat(y), after, o.eps), B.statistics(got, before, o.eps)
    stats = np.concatenate(sa[:2] + sb[:2], 1)
    found = o.grad(got, flat(y), stats, flat(wo) if used != "h" else None, flat(wh) if used != "out" and h is not None else None)
    for name, g in grads.items():
        value, tol = found[name]
        # (the kernel's statistics are off by their own bounds: a relative error of the unit rows, and their shift)
        off = max((t[2] * t[1] + t[3] / t[1]).max() for t in (sa, sb))
        close(ctx.read(g).reshape(value.shape), value, tol + 8 * off * (np.abs(value) + np.abs(value).max()))


@pytest.mark.parametrize("rows,vocab,dim,scale", [(9, 70, 24, 1.0), (130, 1000, 64, 0.7), (1, 33, 5, 1.0)])
def test_head_log_probs_and_their_gradients(ctx, rows, vocab, dim, scale):
    rng = np.random.default_rng(rows)
    h, w = rng.standard_normal((rows, dim)).astype(np.float32), (rng.standard_normal((vocab, dim)) * 0.4).astype(np.float32)
    ids = rng.integers(-1, vocab, rows).astype(np.int32)
    gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    hv, wv = ctx.var(h), ctx.var(np.ascontiguousarray(w.T))  # the weight as a transposed variable
    lp, en = S.head_log_probs(hv, wv.tr(), ctx.var(ids.reshape(rows, 1)), scale)
    dh, dw = S.grad((lp * ctx.var(gl)).sum(None) + (en * ctx.var(ge)).sum(None), [hv, wv])
    ctx.eval(lp, en, dh, dw)
    o = H.Head(h, w, ids, scale, "f32")
    at = np.clip(ids, 0, vocab - 1)[:, None]
    close(ctx.read(lp), np.where(o.scored, np.take_along_axis(o.log_p, at, 1)[:, 0], 0.0), np.take_along_axis(o.tol_log_p, at, 1)[:, 0])
    close(ctx.read(en), o.entropy, o.tol_entropy)
    found = o.gradients(gl, ge, "f32")
    close(ctx.read(dh), *found["dhidden"])
    close(ctx.read(dw).T, *found["dweight"])


def test_refusals(ctx):
    f = lambda *e, d=S.F32: S.Var.empty(e, d)  # noqa: E731
    x, seed = f(6, 8), f(2, d=S.U32)

    def refused(match, call, *a, **k):
        with pytest.raises(S.SageError) as e:
            call(*a, **k)
        assert match in str(e.value), str(e.value)
    refused("seed", S.dropout, x, f(3, d=S.U32), 0.1)
    refused("p must", S.dropout, x, seed, 1.0)
    refused("f32", S.dropout, f(6, d=S.I32), seed, 0.1)
    refused("seed", S.block_norms, x, x, p=0.1)
    refused("need a block", S.block_norms, x, gate=f(8))
    refused("divide", S.block_norms, x, x, gate=f(4, 8))
    refused("without its norm", S.block_norms, x, x, after_weight=f(8))
    refused("extents", S.block_norms, x, f(6, 9))
    refused("eps", S.block_norms, x, x, eps=0.0)
    refused("16384", S.block_norms, f(2, 16385), before="rms")
    refused("called", S.block_norms, x, x, before="batch")
    refused("width", S.head_log_probs, x, f(9, 7), f(6, d=S.I32))
    refused("id for each row", S.head_log_probs, x, f(9, 8), f(5, d=S.I32))
    refused("scale", S.head_log_probs, x, f(9, 8), f(6, d=S.I32), scale=0.0)


class Step:
    """A training step of two residual blocks over embedded tokens, in numpy's 64 bits: the loss alone."""

    def __init__(self, ids, after, seed, p):
        self.ids, self.after, self.seed, self.p = ids, after, seed, p

    def loss(self, t):
        rms = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(1e-5))) * w  # noqa: E731
        x = t["table"][self.ids] * 3.0
        x = x * B.factors(self.seed, 0, x.shape, self.p)
        h = rms(x, t["n0"])
        for i in (1, 2):
            y = np.maximum(h @ t["up%d" % i], 0.0) @ t["down%d" % i]
            y = rms(y, t["a%d" % i]) * B.factors(self.seed, i, y.shape, self.p)
            x = 0.8 * x + t["gate%d" % i] * y
            h = rms(x, t["n%d" % i])
        logits = h @ t["table"].T
        m = logits.max(1, keepdims=True)
        logq = logits - m - np.log(np.exp(logits - m).sum(1, keepdims=True))
        entropy = -(np.exp(logq) * logq).sum(1)
        return -(logq[np.arange(len(self.after)), self.after].mean() + 0.01 * entropy.mean())


def test_a_training_step_of_them_together(ctx):
    """Values against 64 bits, every gradient against differences along a direction, and steps that follow them."""
    rng = np.random.default_rng(11)
    tokens, width, rows, p = 200, 48, 96, 0.2
    draw = lambda *s, std=1.0, mean=0.0: (mean + std * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    host = {"table": draw(tokens, width, std=0.3), "n0": draw(width, std=0.1, mean=1.0)}
    for i in (1, 2):
        host.update({"up%d" % i: draw(width, 96, std=0.15), "down%d" % i: draw(96, width, std=0.1), "a%d" % i: draw(width, std=0.1, mean=1.0), "n%d" % i: draw(width, std=0.1, mean=1.0),
                     "gate%d" % i: draw(width, std=0.1, mean=0.5)})
    ids, after = rng.integers(0, tokens, rows), rng.integers(0, tokens, rows)
    v, sv = {k: ctx.var(a) for k, a in host.items()}, ctx.var(SEED)
    x = S.dropout(S.embedding(v["table"], ctx.var(ids.astype(np.int32)), 3.0), sv, p)
    x, h = S.block_norms(x, before="rms", before_weight=v["n0"])
    for i in (1, 2):
        y = S.relu(h.matmul(v["up%d" % i])).matmul(v["down%d" % i])
        x, h = S.block_norms(x, y, "rms", v["a%d" % i], None, "rms", v["n%d" % i], None, v["gate%d" % i], 0.8, p=p, seed=sv, site=i)
    lp, en = S.head_log_probs(h, v["table"], ctx.var(after.astype(np.int32)))
    loss = -(lp.mean([0]) + en.mean([0]) * 0.01)
    grads = dict(zip(v, S.grad(loss, list(v.values()))))
    ctx.eval(loss, *grads.values())
    step, exact = Step(ids, after, SEED, p), {k: a.astype(np.float64) for k, a in host.items()}
    # (f32 sums of a few hundred terms throughout, a dozen operators deep: 1e-5 of the loss is a hundred roundings of it)
    assert abs(float(ctx.read(loss)[0]) - step.loss(exact)) < 1e-5 * abs(step.loss(exact))
    for name, g in grads.items():
        got = ctx.read(g).astype(np.float64)
        for seed in (1, 2):
            d = np.random.default_rng(seed).standard_normal(got.shape)
            e = 1e-5
            moved = [step.loss({**exact, name: exact[name] + s * e * d}) for s in (1, -1)]
            # a rectifier may switch between the two ends: as many of them as lie within e of zero, each by e at most
            assert abs((got * d).sum() - (moved[0] - moved[1]) / (2 * e)) < 2e-4 * np.abs(got).sum() + 1e-7, name
    opt = S.AdamW(2e-2)
    opt.init(ctx)
    first = float(ctx.read(loss)[0])
    for i in range(8):
        ctx.clear()
        ctx.eval(loss, *grads.values())
        opt.update({v[k]: g for k, g in grads.items()}, ctx)
    ctx.clear()
    ctx.eval(loss)
    assert np.isfinite(float(ctx.read(loss)[0])) and float(ctx.read(loss)[0]) != first


def test_the_example_with_blocks():
    spec = importlib.util.spec_from_file_location("language_model_example", os.path.join(ROOT, "examples", "language_model.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    losses, found = M.main(["--steps", "6", "--tokens", "150", "--width", "32", "--blocks", "2", "--batch", "256"])
    assert len(losses) == 6 and np.isfinite(losses).all() and len(found) == 5
