"""Steps of a training loop over dropout, norms around blocks and log probabilities from hidden states, each against 64 bits from the parameters that the last one left."""
import numpy as np
import pytest

import sage_b200 as S

import language_oracle as O
from test_gpu_blocks_graph import SEED, Step
from test_gpu_language import close

pytestmark = pytest.mark.gpu


def test_losses_and_parameters_follow_the_updates():
    ctx, rng = S.Context(0), np.random.default_rng(12)
    tokens, width, rows, p, lr = 120, 40, 64, 0.2, 1e-2
    draw = lambda *s, std=1.0, mean=0.0: (mean + std * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    host = {"table": draw(tokens, width, std=0.3), "n0": draw(width, std=0.1, mean=1.0)}
    for i in (1, 2):
        host.update({"up%d" % i: draw(width, 80, std=0.15), "down%d" % i: draw(80, width, std=0.1), "a%d" % i: draw(width, std=0.1, mean=1.0), "n%d" % i: draw(width, std=0.1, mean=1.0),
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
    opt = S.AdamW(lr)
    opt.init(ctx)
    o = {"lr": lr, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "grad_scale": 1.0}
    moments = {k: (np.zeros(a.shape), np.zeros(a.shape)) for k, a in host.items()}
    for step in range(1, 6):
        before = {k: ctx.read(a) for k, a in v.items()}
        seed = SEED + np.uint32(step)  # another mask for every step
        ctx.set(sv, seed)
        ctx.clear()
        ctx.eval(loss, *grads.values())
        exact = Step(ids, after, seed, p).loss({k: a.astype(np.float64) for k, a in before.items()})
        # (as the first step's: f32 sums of a few hundred terms, a dozen operators deep)
        assert abs(float(ctx.read(loss)[0]) - exact) < 1e-5 * abs(exact), step
        g = {k: ctx.read(a) for k, a in grads.items()}
        opt.update({v[k]: a for k, a in grads.items()}, ctx)
        for k, a in v.items():
            want, m, n, tol = O.adamw_64(before[k], *moments[k], g[k], {**o, "step": step})
            moments[k] = m, n
            # (the moments themselves are held in f32: two roundings of each for every step behind it)
            close(ctx.read(a), want, tol + 4 * step * O.U * np.abs(want - before[k]) + 4 * step * O.U * lr, k)
    assert ctx.status_word() == 0
    ctx.close()
