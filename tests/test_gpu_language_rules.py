"""Rules of the language-model operators on a B200 that single calls do not show: steps of an optimizer's parameters, codes of states that
lie midway between two."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import language_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


# ------------------------------------------------------------------------------------------ steps of the graph's AdamW
class Followed:
    """A parameter and the 64-bit rule's value of it, by its own count of updates.

    Bound with 32-bit states: adamw_64's of each step, whose 12 roundings become 12 + 4 k <= 12 (k + 1) behind k steps of moments that
    carry four roundings each.  With 8 bits a code is within 1 % of the block's largest, here a few per cent of lr a step."""

    def __init__(self, ctx, rng, shape, rule, bits):
        self.ctx, self.rng, self.rule, self.bits = ctx, rng, rule, bits
        value = rng.standard_normal(shape).astype(np.float32)
        self.var, self.want, self.m, self.v, self.steps, self.bound = ctx.var(value), value.astype(np.float64), np.zeros(shape), np.zeros(shape), 0, np.zeros(shape)

    def gradient(self):
        g = (self.rng.standard_normal(self.want.shape) + 1.0).astype(np.float32)
        self.steps += 1
        self.want, self.m, self.v, bound = O.adamw_64(self.want, self.m, self.v, g, dict(self.rule, step=self.steps, grad_scale=1.0))
        self.bound = self.bound + (self.steps * bound if self.bits == 32 else 0.1 * self.rule["lr"])
        return self.ctx.var(g)

    def check(self):
        off = np.abs(self.ctx.read(self.var).astype(np.float64) - self.want) - self.bound
        assert off.max() <= 0, (self.steps, off.max())


GRAPH_RULE = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_that_joins_later_starts_at_step_1(ctx, bits):
    rng = np.random.default_rng(bits)
    a, b, c = (Followed(ctx, rng, s, GRAPH_RULE, bits) for s in ((300, 40), (40,), (64, 64)))
    opt = S.AdamW(state_bits=bits, **GRAPH_RULE)
    opt.init(ctx)
    for i in range(12):
        now = [a] + [b] * (i >= 5) + [c] * (i >= 5 and i != 8)
        opt.update({p.var: p.gradient() for p in now}, ctx)
        for p in (a, b, c):
            p.check()


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_updated_by_calls_of_their_own(ctx, bits):
    rng = np.random.default_rng(bits + 1)
    groups = [[Followed(ctx, rng, s, GRAPH_RULE, bits) for s in shapes] for shapes in (((300, 40), (1,)), ((64, 64), (7,)))]
    opt = S.AdamW(state_bits=bits, **GRAPH_RULE)
    opt.init(ctx)
    for _ in range(6):
        for group in groups:
            opt.update({p.var: p.gradient() for p in group}, ctx)
            for p in group:
                p.check()


# ------------------------------------------------------------------------------------------ codes midway
@pytest.mark.parametrize("first,last", [(0, 60), (60, 186), (186, 255)])
@pytest.mark.parametrize("moment", ["m", "v"])
def test_codes_near_the_middle_of_two(ctx, moment, first, last):
    """Moments within a few f32 steps of where the code changes: the codes are those of the operations rounded one by one."""
    top = 127 if moment == "m" else 255
    first, last = (first // 2, last // 2) if moment == "m" else (first, last)
    f, blocks = np.float32, 4096
    rng = np.random.default_rng(first + top)
    largest = np.exp2(rng.uniform(-3, 3, (blocks, 1))).astype(f)
    c = rng.integers(first, last, (blocks, 256)) + 0.5
    with np.errstate(divide="ignore"):
        factor = f(1) / (largest if moment == "m" else np.sqrt(largest * largest)) * f(top * top)
    g = (c * c / factor).astype(f)
    g = (g.view(np.int32) + rng.integers(-12, 13, g.shape)).astype(np.int32).view(f)
    g[:, 0] = largest[:, 0]
    n = g.size
    g = g.reshape(-1)
    t = [ctx.tensor(np.zeros(n, f)), ctx.tensor(g), ctx.tensor(np.zeros(n, np.int8), S.I8), ctx.tensor(np.zeros(n, np.uint8), S.U8), ctx.tensor(np.zeros(blocks, f)), ctx.tensor(np.zeros(blocks, f))]
    L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(*t)]), step=1, lr=1e-3, beta1=0.0, beta2=0.0)
    m, v = O.adamw_f32(np.zeros(n, f), np.zeros(n, f), g, 0.0, 0.0, 1.0)
    (mc, ms), (vc, vs) = O.adamw_encode(m, 127), O.adamw_encode(np.sqrt(v), 255)
    got = [x.numpy() for x in t[2:]]
    for x in t:
        x.release()
    assert np.array_equal(got[2], ms) and np.array_equal(got[3], vs)
    assert (got[0] != mc).sum() == 0 and (got[1] != vc).sum() == 0


# ------------------------------------------------------------------------------------------ differences beyond f32
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(3, 40), (2, 70001)])
def test_log_probabilities_of_logits_further_apart_than_f32_reaches(ctx, kind, rows, vocab):
    """Masks of the type's lowest value beside logits of 2e38: their difference is beyond f32, a quarter of it is not."""
    rng = np.random.default_rng(vocab)
    x = np.full((rows, vocab), -3.38e38)
    x[:, 3:9] = rng.uniform(1.9e38, 2e38, (rows, 6))
    x[:, 7] = 2.5e38
    raw, x = O.stored(x, kind)
    ids = np.zeros(rows, np.int32)
    ids[1] = 7
    want = O.LogProbs(x, ids, 0.25)
    t, i = ctx.tensor(raw, S.BF16 if kind == "bf16" else S.F32), ctx.tensor(ids)
    lp, h, dx, one = ctx.empty((rows,)), ctx.empty((rows,)), ctx.empty((rows, vocab), t.dtype), ctx.tensor(np.ones(rows, np.float32))
    top_ids, top = ctx.empty((rows, 8), S.I32), ctx.empty((rows, 8))

    def close(got, value, bound):
        assert np.isfinite(value).all() and (np.abs(got.astype(np.float64) - value) <= bound).all(), (got, value)

    L.token_log_probs(t, i, lp, h, top_ids=top_ids, top_log_probs=top, scale=0.25)
    close(lp.numpy(), want.log_probs, want.tol_log_probs)
    order, value, bound = want.top(8)
    assert np.array_equal(top_ids.numpy(), order)
    close(top.numpy(), value, bound)
    L.token_log_probs_and_grad(t, i, one, one, lp, h, dx, scale=0.25)
    close(lp.numpy(), want.log_probs, want.tol_log_probs)
    g, bound = want.grad(1.0, 1.0, kind)
    close(O.values(dx.numpy(), kind), g, bound)
    for x in (t, i, lp, h, dx, one, top_ids, top):
        x.release()
