"""Rules of the language-model operators on a B200 that single calls do not show: steps of an optimizer's parameters."""
import numpy as np
import pytest

import sage_b200 as S

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
