"""Rules of the language-model operators that a planning context shows: what is accepted, what is launched, whose memory is whose."""
import numpy as np
import pytest

import sage_b200 as S


@pytest.fixture()
def ctx():
    c = S.Context(-1)
    yield c
    c.close()


def test_adamw_launches_once_for_parameters_of_the_same_step(ctx):
    a, b = ctx.var(np.zeros((10, 8), np.float32)), ctx.var(np.zeros((5,), np.float32))
    ga, gb = ctx.var(np.zeros((10, 8), np.float32)), ctx.var(np.zeros((5,), np.float32))
    opt = S.AdamW(1e-3)
    opt.init(ctx)

    def launches(grads):
        ctx.trace_begin()
        opt.update(grads, ctx)
        return ctx.trace().count("adamw_step")

    assert launches({a: ga, b: gb}) == 1
    assert launches({b: gb}) == 1
    assert launches({a: ga, b: gb}) == 2  # steps 2 and 3
    assert launches({a: ga}) == 1
    assert launches({a: ga, b: gb}) == 1  # both step 4
    opt.init(ctx)
    assert launches({a: ga}) == 1 and launches({a: ga, b: gb}) == 2
