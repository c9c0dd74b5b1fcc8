"""The gradient of the norms around a block on a B200 where the block's output is not a number: as the formula has it, whatever kernel takes the call."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import block_oracle as B
from test_gpu_blocks import SEED
from test_gpu_language import Held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim", [("f32", 64), ("bf16", 64), ("bf16", 1032), ("f32", 63)])
@pytest.mark.parametrize("gate", [1, 4])
@pytest.mark.parametrize("carried", [0.0, 1.0])
def test_a_gate_behind_values_that_are_not_numbers(kind, dim, gate, carried):
    """An element that is dropped may be anything.  One that stays makes its gate's gradient what zero or another gradient times it is: not a number."""
    ctx, rng, rows, p = S.Context(0), np.random.default_rng(dim), 12, 0.5
    x, y = rng.standard_normal((rows, dim)), rng.standard_normal((rows, dim))
    y[5, ::2], y[5, 1::2] = np.nan, np.inf
    go, gh = rng.standard_normal((rows, dim)), rng.standard_normal((rows, dim))
    go[5], gh[5] = carried * go[5], 0.0
    with Held(ctx) as d:
        t = lambda a: d.rows(a, kind)[0]  # noqa: E731
        shape = (dim,) if gate == 1 else (gate, dim)
        norms = L.BlockNorms(ctx, before="rms", before_weight=d.put(np.ones(dim, np.float32)), gate=d.put(np.ones(shape, np.float32)), p=p, seed=d.put(SEED), site=4)
        stats = np.tile(np.array([0.0, 1.0, 0.0, 1.0], np.float32), (rows, 1))
        dx, dy, dgate = t(0 * x), t(0 * x), d.empty(shape)
        L.block_norms_grad(norms, t(x), t(y), d.put(stats), t(go), t(gh), dx, dy, dgate=dgate)
        found = dgate.numpy().reshape(-1, dim)
        kept = B.keep(SEED, 4, rows * dim, p).reshape(rows, dim)[5]
        group = 5 // (rows // len(found))
        infinite = np.arange(dim) % 2 == 1
        bad = kept & ~infinite if carried else kept  # (another gradient times an infinity is one)
        assert np.array_equal(np.isnan(found[group]), bad)
        assert np.array_equal(np.isinf(found[group]), kept & infinite if carried else np.zeros(dim, bool))
        assert np.isfinite(np.delete(found, group, 0)).all()
        assert np.isfinite(dy.numpy().astype(np.float64) if kind == "f32" else 0.0).all()
    assert ctx.status_word() == 0
    ctx.close()
