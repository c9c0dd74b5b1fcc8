"""What the language-model operators refuse, and what they launch: argument checks run before anything touches a device, so a planning
context sees all of them."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L


@pytest.fixture()
def ctx():
    c = S.Context(-1)
    yield c
    c.close()


def refused(f, *a, match="", **k):
    with pytest.raises(S.SageError) as e:
        f(*a, **k)
    assert e.value.code == 1 and match in str(e.value), str(e.value)


def test_embedding_refusals(ctx):
    t, i, y = ctx.empty((10, 8)), ctx.empty((4,), S.I32), ctx.empty((4, 8))
    L.embedding(t, i, y)
    refused(L.embedding, t, ctx.empty((5,), S.I32), y, match="ids")
    refused(L.embedding, t, ctx.empty((4,)), y, match="i32")
    refused(L.embedding, t, i, ctx.empty((4, 7)), match="width")
    refused(L.embedding, t, i, ctx.empty((4, 8), S.BF16), match="type")
    refused(L.embedding, ctx.empty((10, 8), S.I32), i, y, match="table")
    refused(L.embedding, ctx.empty((10, 8), S.U8), i, y, match="table")
    refused(L.embedding, t, i, y, scale=float("nan"), match="scale")
    refused(L.embedding, t.view((10, 8), (1, 10)), i, y, match="contiguous")
    refused(L.embedding, t, i, y.view((4, 8), (4, 1)), match="overlap")
    refused(L.embedding, t.view((11, 8), (8, 1)), i, y, match="behind the end")
    refused(L.embedding, t.view((10, 8), (8, 1), 1), i, y, match="behind the end")
    refused(L.embedding, t.view((1, 8), (1 << 60, 1), -1), i, y, match="in front")
    refused(L.embedding, t.view((3, 8), (1 << 62, 1)), i, y, match="behind the end")
    refused(L.embedding, t.view((3, 8), (-8, 1), 16), i, y, match="negative")
    refused(L.embedding, t.view((80,), (1,)), i, y, match="rank 2")


def test_embedding_grad_refusals(ctx):
    g, i, d = ctx.empty((4, 8), S.BF16), ctx.empty((4,), S.U32), ctx.empty((10, 8))
    L.embedding_grad(g, i, d)
    refused(L.embedding_grad, g, i, ctx.empty((10, 8), S.BF16), match="f32")
    refused(L.embedding_grad, g, i, ctx.empty((10, 9)), match="width")
    refused(L.embedding_grad, g, ctx.empty((3,), S.U32), d, match="ids")
    refused(L.embedding_grad, g, i, d.view((10, 8), (0, 1)), match="overlap")
    refused(L.embedding_grad, g, i, d, scale=float("inf"), match="scale")


def test_log_probs_refusals(ctx):
    x, i, lp = ctx.empty((3, 50)), ctx.empty((3,), S.I32), ctx.empty((3,))
    L.token_log_probs(x, i, lp)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(L.token_log_probs, x, i, lp, scale=scale, match="scale")
    refused(L.token_log_probs, ctx.empty((3, 50), S.I32), i, lp, match="logits")
    refused(L.token_log_probs, x, ctx.empty((4,), S.I32), lp, match="ids")
    refused(L.token_log_probs, x, i, ctx.empty((3,), S.I32), match="log_probs")
    refused(L.token_log_probs, x, i, lp.view((3,), (0,)), match="overlap")
    refused(L.token_log_probs, x, i, lp, ctx.empty((2,)), match="entropy")
    refused(L.token_log_probs, x, i, lp, stats=ctx.empty((3, 3)), match="stats")
    refused(L.token_log_probs, x, i, lp, top_ids=ctx.empty((3, 4), S.I32), match="top_log_probs")
    refused(L.token_log_probs, x, i, lp, top_log_probs=ctx.empty((3, 4)), match="top_ids")
    refused(L.token_log_probs, x, i, lp, top_ids=ctx.empty((3, 33), S.I32), top_log_probs=ctx.empty((3, 33)), match="32")
    refused(L.token_log_probs, x, i, lp, top_ids=ctx.empty((3, 4), S.I32), top_log_probs=ctx.empty((3, 5)), match="width")
    refused(L.token_log_probs, x, i, lp, top_ids=ctx.empty((3, 4)), top_log_probs=ctx.empty((3, 4)), match="i32")
    refused(L.token_log_probs, ctx.empty((3, 5)), i, lp, top_ids=ctx.empty((3, 6), S.I32), top_log_probs=ctx.empty((3, 6)), match="more than there are tokens")
    refused(L.token_log_probs, ctx.empty((3, 0)), i, lp, match="without elements")
    L.token_log_probs(ctx.empty((0, 50)), ctx.empty((0,), S.I32), ctx.empty((0,)))


def test_log_probs_grad_refusals(ctx):
    x, i, st, en, g = ctx.empty((3, 50), S.F16), ctx.empty((3,), S.I32), ctx.empty((3, 2)), ctx.empty((3,)), ctx.empty((3,))
    dx = ctx.empty((3, 50), S.F16)
    L.token_log_probs_grad(x, i, st, en, g, g, dx)
    L.token_log_probs_grad(x, i, st, None, None, None, x)
    refused(L.token_log_probs_grad, x, i, st, None, g, g, dx, match="entropy")
    refused(L.token_log_probs_grad, x, i, st, en, g, g, ctx.empty((3, 50)), match="dlogits")
    refused(L.token_log_probs_grad, x, i, ctx.empty((3, 2), S.I32), en, g, g, dx, match="stats")
    refused(L.token_log_probs_grad, x, i, st, en, ctx.empty((2,)), g, dx, match="g_log_probs")
    refused(L.token_log_probs_and_grad, x, i, g, ctx.empty((3,), S.I32), en, en, dx, match="g_entropy")
    refused(L.token_log_probs_and_grad, x, i, g, g, en, en, dx.view((3, 50), (0, 1)), match="overlap")


def test_adamw_refusals(ctx):
    f, n = (lambda *s, d=S.F32: ctx.empty(s, d)), 300
    step = lambda *t, **o: L.adamw_step(L.AdamWTensors(ctx, t), **dict(dict(step=1, lr=1e-3), **o))  # noqa: E731
    ok = L.adamw_tensor(f(n), f(n), f(n), f(n))
    ok8 = L.adamw_tensor(f(n), f(n), f(n, d=S.I8), f(n, d=S.U8), f(2), f(2))
    step(ok)
    step(ok8)
    step()
    for o in (dict(step=0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(lr=float("nan")), dict(grad_scale=float("inf")), dict(weight_decay=float("nan"))):
        refused(step, ok, **o)
    refused(step, ok, ok8, match="kind")
    refused(step, ok8, ok, match="kind")
    refused(step, L.adamw_tensor(f(n), f(n + 1), f(n), f(n)), match="grad")
    refused(step, L.adamw_tensor(f(n, d=S.BF16), f(n), f(n), f(n)), match="param")
    refused(step, L.adamw_tensor(f(n), f(n, d=S.I32), f(n), f(n)), match="grad")
    refused(step, L.adamw_tensor(f(n), f(n), f(n, d=S.I8), f(n, d=S.U8), f(1), f(2)), match="m_scale")
    refused(step, L.adamw_tensor(f(n), f(n), f(n, d=S.I8), f(n, d=S.U8)), match="scale")
    refused(step, L.adamw_tensor(f(n), f(n), f(n), f(n), copy=f(n)), match="copy")
    refused(step, L.adamw_tensor(f(2 * n).view((n,), (2,)), f(n), f(n), f(n)), match="contiguous")
    m, v = f(n, d=S.I8), f(n, d=S.U8)
    L.adamw_states(m, f(2), v, f(2), f(n), f(n))
    refused(L.adamw_states, v, f(2), v, f(2), f(n), f(n), match="i8")
    refused(L.adamw_states, m, f(3), v, f(2), f(n), f(n), match="m_scale")
    refused(L.adamw_states, m, f(2), v, f(2), f(n), f(n - 1), match="v_out")


def test_another_contexts_buffers_are_refused(ctx):
    other = S.Context(-1)
    t = other.empty((10, 8))
    refused(lambda: L.embedding(t, ctx.empty((4,), S.I32), ctx.empty((4, 8))), match="another context")
    other.close()


def test_missing_operands_are_refused(ctx):
    for call in ("sage_embedding", "sage_embedding_grad", "sage_token_log_probs", "sage_token_log_probs_grad", "sage_token_log_probs_and_grad"):
        n = {"sage_embedding": 2, "sage_embedding_grad": 2}.get(call, 2)
        args = [None] * n + [S.ctypes.c_float(1.0)] + [None] * 8
        if call == "sage_embedding_grad":
            args = [None, None, S.ctypes.c_float(1.0), 0, None]
        assert getattr(S.lib, call)(ctx.h, *args) == 1
        assert getattr(S.lib, call)(None, *args) == 1
    assert S.lib.sage_adamw_step(ctx.h, None, 1, None) == 1


def test_other_operators_refuse_narrow_elements(ctx):
    """Elements of 2 and 1 bytes are for these operators; one that reads 4 bytes an element would read behind the end."""
    y = ctx.empty((4, 8))
    for d in (S.F16, S.BF16, S.I8, S.U8):
        x = ctx.empty((4, 8), d)
        assert S.lib.sage_map(ctx.h, b"x0", x.ref(), 1, y.ref()) == 1
        assert S.lib.sage_map(ctx.h, b"x0", y.ref(), 1, x.ref()) == 1
        assert S.lib.sage_softmax(ctx.h, x.ref(), S.ctypes.c_int64(4), S.ctypes.c_int64(8), y.ref()) == 1
        assert S.lib.sage_log_sum_exp(ctx.h, x.ref(), S.ctypes.c_int64(4), S.ctypes.c_int64(8), y.ref()) == 1
        assert S.lib.sage_reduce(ctx.h, 0, x.ref(), (S.ctypes.c_int32 * 1)(1), 1, ctx.empty((4,)).ref()) == 1
        assert S.lib.sage_concat(ctx.h, x.ref(), 1, 0, y.ref()) == 1
        assert S.lib.sage_gather(ctx.h, x.ref(), y.ref(), 0, y.ref()) == 1
        with pytest.raises(S.SageError):
            S.Var.empty([4], d)


def test_wrapped_memory_is_not_freed(ctx):
    used = ctx.mem_stats()["mem_used"]
    t = ctx.wrap(0x1000, (4, 8), S.BF16, (16, 1))
    assert S.lib.sage_buf_size(t.buf) == 2 * (3 * 16 + 8) and S.lib.sage_buf_ptr(t.buf) == 0x1000
    t.release()
    assert ctx.mem_stats()["mem_used"] == used
    with pytest.raises(S.SageError):
        ctx.wrap(0, (4,))


# ------------------------------------------------------------------------------------------ the lazy graph
def test_graph_shapes_and_launches(ctx):
    table, ids = ctx.var(np.zeros((10, 8), np.float32)), ctx.var(np.zeros((2, 3), np.uint32))
    y = S.embedding(table, ids, 2.0)
    assert y.extents == (2, 3, 8)
    logits = S.view(y, [6, 8]).matmul(table.tr())
    lp, h = S.token_log_probs(logits, ctx.var(np.zeros(6, np.int32)))
    assert lp.extents == (6,) and h.extents == (6,)
    top = S.top_tokens(logits, 3)
    assert top.extents == (6, 3) and top.dtype == S.U32
    loss = -(lp.mean([0]) + h.mean([0]) * 0.1)
    ctx.trace_begin()
    ctx.eval(loss, top, table.grad(loss))
    names = ctx.trace()
    for name in ("embedding", "token_log_probs", "token_log_probs_grad", "embedding_sort", "embedding_grad"):
        assert name in names, names
    opt = S.AdamW(1e-3, state_bits=8)
    opt.init(ctx)
    ctx.trace_begin()
    opt.update({table: ctx.var(np.zeros((10, 8), np.float32))}, ctx)
    assert "adamw_step" in ctx.trace()


def test_graph_refusals(ctx):
    table, ids = ctx.var(np.zeros((10, 8), np.float32)), ctx.var(np.zeros((6,), np.uint32))
    f = ctx.var(np.zeros((6,), np.float32))
    for call in (lambda: S.embedding(table, f), lambda: S.embedding(f, ids), lambda: S.token_log_probs(table, ids), lambda: S.token_log_probs(f, ids),
                 lambda: S.token_log_probs(ctx.var(np.zeros((6, 8), np.float32)), f), lambda: S.token_log_probs(ctx.var(np.zeros((6, 8), np.float32)), ids, 0.0),
                 lambda: S.top_tokens(table, 0), lambda: S.top_tokens(table, 9), lambda: S.top_tokens(f, 1),
                 lambda: S.AdamW(1e-3, state_bits=16), lambda: S.AdamW(1e-3, beta1=1.0), lambda: S.AdamW(1e-3, eps=0.0), lambda: S.AdamW(float("nan"))):
        with pytest.raises(S.SageError) as e:
            call()
        assert e.value.code == 1
    lp, _ = S.token_log_probs(ctx.var(np.zeros((6, 8), np.float32)), ids)
    x = ctx.var(np.zeros((6, 8), np.float32))
    lp, _ = S.token_log_probs(x, ids)
    with pytest.raises(S.SageError):
        x.grad(x.grad(lp.sum(None)).sum(None))  # differentiated once
