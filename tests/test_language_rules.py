"""Rules of the language-model operators that a planning context shows: what is accepted, what is launched, whose memory is whose."""
import os
import re

import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

KERNELS = os.path.join(os.path.dirname(os.path.abspath(S.__file__)), "csrc", "kernels")


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


def test_margins_within_which_codes_take_exact_roots():
    """Codes of 8-bit states are found from square roots that are 2^-23 off at most (the instruction's bound); the margins around one half
    within which exact roots decide have to cover all that separates the two ways: no run shows errors that this GPU's roots do not make."""
    text = open(os.path.join(KERNELS, "adamw.cu")).read()
    m_off, v_off = (float.fromhex(x) if "p" in x else float(x) for x in re.search(r"kMOff = ([^f;]*)f, kVOff = ([^f;]*)f;", text).groups())
    u, fast = 2.0 ** -24, 2.0 ** -23
    assert m_off > 127 * fast + 0.5 * 2.0 ** -17  # the exact root is rounded to the f32 grid, which has the middles
    # root, product, root; an error in front of a root halves
    assert v_off > 255 * ((fast + (u + fast) / 2) + (u + (u + u) / 2))


def test_token_ids_without_axes_are_refused(ctx):
    """Logits of one row and an id that has no axis: refused, however the variable came to have none."""
    logits = ctx.var(np.zeros((1, 8), np.float32))
    one = ctx.var(np.zeros(1, np.int32))
    S.token_log_probs(logits, one)
    for ids in (S.squeeze(one, 0), S.squeeze(S.squeeze(ctx.var(np.zeros((1, 1), np.int32)), 0), 0), S.Var.empty([], S.I32)):
        assert ids.extents == ()
        with pytest.raises(S.SageError) as e:
            S.token_log_probs(logits, ids)
        assert e.value.code == 1 and "one token id for each row" in str(e.value)


def test_adamw_refuses_weight_decay_that_is_not_finite(ctx):
    """As the constructor does, so that no update can make parameters NaN; the old value stays."""
    for opt, bad in ((S.AdamW(1e-3), (float("nan"), float("inf"), 1e39)), (S.AdamW(1e30), (1e20,))):
        opt.set_weight_decay(0.5)
        for w in bad:
            with pytest.raises(S.SageError) as e:
                opt.set_weight_decay(w)
            assert e.value.code == 1 and "finite" in str(e.value)
    for lr, w in ((1e-3, float("inf")), (0.0, float("nan")), (1e-40, 1e39)):
        with pytest.raises(S.SageError):
            S.AdamW(lr, weight_decay=w)
    for opt in (S.Sgd(1e-3), S.Adam(1e-3)):
        opt.set_weight_decay(0.5)


def test_graph_refuses_more_rows_or_columns_than_the_kernels_count(ctx):
    """2^31 - 2^16 rows, tokens or columns, as the operators on tensors; the kernels number rows and columns in 32 bits."""
    most = 2 ** 31 - 2 ** 16
    f, i = (lambda *e: S.Var.empty(e)), (lambda *e: S.Var.empty(e, S.I32))
    assert S.embedding(f(most, 1), i(1)).extents == (1, 1) and S.embedding(f(1, most), i(1)).extents == (1, most) and S.embedding(f(1, 1), i(most)).extents == (most, 1)
    S.token_log_probs(f(most, 1), i(most))
    S.token_log_probs(f(1, most), i(1))
    S.top_tokens(f(most, 1), 1)
    for call in (lambda: S.embedding(f(most + 1, 1), i(1)), lambda: S.embedding(f(1, most + 1), i(1)), lambda: S.embedding(f(1, 1), i(most + 1)), lambda: S.embedding(f(1, 1), i(2 ** 16, 2 ** 16)),
                 lambda: S.token_log_probs(f(most + 1, 1), i(most + 1)), lambda: S.token_log_probs(f(1, most + 1), i(1)), lambda: S.top_tokens(f(most + 1, 1), 1), lambda: S.top_tokens(f(1, most + 1), 1)):
        with pytest.raises(S.SageError) as e:
            call()
        assert e.value.code == 1 and "2^31 - 2^16" in str(e.value)


def test_views_of_any_size_are_checked_without_overflow(ctx):
    """Extents and strides whose products pass 64 and 128 bits reach behind the end of every buffer; views of nothing reach nowhere."""
    most = 2 ** 63 - 1
    step = lambda *t: L.adamw_step(L.AdamWTensors(ctx, [L.adamw_tensor(*t)]), step=1, lr=1e-3)  # noqa: E731
    for extents, strides in (((most, most), (most, 1)), ((most,) * 8, (most,) * 7 + (1,)), ((1, most, most), (1, most, 1)), ((2 ** 62, 4), (4, 1))):
        t = [ctx.empty((1,)).view(extents, strides) for _ in range(4)]
        with pytest.raises(S.SageError) as e:
            step(*t)
        assert e.value.code == 1 and "behind the end" in str(e.value)
    for extents, strides in (((0, most, most), (most, most, 1)), ((5, 0), (1, 1)), ((0,), (3,))):
        step(*[ctx.empty((1,)).view(extents, strides) for _ in range(4)])


def test_scales_whose_base_2_form_is_not_finite_are_refused(ctx):
    """Above 2.35e38 scale * log2(e), by which differences of logits are multiplied, is infinite, and 0 times that is no number."""
    x, i, v, st, dx = ctx.empty((3, 50)), ctx.empty((3,), S.I32), ctx.empty((3,)), ctx.empty((3, 2)), ctx.empty((3, 50))
    xv, iv = ctx.var(np.zeros((3, 50), np.float32)), ctx.var(np.zeros(3, np.int32))
    calls = (lambda s: L.token_log_probs(x, i, v, scale=s), lambda s: L.token_log_probs_grad(x, i, st, v, v, v, dx, scale=s),
             lambda s: L.token_log_probs_and_grad(x, i, v, v, ctx.empty((3,)), None, dx, scale=s), lambda s: S.token_log_probs(xv, iv, s))
    for call in calls:
        call(2.3e38)
        for scale in (2.4e38, 3.4e38):
            with pytest.raises(S.SageError) as e:
                call(scale)
            assert e.value.code == 1 and "scale" in str(e.value)
    table = ctx.var(np.zeros((3, 50), np.float32))
    for scale in (float("nan"), float("inf")):
        with pytest.raises(S.SageError) as e:  # as the operator on tensors
            S.embedding(table, iv, scale)
        assert e.value.code == 1 and "scale" in str(e.value)


# ------------------------------------------------------------------------------------------ memory of something else
class Foreign:
    """What Context.borrow takes of another package's tensor."""

    def __init__(self, shape=(4, 8), stride=(8, 1), dtype="float32", address=0x10000):
        self.shape, self._stride, self.dtype, self._address = shape, stride, dtype, address

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self._address


@pytest.fixture()
def freed(monkeypatch):
    """The handles that were released so far."""
    free, handles = S.lib.sage_free, []

    def counted(ctx, buf):
        handles.append(buf.value)
        return free(ctx, buf)

    monkeypatch.setattr(S.lib, "sage_free", counted)
    return handles


def test_handles_of_borrowed_memory_go_with_their_last_holder(ctx, freed):
    for make in (lambda: ctx.borrow(Foreign()), lambda: ctx.wrap(0x10000, (4, 8))):
        del freed[:]
        t = make()
        handle = t.buf.value
        del t
        assert freed == [handle]
        view = make().view((8,), (1,), 8)  # a view, a struct and a reference each keep it
        assert len(freed) == 1 and S.lib.sage_buf_size(view.buf) == 4 * 8 * 4
        struct = view.c()
        del view
        assert len(freed) == 1 and struct.buf
        del struct
        assert len(freed) == 2
        assert S.lib.sage_softmax(ctx.h, make().ref(), S.ctypes.c_int64(4), S.ctypes.c_int64(8), make().ref()) == 0
        assert len(freed) == 4
        tensors = L.AdamWTensors(ctx, [L.adamw_tensor(*[make() for _ in range(4)])])
        L.adamw_step(tensors, step=1, lr=1e-3)
        assert len(freed) == 4
        del tensors
        assert len(freed) == 8
        t = make()
        view = t.view((8,), (1,))
        t.release()  # at once; nothing is left to release behind it, and views have lost it too
        t.release()
        assert len(freed) == 9
        with pytest.raises(S.SageError):
            L.embedding(view, view, view)
        del t, view
        assert len(freed) == 9


def test_borrowed_memory_stays_while_a_view_has_it(ctx):
    import weakref
    foreign = Foreign()
    alive = weakref.ref(foreign)
    view = ctx.borrow(foreign).view((8,), (1,))
    del foreign
    assert alive() is not None
    del view
    assert alive() is None


def test_handles_that_outlive_their_context(freed):
    c = S.Context(-1)
    t = c.borrow(Foreign())
    c.close()
    del t
    assert not freed


def test_borrowing_reports_the_failure_that_it_met(ctx, monkeypatch):
    monkeypatch.setattr(S, "_buf_wrap", lambda *a: 4)
    for make in (lambda: ctx.borrow(Foreign()), lambda: ctx.wrap(0x10000, (4, 8))):
        with pytest.raises(S.SageError) as e:
            make()
        assert e.value.code == 4


def test_memory_of_something_else_has_no_negative_strides(ctx):
    """A size worked out of them would reach over all memory."""
    for make in (lambda: ctx.wrap(0x10000, (4,), S.F32, (-1,)), lambda: ctx.wrap(0x10000, (-4,)), lambda: ctx.borrow(Foreign((4, 8), (-8, 1)))):
        with pytest.raises(S.SageError) as e:
            make()
        assert e.value.code == 1


def test_released_tensors_are_refused_wherever_they_were_prepared(ctx):
    """Views, references and prepared updates hold a buffer's address; once it is released there is nothing behind it."""
    make = (lambda: ctx.empty((8,))), (lambda: ctx.borrow(Foreign((8,), (1,))))
    for new in make:
        t = [new() for _ in range(4)]
        update = L.AdamWTensors(ctx, [L.adamw_tensor(*t)])
        parts = L.AdamWTensors(ctx, [L.adamw_tensor(*[x.view((4,), (1,), 4) for x in t])])
        view, ids, y = t[0].view((2, 4), (4, 1)), ctx.empty((1,), S.I32), ctx.empty((1, 4))
        L.embedding(view, ids, y)
        L.adamw_step(update, step=1, lr=1e-3)
        new().release()  # others do not matter
        L.adamw_step(update, step=2, lr=1e-3)
        t[0].release()
        for call in (lambda: L.adamw_step(update, step=3, lr=1e-3), lambda: L.adamw_step(parts, step=3, lr=1e-3), lambda: L.embedding(view, ids, y), lambda: L.embedding(t[0], ids, y)):
            for _ in range(2):
                with pytest.raises(S.SageError) as e:
                    call()
                assert e.value.code == 1 and ("released" in str(e.value) or "missing" in str(e.value)), str(e.value)
