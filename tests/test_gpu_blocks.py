"""Dropout and the norms around a block on a B200 against plain implementations in 64 bits (block_oracle.py, which derives the bounds), through the
public package, at sizes, layouts, masks and values where they can go wrong."""
import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

import block_oracle as B
import language_oracle as O
from test_gpu_language import KIND, Held, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


def values(t, kind):
    return O.values(t.numpy(), kind)


SEED = np.array([0x89abcdef, 0x01234567], np.uint32)


# ------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pitch,lead,p,site", [
    (1, 1, None, 0, 0.5, 0), (1, 8, None, 0, 0.5, 1), (3, 5, None, 0, 0.25, 1 << 40), (7, 24, 32, 0, 0.1, 3), (7, 24, 25, 1, 0.1, 3), (5, 13, 13, 3, 0.9, (1 << 64) - 1),
    (24, 768, None, 0, 0.1, 0), (300, 1001, 1008, 0, 0.5, 7), (64, 4096, None, 0, 0.0, 2), (9, 17, None, 0, 1e-7, 5), (9, 40, None, 0, 0.9999999, 5)])
def test_dropout(ctx, kind, rows, cols, pitch, lead, p, site):
    rng = np.random.default_rng(rows * 1000 + cols)
    with Held(ctx) as d:
        x, xv = d.rows(rng.standard_normal((rows, cols)), kind, pitch, lead)
        y = d.empty((rows * (pitch or cols) + lead,), KIND[kind]).view((rows, cols), (pitch or cols, 1), lead)
        before = ctx.download(y.buf, (rows * (pitch or cols) + lead,), S._NP[KIND[kind]]).copy()
        L.dropout(x, y, d.put(SEED), p, site=site)
        f = B.factors(SEED, site, (rows, cols), p)
        close(values(y, kind), xv * f, B.stored_tol(xv * f, 2 * O.U * np.abs(xv * f), kind))
        assert np.array_equal(values(y, kind) == 0, (f == 0) | (xv == 0))
        after = ctx.download(y.buf, (rows * (pitch or cols) + lead,), S._NP[KIND[kind]])  # what lies between the rows stays as it was
        inside = np.zeros(before.size, bool)
        for r in range(rows):
            inside[lead + r * (pitch or cols):lead + r * (pitch or cols) + cols] = True
        assert np.array_equal(after[~inside], before[~inside])


def test_dropout_in_place_of_strange_values_and_by_the_seed_of_the_moment(ctx):
    with Held(ctx) as d:
        x = np.full((64, 64), np.nan, np.float32)
        x[::2] = np.inf
        t, seed = d.put(x), d.put(np.array([0, -5, 0, 7], np.int32)).view((2,), (2,), 1)
        L.dropout(t, t, seed, 0.5, site=9)
        kept = B.keep((-5, 7), 9, x.size, 0.5).reshape(x.shape)
        got = t.numpy()
        assert np.array_equal(got == 0, ~kept) and np.isnan(got[1::2][kept[1::2]]).all() and np.isposinf(got[::2][kept[::2]]).all()
        ones, s = d.put(np.ones((3, 1000), np.float32)), d.put(SEED)
        y = d.empty((3, 1000))
        L.dropout(ones, y, s, 0.3)
        ctx.upload(s.buf, SEED + np.uint32(1))
        z = d.empty((3, 1000))
        L.dropout(ones, z, s, 0.3)
        for got, key in ((y, SEED), (z, SEED + np.uint32(1))):
            assert np.array_equal(got.numpy() != 0, B.keep(key, 0, 3000, 0.3).reshape(3, 1000))
        L.dropout(ones, y, None, 0.0)
        assert (y.numpy() == 1).all()
        L.dropout(d.empty((0, 5)), d.empty((0, 5)), s, 0.3)


def test_dropout_of_broadcast_rows_and_shares(ctx):
    """The share that stays, of many elements, within six deviations; one row read for all."""
    with Held(ctx) as d:
        one, y, n = d.put(np.ones((1, 1 << 12), np.float32)), d.empty((256, 1 << 12)), 1 << 20
        for p in (0.1, 0.5):
            L.dropout(one.view((256, 1 << 12), (0, 1)), y, d.put(SEED), p, site=4)
            got = y.numpy()
            assert abs((got != 0).mean() - (1 - p)) < 6 * np.sqrt(p * (1 - p) / n) + 2.0 ** -17
            assert np.array_equal(got != 0, B.keep(SEED, 4, n, p).reshape(got.shape))


def test_dropout_of_more_elements_than_32_bits_count(ctx):
    """Rows far apart in the mask's count: the last ones of 2^33 elements (a broadcast row in, rows of one place out)."""
    rows, cols = (1 << 33) // 4096 + 3, 4096
    with Held(ctx) as d:
        y = d.empty((rows, cols), S.F16)
        x = d.put(np.ones((1, cols), np.float16), S.F16)
        L.dropout(x.view((rows, cols), (0, 1)), y, d.put(SEED), 0.5, site=1)
        tail = ctx.download(y.buf, (5 * cols,), np.float16, offset=(rows - 5) * cols * 2)
        first = (rows - 5) * cols
        want = np.concatenate([keep_block(SEED, 1, first // 8 + i) for i in range(5 * cols // 8)]) >= B.bar_of(0.5)
        assert np.array_equal(tail != 0, want)


def keep_block(seed, site, block):
    """Eight sixteen-bit numbers of one block, in Python's whole numbers."""
    x, key = [block & 0xffffffff, block >> 32, site & 0xffffffff, site >> 32], [int(seed[0]), int(seed[1])]
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(p1 >> 32) ^ x[1] ^ key[0], p1 & 0xffffffff, (p0 >> 32) ^ x[3] ^ key[1], p0 & 0xffffffff]
        key = [(key[0] + 0x9E3779B9) & 0xffffffff, (key[1] + 0xBB67AE85) & 0xffffffff]
    return np.array([h for w in x for h in (w & 0xffff, w >> 16)])


# ------------------------------------------------------------------------------------------ norms around a block
class Case:
    """Device tensors and the oracle of one description."""

    def __init__(self, d, rng, rows, dim, xk, k, after, before, gate=0, scale=1.0, p=0.0, affine=True, pitch=0, lead=0, site=11):
        self.d, self.rows, self.dim, self.xk, self.k, self.pitch, self.lead = d, rows, dim, xk, k, dim + pitch, lead
        w = lambda on, base: (base + 0.2 * rng.standard_normal(dim)).astype(np.float32) if on and affine else None  # noqa: E731
        self.host = dict(aw=w(after != "none", 1.0), ab=w(after == "layer", 0.0), bw=w(before != "none", 1.0), bb=w(before == "layer", 0.0),
                         gate=None if not gate else (0.5 + 0.3 * rng.standard_normal((dim,) if gate == 1 else (gate, dim))).astype(np.float32))
        self.oracle = B.Norms(after, before, scale=scale, p=p, seed=SEED, site=site, **self.host)
        t = {n: None if a is None else d.put(a) for n, a in self.host.items()}
        self.norms = L.BlockNorms(d.ctx, after=after, after_weight=t["aw"], after_bias=t["ab"], before=before, before_weight=t["bw"], before_bias=t["bb"], gate=t["gate"],
                                  residual_scale=scale, eps=1e-5, p=p, seed=d.put(SEED) if p else None, site=site)
        loud = np.exp(0.5 * rng.standard_normal(dim))
        self.x, self.xv = self.rows_of(rng.standard_normal((rows, dim)) * loud + 0.3, xk)
        self.y, self.yv = self.rows_of(rng.standard_normal((rows, dim)) * loud - 0.2, k)

    def rows_of(self, a, kind):
        return self.d.rows(a, kind, self.pitch, self.lead)

    def empty(self, kind):
        n = self.lead + max(self.rows, 1) * self.pitch
        return self.d.empty((n,), KIND[kind]).view((self.rows, self.dim), (self.pitch, 1), self.lead)

    def forward(self, branch=True):
        o, c = self.oracle, self
        c.out, c.h, c.stats = c.empty(c.xk), c.empty(c.k) if o.before != "none" else None, c.d.empty((c.rows, 4))
        L.block_norms(c.norms, c.x, c.y if branch else None, c.out, c.h, c.stats)
        want, tol = o.out(c.xv, c.yv if branch else None)
        c.ov = values(c.out, c.xk)
        close(c.ov, want, B.stored_tol(want, tol, c.xk), "out")
        if c.h is not None:
            want, tol = o.h(c.ov)  # of what is stored
            close(values(c.h, c.k), want, B.stored_tol(want, tol, c.k), "h")
        c.sv = c.stats.numpy()
        for at, (rows, kind) in enumerate(((c.yv if branch else None, o.after if branch else "none"), (c.ov, o.before))):
            if rows is None:
                assert np.array_equal(c.sv[:, :2], np.tile([0.0, 1.0], (c.rows, 1)))
                continue
            mean, rstd, t_mean, t_rstd = B.statistics(rows, kind, o.eps)
            close(c.sv[:, 2 * at], mean[:, 0], t_mean[:, 0], "mean")
            close(c.sv[:, 2 * at + 1], rstd[:, 0], t_rstd[:, 0], "1 / deviation")

    def backward(self, rng, branch=True, carried=True, second=True):
        o, c = self.oracle, self
        go, gov = c.rows_of(rng.standard_normal((c.rows, c.dim)), c.xk) if carried else (None, None)
        gh, ghv = c.rows_of(rng.standard_normal((c.rows, c.dim)), c.k) if second and o.before != "none" else (None, None)
        want = o.grad(c.ov, c.yv if branch else None, c.sv, gov, ghv)
        got = {"dx": c.empty(c.xk)}
        if branch:
            got["dy"] = c.empty(c.k)
        for name, there in (("dafter_weight", branch and o.after != "none"), ("dafter_bias", branch and o.after != "none"), ("dbefore_weight", o.before != "none"),
                            ("dbefore_bias", o.before != "none"), ("dgate", branch and o.gate is not None)):
            if there:
                got[name] = c.d.empty(c.host["gate"].shape if name == "dgate" else (c.dim,))
        L.block_norms_grad(c.norms, c.out, c.y if branch else None, c.stats, go, gh, **got)
        for name, t in got.items():
            value, tol = want.get(name, (np.zeros(c.dim), np.zeros(c.dim)))
            kind = {"dx": c.xk, "dy": c.k}.get(name, "f32")
            close(values(t, kind), value, B.stored_tol(value, tol, kind), name)
        return got, go, gh


@pytest.mark.parametrize("xk,k", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("rows,dim,pitch,lead", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 8, 8, 0), (6, 24, 0, 0), (37, 257, 3, 1), (8, 264, 0, 0), (130, 768, 0, 0), (9, 1000, 0, 0), (4, 2056, 8, 8),
                                                (3, 4096, 0, 0), (5, 4104, 0, 0), (2, 5001, 0, 1), (3, 8192, 0, 0), (2, 8200, 0, 0), (2, 16384, 0, 0)])
def test_block_norms_sizes_and_layouts(ctx, xk, k, rows, dim, pitch, lead):
    rng = np.random.default_rng(dim * 7 + rows)
    with Held(ctx) as d:
        c = Case(d, rng, rows, dim, xk, k, "rms" if dim % 3 else "layer", "layer" if dim % 3 else "rms", gate=1, scale=0.75, p=0.25, pitch=pitch, lead=lead)
        c.forward()
        c.backward(rng)


@pytest.mark.parametrize("after", ["none", "rms", "layer"])
@pytest.mark.parametrize("before", ["none", "rms", "layer"])
@pytest.mark.parametrize("gate,p,affine", [(0, 0.0, True), (1, 0.5, True), (6, 0.1, False), (42, 0.0, True)])
def test_block_norms_kinds(ctx, after, before, gate, p, affine):
    rng = np.random.default_rng(gate + len(after) * 10 + len(before))
    with Held(ctx) as d:
        c = Case(d, rng, 42, 136, "f32", "bf16", after, before, gate=gate, p=p, affine=affine)
        c.forward()
        c.backward(rng)
        c.backward(rng, carried=False) if before != "none" else None
        c.backward(rng, second=False)


@pytest.mark.parametrize("rows,dim,gate", [(5000, 40, 8), (3001, 768, 1), (2048, 264, 2048), (1500, 2056, 3), (900, 4104, 2)])
def test_block_norms_many_rows(ctx, rows, dim, gate):
    rng = np.random.default_rng(rows)
    with Held(ctx) as d:
        c = Case(d, rng, rows, dim, "bf16", "bf16", "rms", "layer", gate=gate, p=0.1)
        c.forward()
        first, go, gh = c.backward(rng)
        again = {n: d.empty(t.extents, t.dtype) for n, t in first.items() if n not in ("dx", "dy")}
        L.block_norms_grad(c.norms, c.out, c.y, c.stats, go, gh, **again)
        for n, t in again.items():  # sums over rows in a fixed order
            assert np.array_equal(t.numpy(), first[n].numpy()), n


@pytest.mark.parametrize("rows,dim,gate", [(9000, 136, 9000), (6000, 1160, 3000), (5000, 1032, 1), (1200, 2056, 600)])
@pytest.mark.parametrize("after,before", [("layer", "rms"), ("rms", "rms"), ("none", "layer")])
def test_block_norms_gates_of_one_group_and_of_many(ctx, rows, dim, gate, after, before):
    """Gates whose row serves all of a team's rows, and gates that change on the way; and each sum when it is asked for alone."""
    rng = np.random.default_rng(rows + dim)
    with Held(ctx) as d:
        c = Case(d, rng, rows, dim, "bf16", "bf16", after, before, gate=gate, p=0.1)
        c.forward()
        all_of, go, gh = c.backward(rng)
        want = c.oracle.grad(c.ov, c.yv, c.sv, values(go, "bf16"), values(gh, "bf16"))
        for name in [n for n in all_of if n not in ("dx", "dy") and n in want]:
            alone = d.empty(all_of[name].extents)
            L.block_norms_grad(c.norms, c.out, c.y, c.stats, go, gh, **{name: alone})
            value, tol = want[name]
            close(alone.numpy(), value, B.stored_tol(value, tol, "f32"), name)


def test_block_norms_without_a_branch(ctx):
    rng = np.random.default_rng(5)
    with Held(ctx) as d:
        c = Case(d, rng, 11, 72, "bf16", "bf16", "none", "layer", scale=0.5)
        c.forward(branch=False)
        c.backward(rng, branch=False)
        c.backward(rng, branch=False, carried=False)
        c = Case(d, rng, 11, 72, "f32", "f16", "none", "rms")
        c.forward(branch=False)
        h = c.empty("f16")
        L.block_norms(c.norms, c.x, None, None, h)  # nothing but the norm
        assert np.array_equal(h.numpy(), c.h.numpy())


def test_block_norms_in_place(ctx):
    rng = np.random.default_rng(6)
    for dim in (256, 257):
        with Held(ctx) as d:
            c = Case(d, rng, 50, dim, "bf16", "bf16", "layer", "rms", gate=1, p=0.2)
            c.forward()
            L.block_norms(c.norms, c.x, c.y, c.x, c.y)
            assert np.array_equal(c.x.numpy(), c.out.numpy()) and np.array_equal(c.y.numpy(), c.h.numpy())


@pytest.mark.parametrize("dim", [64, 769])
def test_block_norms_of_no_rows_and_strange_rows(ctx, dim):
    rng = np.random.default_rng(7)
    with Held(ctx) as d:
        c = Case(d, rng, 0, dim, "f32", "f32", "layer", "layer", gate=1)
        c.forward()
        got, _, _ = c.backward(rng)
        assert all((t.numpy() == 0).all() for n, t in got.items() if n not in ("dx", "dy"))
        c = Case(d, rng, 6, dim, "f32", "f32", "layer", "layer")
        rows = np.stack([np.zeros(dim), np.full(dim, 3e4), 1e6 + 0.01 * rng.standard_normal(dim), 1e-20 * rng.standard_normal(dim), np.full(dim, np.nan), rng.standard_normal(dim)])
        (c.x, c.xv), (c.y, c.yv) = c.rows_of(0 * rows, "f32"), c.rows_of(rows, "f32")
        out, h, st = c.empty("f32"), c.empty("f32"), d.empty((6, 4))
        L.block_norms(c.norms, c.x, c.y, out, h, st)
        want, tol = c.oracle.out(c.xv, c.yv)
        fine = [0, 2, 3, 5]
        close(out.numpy()[fine], want[fine], tol[fine] + 1e-30)
        # (a row of one value: its mean in 32 bits is off by 53 U of it at most, which a deviation of the root of eps makes as large as this)
        assert np.all(np.abs(out.numpy()[1] - c.host["ab"]) <= np.abs(c.host["aw"]) * 53 * O.U * 3e4 / np.sqrt(1e-5) + 1e-6)
        assert np.isnan(out.numpy()[4]).all() and np.isnan(h.numpy()[4]).all() and not np.isnan(h.numpy()[5]).any()


# ------------------------------------------------------------------------------------------ captured
def test_a_captured_run_follows_its_operands():
    """Dropout, both directions of the norms and of the head, captured once and replayed on new contents: the same bits as calls, and masks by the seed of the moment."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s, t=torch.bfloat16: torch.randn(s, generator=g, device="cuda").to(t)  # noqa: E731
    rows, dim, vocab = 300, 264, 1000
    t = {"x": n(rows, dim), "y": n(rows, dim), "w": n(dim, t=torch.float32), "gate": n(4, dim, t=torch.float32), "table": n(vocab, dim), "gl": n(rows, t=torch.float32)}
    t["seed"] = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    t["ids"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    e = lambda *s, d=torch.bfloat16: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
    f32 = torch.float32
    r = {"drop": e(rows, dim), "out": e(rows, dim), "h": e(rows, dim), "stats": e(rows, 4, d=f32), "logp": e(rows, d=f32), "ent": e(rows, d=f32), "st": e(rows, 2, d=f32), "dh": e(rows, dim),
         "dtable": e(vocab, dim), "dx": e(rows, dim), "dy": e(rows, dim), "dw": e(dim, d=f32), "dgate": e(4, dim, d=f32)}
    ctx, stream = S.Context(0), torch.cuda.Stream()
    ctx.use_stream(stream.cuda_stream)
    b = {k: ctx.borrow(v) for k, v in {**t, **r}.items()}
    norms = L.BlockNorms(ctx, after="rms", before="rms", before_weight=b["w"], gate=b["gate"], p=0.2, seed=b["seed"], site=4)

    def step():
        L.dropout(b["x"], b["drop"], b["seed"], 0.1, site=1)
        L.block_norms(norms, b["drop"], b["y"], b["out"], b["h"], b["stats"])
        L.head_log_probs(b["h"], b["table"], b["ids"], b["logp"], b["ent"], b["st"])
        L.head_log_probs_grad(b["h"], b["table"], b["ids"], b["st"], b["ent"], b["gl"], b["gl"], b["dh"], b["dtable"])
        L.block_norms_grad(norms, b["out"], b["y"], b["stats"], None, b["dh"], b["dx"], b["dy"], dgate=b["dgate"], dbefore_weight=b["dw"])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()  # the pool's memory is there before anything is captured
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for seed in ((5, 6), (-1, 9)):
        with torch.cuda.stream(stream):
            t["seed"].copy_(torch.tensor(seed, dtype=torch.int32))
            t["y"].mul_(1.5)
            step()
            stream.synchronize()
            want = {k: v.clone() for k, v in r.items()}
            for v in r.values():
                v.zero_()
            graph.replay()
            stream.synchronize()
        for k, v in r.items():
            assert torch.equal(v, want[k]), k
        kept = torch.from_numpy(B.keep(np.array(seed, np.int32).astype(np.uint32), 1, rows * dim, 0.1).reshape(rows, dim)).cuda()
        assert torch.equal(r["drop"] != 0, kept & (t["x"] != 0))
    del graph
    assert ctx.status_word() == 0
    ctx.close()
