"""Captured language-model calls on a B200 beside other users of the context's pool: what a graph works in is its own until it is gone."""
import time

import numpy as np
import pytest

import sage_b200 as S
from sage_b200 import language as L

pytestmark = pytest.mark.gpu
ROWS, DIM, VOCAB = 300, 264, 1000
SIZES = [512, 40_000, 300_000, 700_000, 1 << 20, 3 << 20, 9 << 20, 24 << 20]  # bytes: one of each way the pool finds a block


class Step:
    """The operators that need memory of the pool, on buffers of another runtime."""

    def __init__(self, ctx, seed):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s, t=torch.bfloat16: torch.randn(s, generator=g, device="cuda").to(t)  # noqa: E731
        e = lambda *s, t=torch.bfloat16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        f32 = torch.float32
        operands = {"x": n(ROWS, DIM), "y": n(ROWS, DIM), "w": n(DIM, t=f32), "gate": n(4, DIM, t=f32), "table": n(VOCAB, DIM), "gl": n(ROWS, t=f32), "logits": n(ROWS, VOCAB),
                    "xf": n(ROWS, DIM, t=f32), "tf": n(VOCAB, DIM, t=f32), "ids": torch.randint(0, VOCAB, (ROWS,), generator=g, device="cuda", dtype=torch.int32)}
        self.results = {"out": e(ROWS, DIM), "h": e(ROWS, DIM), "stats": e(ROWS, 4, t=f32), "logp": e(ROWS, t=f32), "ent": e(ROWS, t=f32), "st": e(ROWS, 2, t=f32), "dh": e(ROWS, DIM),
                        "dtable": e(VOCAB, DIM), "dx": e(ROWS, DIM), "dy": e(ROWS, DIM), "dw": e(DIM, t=f32), "dgate": e(4, DIM, t=f32), "demb": e(VOCAB, DIM, t=f32),
                        "logp2": e(ROWS, t=f32), "ent2": e(ROWS, t=f32), "st2": e(ROWS, 2, t=f32), "dlogits": e(ROWS, VOCAB),
                        "logpf": e(ROWS, t=f32), "entf": e(ROWS, t=f32), "stf": e(ROWS, 2, t=f32), "dhf": e(ROWS, DIM, t=f32), "dtf": e(VOCAB, DIM, t=f32)}
        self.b = {k: ctx.borrow(v) for k, v in {**operands, **self.results}.items()}
        self.norms = L.BlockNorms(ctx, after="rms", before="rms", before_weight=self.b["w"], gate=self.b["gate"])

    def __call__(self):
        b = self.b
        L.block_norms(self.norms, b["x"], b["y"], b["out"], b["h"], b["stats"])
        L.head_log_probs(b["h"], b["table"], b["ids"], b["logp"], b["ent"], b["st"])
        L.head_log_probs_grad(b["h"], b["table"], b["ids"], b["st"], b["ent"], b["gl"], b["gl"], b["dh"], b["dtable"])
        L.block_norms_grad(self.norms, b["out"], b["y"], b["stats"], None, b["dh"], b["dx"], b["dy"], dgate=b["dgate"], dbefore_weight=b["dw"])
        L.embedding_grad(b["dx"], b["ids"], b["demb"])
        L.token_log_probs(b["logits"], b["ids"], b["logp2"], b["ent2"], b["st2"])
        L.token_log_probs_grad(b["logits"], b["ids"], b["st2"], b["ent2"], b["gl"], b["gl"], b["dlogits"])
        L.head_log_probs(b["xf"], b["tf"], b["ids"], b["logpf"], b["entf"], b["stf"])
        L.head_log_probs_grad(b["xf"], b["tf"], b["ids"], b["stf"], b["entf"], b["gl"], b["gl"], b["dhf"], b["dtf"])

    def called(self, stream):
        """What calls give, and the results cleared behind that."""
        import torch
        with torch.cuda.stream(stream):
            self()
            stream.synchronize()
            want = {k: v.clone() for k, v in self.results.items()}
            for v in self.results.values():
                v.zero_()
        stream.synchronize()
        return want


def captured(step, stream):
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    return graph


def same(step, want):
    import torch
    for k, v in step.results.items():
        assert torch.equal(v, want[k]), k


def pattern(ctx):
    host = [np.arange(n // 4, dtype=np.float32) + n for n in SIZES]
    return [(ctx.tensor(h), h) for h in host]


@pytest.mark.parametrize("warm", [True, False])
def test_replays_leave_other_tensors_of_the_pool_alone(warm):
    """Tensors of every size made behind a capture, and calls with scratch of their own between replays; with and without memory in the pool before it."""
    import torch
    first = S.Context(0)  # (the kernels have run once in this process)
    stream = torch.cuda.Stream()
    first.use_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    want = Step(first, 1).called(stream)
    ctx = S.Context(0)
    ctx.use_stream(stream.cuda_stream)
    step, other = Step(ctx, 1), Step(ctx, 2)
    torch.cuda.synchronize()
    if warm:
        step.called(stream)
    graph = captured(step, stream)
    held = ctx.mem_stats()["mem_used"]
    assert held > 0
    ctx._ck(S.lib.sage_release_cached(ctx.h))
    mine = pattern(ctx)
    other_want = other.called(stream)
    for _ in range(3):
        with torch.cuda.stream(stream):
            for v in step.results.values():
                v.zero_()
            graph.replay()
            other()
            graph.replay()
        stream.synchronize()
        same(step, want)
        same(other, other_want)
        for t, h in mine:
            assert np.array_equal(t.numpy(), h), h.nbytes
    for t, _ in mine:
        t.release()
    del graph
    torch.cuda.synchronize()
    for _ in range(100):  # the driver says so from a thread of its own
        if ctx.mem_stats()["mem_used"] == 0:
            break
        time.sleep(0.05)
    assert ctx.mem_stats()["mem_used"] == 0
    for c in (ctx, first):
        assert c.status_word() == 0
        c.close()


def test_two_graphs_of_a_context_run_side_by_side():
    """Each has memory of its own, so they may be replayed on streams of their own at the same time."""
    import torch
    ctx, stream = S.Context(0), torch.cuda.Stream()
    ctx.use_stream(stream.cuda_stream)
    steps = [Step(ctx, 3), Step(ctx, 4)]
    torch.cuda.synchronize()
    want = [s.called(stream) for s in steps]
    graphs = [captured(s, stream) for s in steps]
    stream.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        same(s, w)
    del graphs, g
    assert ctx.status_word() == 0
    ctx.close()
