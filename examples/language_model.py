"""A small language model trained and asked: the embedding with its gradient, the log probabilities of the next tokens with an entropy
bonus, and AdamW with 8-bit states, as one lazy graph; then single contexts with their likeliest continuations.

    python examples/language_model.py [--steps 60] [--tokens 2000] [--width 64]

The data is a made-up language: a sentence steps through the vocabulary by one of three strides that its first token names.
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sage_b200 as S  # noqa: E402

CONTEXT = 3


class Model:
    """Three tokens -> the next: embeddings side by side, two dense layers, and the embedding table again as the last product."""

    def __init__(self, ctx, tokens, width, rng):
        def param(*extents, std):
            v = S.Var.empty(extents)
            ctx.set(v, (rng.standard_normal(extents) * std).astype(np.float32))
            return v
        self.width = width
        self.table = param(tokens, width, std=1.0 / width)  # scaled by the root of the width where it is looked up
        self.w1, self.b1 = param(CONTEXT * width, 4 * width, std=(CONTEXT * width) ** -0.5), param(4 * width, std=0.0)
        self.w2, self.b2 = param(4 * width, width, std=(4 * width) ** -0.5), param(width, std=0.0)

    def params(self):
        return [self.table, self.w1, self.b1, self.w2, self.b2]

    def logits(self, ids):  # [rows, CONTEXT]
        x = S.embedding(self.table, ids, scale=self.width ** 0.5)
        x = x.view([ids.extents[0], CONTEXT * self.width])
        x = S.relu(x.matmul(self.w1) + self.b1)
        return (x.matmul(self.w2) + self.b2).matmul(self.table.tr())


def sentences(rng, rows, tokens):
    first = rng.integers(0, tokens, rows)
    stride = np.array([1, 7, 31])[first % 3]
    return ((first[:, None] + stride[:, None] * np.arange(CONTEXT + 1)) % tokens).astype(np.uint32)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=2000)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--batch", type=int, default=1024)
    ap.add_argument("--device", type=int, default=0)
    a = ap.parse_args(argv)
    rng, ctx = np.random.default_rng(0), S.Context(a.device)
    model = Model(ctx, a.tokens, a.width, rng)
    ids, after = ctx.var(np.zeros((a.batch, CONTEXT), np.uint32)), ctx.var(np.zeros(a.batch, np.uint32))
    log_probs, entropy = S.token_log_probs(model.logits(ids), after)
    loss = -(log_probs.mean([0]) + entropy.mean([0]) * 0.01)
    grads = dict(zip(model.params(), S.grad(loss, model.params())))
    opt = S.AdamW(3e-3, state_bits=8)
    opt.init(ctx)
    losses = []
    for step in range(a.steps):
        s = sentences(rng, a.batch, a.tokens)
        ctx.set(ids, s[:, :CONTEXT])
        ctx.set(after, np.ascontiguousarray(s[:, CONTEXT]))
        ctx.clear()
        ctx.eval(loss, *grads.values())
        losses.append(float(ctx.read(loss)[0]))
        opt.update(grads, ctx)
        if step % 10 == 0 or step == a.steps - 1:
            print("step %3d  loss %.4f" % (step, losses[-1]))

    # one context at a time: the log probability of what follows, and the five likeliest tokens
    one, following = ctx.var(np.zeros((1, CONTEXT), np.uint32)), ctx.var(np.zeros(1, np.uint32))
    logits = model.logits(one)
    lp, h = S.token_log_probs(logits, following)
    top = S.top_tokens(logits, 5)
    found = []
    for s in sentences(rng, 5, a.tokens):
        ctx.set(one, s[None, :CONTEXT])
        ctx.set(following, s[CONTEXT:])
        ctx.clear()
        ctx.eval(lp, h, top)
        tops = ctx.read(top)[0]
        found.append(int(s[CONTEXT]) in tops)
        print("%s -> %d: log probability %.3f, entropy %.3f, likeliest %s" % (s[:CONTEXT], s[CONTEXT], ctx.read(lp)[0], ctx.read(h)[0], tops))
    ctx.close()
    return losses, found


if __name__ == "__main__":
    main()
