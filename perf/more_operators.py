"""Operators between the embedding and the update of a language model's training step, as cases that can be timed and compared:
dropout whose mask is drawn from a counter and never stored, the norms before and after a block with its gate and residual scale,
and the log probabilities of given tokens straight from hidden states, in pieces of the vocabulary; each with its gradient.

  listed()            the cases
  draw(rng)           one more case of the same ranges
  prepare(case, seed) inputs, buffers and handles of a program that is about to run the case, on the GPU
  run(state)          one pass: in plain torch operations, or (`own`) through the package's entry points
  work(case)          the bytes and operations one pass cannot do without
  exact(case, seed)   what run() returns, computed in 64 bits from the operator's definition
"""
import math

import numpy as np
import torch

own = False

F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # The embeddings of a few short sequences while a model is tuned: latency.
        {"name": "dropout_24x768_f32", "kind": "dropout", "rows": 24, "cols": 768, "type": "f32", "p": 0.1, "site": 0},
        # A half-precision batch of hidden states, and as much again as its gradient: the same call.
        {"name": "dropout_16384x4096_bf16", "kind": "dropout", "rows": 16384, "cols": 4096, "type": "bf16", "p": 0.1, "site": 7},
        # One token being generated, norms on both sides of the block and a gate for each channel.
        {"name": "norms_1x4096_bf16", "kind": "norms", "rows": 1, "dim": 4096, "x": "bf16", "type": "bf16", "after": "rms", "before": "rms", "gate": 1, "scale": 1.0, "p": 0.0},
        # The base encoder's training batch (32 x 128 tokens): dropout, residual, layer norm.
        {"name": "norms_4096x768_f32", "kind": "norms", "rows": 4096, "dim": 768, "x": "f32", "type": "f32", "after": "none", "before": "layer", "gate": 0, "scale": 1.0, "p": 0.1},
        # A long prompt batch: half-precision blocks around a residual stream that is kept in 32 bits, its branches scaled by channel.
        {"name": "norms_16384x4096_bf16", "kind": "norms", "rows": 16384, "dim": 4096, "x": "f32", "type": "bf16", "after": "rms", "before": "rms", "gate": 1, "scale": 1.0, "p": 0.0},
        # The gradient of the base encoder's.
        {"name": "norms_grad_4096x768_f32", "kind": "norms_grad", "rows": 4096, "dim": 768, "x": "f32", "type": "f32", "after": "none", "before": "layer", "gate": 0, "scale": 1.0, "p": 0.1},
        # The gradient with everything: norms on both sides, gates that a condition gives each of eight sequences, dropout, a residual scale; odd rows.
        {"name": "norms_grad_16376x2056_bf16", "kind": "norms_grad", "rows": 16376, "dim": 2056, "x": "bf16", "type": "bf16", "after": "rms", "before": "layer", "gate": 8, "scale": 0.7, "p": 0.1},
        # The log probability of the token just generated, for one sequence.
        {"name": "head_1x131072x4096_bf16", "kind": "head", "rows": 1, "vocab": 131072, "dim": 4096, "type": "bf16", "scale": 1.0},
        # Scoring a corpus, an odd vocabulary, at a temperature.
        {"name": "head_8192x50021x2048_bf16", "kind": "head", "rows": 8192, "vocab": 50021, "dim": 2048, "type": "bf16", "scale": 1.25},
        # The masked tokens of the base encoder's batch, 32 bits throughout: values and gradients.
        {"name": "head_grad_640x30522x768_f32", "kind": "head_grad", "rows": 640, "vocab": 30522, "dim": 768, "type": "f32", "scale": 1.0},
        # A small batch of a narrow model in half precision, odd sizes.
        {"name": "head_grad_509x10007x264_f16", "kind": "head_grad", "rows": 509, "vocab": 10007, "dim": 264, "type": "f16", "scale": 1.0},
        # A large model's training batch: a weighted likelihood with an entropy bonus.
        {"name": "head_grad_8192x131072x4096_bf16", "kind": "head_grad", "rows": 8192, "vocab": 131072, "dim": 4096, "type": "bf16", "scale": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["dropout", "dropout", "norms", "norms", "norms_grad", "norms_grad", "head", "head_grad", "head_grad"])
    cost = lambda c: work(c)["bytes"] / 6.5 + work(c)["flops"] / (200 if c.get("type") != "f32" else 30)  # noqa: E731
    most = max(cost(c) for c in listed() if c["kind"] == kind)
    while True:
        t = rng.choice(["f32", "bf16", "f16"])
        if kind == "dropout":
            c = {"kind": kind, "rows": _log_int(rng, 1, 32768), "cols": _log_int(rng, 8, 8192), "type": t, "p": rng.choice([0.05, 0.1, 0.5]), "site": rng.randint(0, 1 << 40)}
            width = "cols"
        elif kind in ("norms", "norms_grad"):
            c = {"kind": kind, "rows": _log_int(rng, 1, 32768), "dim": _log_int(rng, 16, 8192), "x": rng.choice(["f32", t]), "type": t, "after": rng.choice(["none", "rms", "layer"]),
                 "before": rng.choice(["rms", "layer", "layer", "none"]), "gate": rng.choice([0, 1, 1, 4]), "scale": rng.choice([1.0, 0.5]), "p": rng.choice([0.0, 0.1])}
            if c["gate"] > 1:
                c["rows"] = (c["rows"] + 3) // 4 * 4
            width = "dim"
        else:
            c = {"kind": kind, "rows": _log_int(rng, 1, 16384), "vocab": _log_int(rng, 100, 131072), "dim": _log_int(rng, 32, 4096), "type": t, "scale": rng.choice([1.0, 1.0, 0.8])}
            width = "dim"
        if rng.random() < 0.6:  # widths are round more often than not
            c[width] = (c[width] + 63) // 64 * 64
        if cost(c) <= most:
            return c


# ------------------------------------------------------------------------------------------ inputs
def _tokens(g, n, vocab, none):
    """Token numbers whose frequencies fall with their number as words' do; a share `none` of them is not scored."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().clamp(0, vocab - 1).to(torch.int32)
    if none:
        ids[torch.rand(n, generator=g, device="cuda") < none] = -1
    return ids


def prepare(case, seed):
    g, kind, dev = torch.Generator(device="cuda").manual_seed(seed), case["kind"], {"device": "cuda"}
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case, "kind": kind, "handles": None}
    s["seed"] = torch.randint(-2 ** 31, 2 ** 31, (2,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if kind == "dropout":
        s["x"] = normal(case["rows"], case["cols"]).to(F[case["type"]])
        s["y"] = torch.empty_like(s["x"])
    elif kind in ("norms", "norms_grad"):
        r, d, tx, t = case["rows"], case["dim"], F[case["x"]], F[case["type"]]
        loud = torch.exp(0.5 * normal(d))  # some channels are louder than others
        s["y"] = (normal(r, d) * loud * 0.5).to(t)
        for name in ("after", "before"):
            if case[name] != "none":
                s[name + "_weight"] = 1.0 + 0.1 * normal(d)
            if case[name] == "layer":
                s[name + "_bias"] = 0.1 * normal(d)
        if case["gate"]:
            s["gate"] = 0.5 + 0.3 * normal(*((d,) if case["gate"] == 1 else (case["gate"], d)))
        stream = normal(r, d) * loud + 0.3
        if kind == "norms":
            s["x"] = stream.to(tx)
            s["out"], s["h"] = torch.empty((r, d), dtype=tx, **dev), torch.empty((r, d), dtype=t, **dev) if case["before"] != "none" else None
        else:  # what the forward pass kept: the stream behind the block and both norms' statistics; and the gradients that arrive
            s["out"] = stream.to(tx)
            s["stats"] = torch.stack(_statistics(s["y"].float(), case["after"]) + _statistics(s["out"].float(), case["before"]), 1)
            s["g_out"] = (normal(r, d) * 1e-2).to(tx)
            s["g_h"] = (normal(r, d) * 1e-2).to(t) if case["before"] != "none" else None
            s["dx"], s["dy"] = torch.empty((r, d), dtype=tx, **dev), torch.empty((r, d), dtype=t, **dev)
            for name in ("gate", "after_weight", "after_bias", "before_weight", "before_bias"):
                if name in s:
                    s["d" + name] = torch.empty_like(s[name])
    else:
        r, v, d, t = case["rows"], case["vocab"], case["dim"], F[case["type"]]
        w = normal(v, d) / math.sqrt(d)
        s["ids"] = _tokens(g, r, v, 0.1 if r > 1 else 0.0)
        # a trained model's states lean towards their tokens' rows
        s["hidden"] = (2.0 * normal(r, d) + 8.0 * w[s["ids"].clamp(0, v - 1).long()]).to(t)
        s["weight"] = w.to(t)
        s["logp"], s["entropy"] = torch.empty(r, **dev), torch.empty(r, **dev)
        if kind == "head_grad":
            s["gl"] = -torch.rand(r, generator=g, device="cuda") / r
            s["ge"] = -torch.rand(r, generator=g, device="cuda") * (0.01 / r)
            s["stats"] = torch.empty((r, 2), **dev)
            s["dhidden"], s["dweight"] = torch.empty((r, d), dtype=t, **dev), torch.empty((v, d), dtype=t, **dev)
    return s


EPS = 1e-5


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


_context = None


def _program():
    """The context of the process, on the stream that torch works on."""
    global _context
    if _context is None:
        import sage_b200 as S
        _context = S.Context(0)
        _context.use_stream(torch.cuda.current_stream().cuda_stream)
    return _context


def _run_own(s):
    from sage_b200 import language as L
    ctx, kind, case, h = _program(), s["kind"], s["case"], s["handles"]
    if h is None:  # handles of the program's buffers: addresses, shapes and types
        h = {k: ctx.borrow(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        if kind in ("norms", "norms_grad"):
            h["norms"] = L.BlockNorms(ctx, after=case["after"], after_weight=h.get("after_weight"), after_bias=h.get("after_bias"), before=case["before"],
                                      before_weight=h.get("before_weight"), before_bias=h.get("before_bias"), gate=h.get("gate"), residual_scale=case["scale"],
                                      eps=EPS, p=case["p"], seed=h["seed"], site=3)
        s["handles"] = h
    if kind == "dropout":
        L.dropout(h["x"], h["y"], h["seed"], case["p"], site=case["site"])
        return s["y"]
    if kind == "norms":
        L.block_norms(h["norms"], h["x"], h["y"], h["out"], h.get("h"))
        return {k: s[k] for k in ("out", "h") if s[k] is not None}
    if kind == "norms_grad":
        L.block_norms_grad(h["norms"], h["out"], h["y"], h["stats"], h["g_out"], h.get("g_h"), h["dx"], h["dy"], dgate=h.get("dgate"), dafter_weight=h.get("dafter_weight"),
                           dafter_bias=h.get("dafter_bias"), dbefore_weight=h.get("dbefore_weight"), dbefore_bias=h.get("dbefore_bias"))
        return {k: s[k] for k in NORMS_GRADS if k in s}
    if kind == "head":
        L.head_log_probs(h["hidden"], h["weight"], h["ids"], h["logp"], h["entropy"], scale=case["scale"])
        return s["logp"], s["entropy"]
    L.head_log_probs(h["hidden"], h["weight"], h["ids"], h["logp"], h["entropy"], stats=h["stats"], scale=case["scale"])
    L.head_log_probs_grad(h["hidden"], h["weight"], h["ids"], h["stats"], h["entropy"], h["gl"], h["ge"], h["dhidden"], h["dweight"], scale=case["scale"])
    return s["logp"], s["entropy"], s["dhidden"], s["dweight"]


NORMS_GRADS = ("dx", "dy", "dgate", "dafter_weight", "dafter_bias", "dbefore_weight", "dbefore_bias")
LOW = 0xFFFFFFFF


def _keep(seed, site, shape, p):
    """Which elements stay, and the factor on them.  Sixteen bits an element out of Philox4x32-10: element i takes half i % 2 of word
    i // 2 % 4 of the block whose counter is (i // 8, site), keyed by the seed; it is dropped where they are below 65536 p."""
    n = math.prod(shape)
    block = torch.arange((n + 7) // 8, device="cuda")
    a, b = block & LOW, block >> 32
    c, d = torch.full_like(block, site & LOW), torch.full_like(block, site >> 32)
    key = seed.long() & LOW
    for step in range(10):
        p0, p1 = a * 0xD2511F53, c * 0xCD9E8D57
        k0, k1 = (key[0] + step * 0x9E3779B9) & LOW, (key[1] + step * 0xBB67AE85) & LOW
        a, b, c, d = ((p1 >> 32) & LOW) ^ b ^ k0, p1 & LOW, ((p0 >> 32) & LOW) ^ d ^ k1, p0 & LOW
    words = torch.stack((a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16, c & 0xFFFF, c >> 16, d & 0xFFFF, d >> 16), 1)
    drop = min(65535, round(p * 65536))
    return (words.reshape(-1)[:n] >= drop).reshape(shape), 65536.0 / (65536 - drop)


def _dropped(x, s, site, p):
    if not p:
        return x
    keep, factor = _keep(s["seed"], site, x.shape, p)
    return torch.where(keep, x * factor, 0.0)


def _statistics(x, kind):
    """Mean and reciprocal deviation of the rows, as the norm takes them."""
    mean = x.mean(1) if kind == "layer" else torch.zeros_like(x[:, 0])
    return (mean, torch.rsqrt(torch.square(x - mean[:, None]).mean(1) + EPS)) if kind != "none" else (mean, torch.ones_like(mean))


def _unit(x, kind):
    mean, rstd = _statistics(x, kind)
    return (x - mean[:, None]) * rstd[:, None], rstd[:, None]


def _affine(u, s, name):
    y = u * s[name + "_weight"] if name + "_weight" in s else u
    return y + s[name + "_bias"] if name + "_bias" in s else y


def _through(g, u, rstd, kind):
    """The gradient in front of a norm, from that of its unit rows."""
    if kind == "none":
        return g
    d = g - u * (g * u).mean(1, keepdim=True)
    return rstd * (d - g.mean(1, keepdim=True) if kind == "layer" else d)


def _gates(s, rows):
    if "gate" not in s:
        return 1.0
    return s["gate"] if s["gate"].dim() == 1 else s["gate"].repeat_interleave(rows // s["gate"].shape[0], 0)


def _run_plain(s):
    kind, case = s["kind"], s["case"]
    if kind == "dropout":
        return _dropped(s["x"].float(), s, case["site"], case["p"]).to(s["x"].dtype)
    if kind == "norms":
        branch = _dropped(_affine(_unit(s["y"].float(), case["after"])[0], s, "after"), s, 3, case["p"])
        out = s["x"].float() * case["scale"] + _gates(s, case["rows"]) * branch
        found = {"out": out.to(s["out"].dtype)}
        if case["before"] != "none":
            found["h"] = _affine(_unit(out, case["before"])[0], s, "before").to(s["h"].dtype)
        return found
    if kind == "norms_grad":
        r, found = case["rows"], {}
        g = s["g_out"].float()
        if case["before"] != "none":
            u, rstd = _unit(s["out"].float(), case["before"])
            gh = s["g_h"].float()
            g = g + _through(gh * s["before_weight"], u, rstd, case["before"])
            found["dbefore_weight"] = (gh * u).sum(0)
            if "before_bias" in s:
                found["dbefore_bias"] = gh.sum(0)
        u, rstd = _unit(s["y"].float(), case["after"])
        found["dx"] = (g * case["scale"]).to(s["dx"].dtype)
        if "gate" in s:
            by = g * _dropped(_affine(u, s, "after"), s, 3, case["p"])
            found["dgate"] = by.sum(0) if s["gate"].dim() == 1 else by.reshape(case["gate"], r // case["gate"], -1).sum(1)
        gn = _dropped(g * _gates(s, r), s, 3, case["p"])
        if "after_weight" in s:
            found["dafter_weight"] = (gn * u).sum(0)
        if "after_bias" in s:
            found["dafter_bias"] = gn.sum(0)
        found["dy"] = _through(gn * s["after_weight"] if "after_weight" in s else gn, u, rstd, case["after"]).to(s["dy"].dtype)
        return {k: found[k] for k in NORMS_GRADS if k in found}
    hidden, weight, v = s["hidden"].float(), s["weight"].float(), case["vocab"]
    x = (hidden @ weight.T) * case["scale"]
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    there = (s["ids"] >= 0) & (s["ids"] < v)
    at = s["ids"].clamp(0, v - 1).long()[:, None]
    logp = torch.where(there, (d.gather(1, at) - log_z)[:, 0], 0.0)
    p = e / z
    entropy = log_z - (p * d).sum(1, keepdim=True)
    if kind == "head":
        return logp, entropy[:, 0]
    gl, ge = torch.where(there, s["gl"], 0.0)[:, None], s["ge"][:, None]
    dx = p * (-gl - ge * (d - log_z + entropy))
    dx = dx.scatter_add_(1, at, gl) * case["scale"]
    return logp, entropy[:, 0], (dx @ weight).to(s["hidden"].dtype), (dx.T @ hidden).to(s["weight"].dtype)


# ------------------------------------------------------------------------------------------ in 64 bits
def _factors(s, site, shape, p):
    """What dropout multiplies each element by, on the host with numpy's unsigned numbers."""
    if not p:
        return 1.0
    n, u = math.prod(shape), np.uint64
    key = s["seed"].cpu().numpy().astype(np.uint32).astype(u)
    count = np.arange((n + 7) // 8, dtype=u)
    low, half = u(LOW), u(32)
    x = [count & low, count >> half, np.full_like(count, site % 2 ** 32), np.full_like(count, site // 2 ** 32)]
    for _ in range(10):
        left, right = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(right >> half) ^ x[1] ^ key[0], right & low, (left >> half) ^ x[3] ^ key[1], left & low]
        key = (key + np.array([0x9E3779B9, 0xBB67AE85], dtype=u)) & low
    parts = np.empty((len(count), 8), dtype=np.uint16)
    for k in range(8):
        parts[:, k] = (x[k // 2] >> u(16 * (k % 2))) & u(0xFFFF)
    bar = min(65535, round(p * 65536))
    kept = torch.from_numpy((parts.reshape(-1)[:n] >= bar).reshape(shape)).to("cuda")
    return kept.double() / (1.0 - bar / 65536.0)


def exact(case, seed):
    s, kind, D = prepare(case, seed), case["kind"], torch.float64
    if kind == "dropout":
        return s["x"].to(D) * _factors(s, case["site"], (case["rows"], case["cols"]), case["p"])
    if kind in ("norms", "norms_grad"):
        leaf = {k: s[k].to(D).requires_grad_(kind == "norms_grad") for k in ("y", "gate", "after_weight", "after_bias", "before_weight", "before_bias") if k in s}

        def norm(x, name):
            if case[name] == "none":
                return x
            if case[name] == "layer":
                x = x - x.mean(1, keepdim=True)
            x = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
            return x * leaf[name + "_weight"] + leaf.get(name + "_bias", 0.0)

        def gated(b):
            if "gate" not in leaf:
                return b
            return b * leaf["gate"] if case["gate"] == 1 else (b.unflatten(0, (case["gate"], -1)) * leaf["gate"][:, None]).flatten(0, 1)

        branch = gated(norm(leaf["y"], "after") * _factors(s, 3, (case["rows"], case["dim"]), case["p"]))
        if kind == "norms":
            out = s["x"].to(D) * case["scale"] + branch
            return {"out": out, "h": norm(out, "before")} if case["before"] != "none" else {"out": out}
        # the stream behind the block is given; its gradient goes through the second norm, then to both addends
        leaf["out"] = s["out"].to(D).requires_grad_()
        if case["before"] != "none":
            norm(leaf["out"], "before").backward(s["g_h"].to(D))
        g = s["g_out"].to(D) + (leaf["out"].grad if leaf["out"].grad is not None else 0.0)
        branch.backward(g)
        found = {"d" + k: t.grad for k, t in leaf.items()} | {"dx": g * case["scale"]}
        return {k: found[k] for k in NORMS_GRADS if k in found}
    w, parts, v, c = s["weight"].to(D), [], case["vocab"], case["scale"]
    dw = torch.zeros_like(w) if kind == "head_grad" else None
    for at in range(0, case["rows"], 1024):
        rows = slice(at, min(case["rows"], at + 1024))
        x, ids = s["hidden"][rows].to(D), s["ids"][rows].long()
        logq = torch.log_softmax(c * (x @ w.T), 1)
        q = torch.exp(logq)
        h = -(q * logq).sum(1)
        scored = (ids >= 0) & (ids < v)
        token = torch.arange(len(ids), device="cuda"), ids.clamp(0, v - 1)
        logp = torch.where(scored, logq[token], 0.0)
        if kind == "head":
            parts.append((logp, h))
            continue
        gl, ge = torch.where(scored, s["gl"][rows].to(D), 0.0), s["ge"][rows].to(D)
        logq += h[:, None]
        q *= -gl[:, None] - ge[:, None] * logq
        q[token] += gl
        q *= c
        parts.append((logp, h, q @ w))
        dw += q.T @ x
    joined = [torch.cat(p) for p in zip(*parts)]
    return joined if kind == "head" else joined + [dw]


# ------------------------------------------------------------------------------------------ bounds
def work(case):
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * SIZE[case["type"]] + 8, "flops": 2 * n}
    if kind in ("norms", "norms_grad"):
        r, d, x, t, second = case["rows"], case["dim"], SIZE[case["x"]], SIZE[case["type"]], case["before"] != "none"
        weights = sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("after", "before")) + case["gate"]
        if kind == "norms":  # stream and branch in; stream and, normed, the next block's input out
            return {"bytes": r * d * (2 * x + t * (1 + second)) + 4 * d * weights, "flops": 12 * r * d}
        # the stream kept, both gradients and the branch in; both gradients out
        return {"bytes": r * d * (x * (2 + second) + t * (2 + second)) + 16 * r + 8 * d * weights, "flops": 30 * r * d}
    r, v, d, t = case["rows"], case["vocab"], case["dim"], SIZE[case["type"]]
    if kind == "head":
        return {"bytes": t * d * (r + v) + 12 * r, "flops": 2 * r * v * d}
    return {"bytes": 2 * t * d * (r + v) + 20 * r, "flops": 6 * r * v * d}  # each of the three products once
