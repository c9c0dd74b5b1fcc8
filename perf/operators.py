"""The operators at the two ends of a language model and its update, as cases that can be timed and compared: token
embedding and its gradient, log probabilities of given tokens (entropy, top alternatives, gradient), AdamW over many
tensors with states in 32 or 8 bits.

  listed()            the cases
  draw(rng)           one more case of the same ranges
  prepare(case, seed) inputs, buffers and states of a program that is about to run the case, on the GPU
  run(state)          one pass: in plain torch operations, or (`own`) through the package's entry points
  work(case)          the bytes and operations one pass cannot do without
  exact(case, seed)   what run() returns, computed in 64 bits from the operator's definition
"""
import math

import torch

own = False

F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256  # elements of an 8-bit state that share a scale; every tensor of an update starts on such a boundary


def listed():
    return [
        # The next token of eight sequences being generated: latency.
        {"name": "embed_8x768_f32", "kind": "embed", "tokens": 8, "vocab": 30522, "dim": 768, "table": "f32", "out": "f32", "scale": 1.0},
        # A prompt batch of a large half-precision model whose embeddings are scaled by the root of the width.
        {"name": "embed_32768x4096_bf16", "kind": "embed", "tokens": 32768, "vocab": 131072, "dim": 4096, "table": "bf16", "out": "bf16", "scale": 64.0},
        # The headline training batch of the base encoder (32 x 128 tokens): a dense gradient of its table.
        {"name": "embed_grad_4096x768_f32", "kind": "embed_grad", "tokens": 4096, "vocab": 30522, "dim": 768, "grad": "f32", "scale": 1.0, "add": False},
        # A long batch of half-precision gradients, odd vocabulary and width, added to a gradient that is already there (a tied table).
        {"name": "embed_grad_65521x1000_bf16", "kind": "embed_grad", "tokens": 65521, "vocab": 50021, "dim": 1000, "grad": "bf16", "scale": 31.6, "add": True},
        # One step of generation for one sequence: the log probability of the sampled token and its five alternatives.
        {"name": "logp_1x30522_f32_top5", "kind": "logp", "rows": 1, "vocab": 30522, "logits": "f32", "scale": 1.0, "top": 5, "masked": False},
        # A server's step for 64 sequences at a temperature, 20 alternatives each, some rows under a vocabulary mask.
        {"name": "logp_64x131072_bf16_top20", "kind": "logp", "rows": 64, "vocab": 131072, "logits": "bf16", "scale": 1.25, "top": 20, "masked": True},
        # Scoring a corpus: fp32 logits, an odd vocabulary, no alternatives.
        {"name": "logp_8192x50021_f32", "kind": "logp", "rows": 8192, "vocab": 50021, "logits": "f32", "scale": 1.0, "top": 0, "masked": False},
        # The same with its gradient, where what the loss makes of the log probabilities is known only after them.
        {"name": "logp_grad_4096x30522_f32", "kind": "logp_grad", "rows": 4096, "vocab": 30522, "logits": "f32", "scale": 1.0, "masked": False},
        # A weighted likelihood with an entropy bonus over half-precision logits: values and gradient in one call.
        {"name": "loss_8192x131072_bf16", "kind": "loss", "rows": 8192, "vocab": 131072, "logits": "bf16", "scale": 1.0, "masked": False},
        # Every tensor of the base encoder, fp32 throughout.
        {"name": "adamw_base_32bit", "kind": "adamw", "layers": 12, "width": 768, "vocab": 30522, "bits": 32, "grad": "f32", "copy": False},
        # The update of a small adapter: a few dozen small tensors, states in 8 bits.
        {"name": "adamw_small_8bit", "kind": "adamw", "layers": 2, "width": 72, "vocab": 997, "bits": 8, "grad": "f32", "copy": False},
        # A large encoder in mixed precision: half-precision gradients and copies of the weights, states in 8 bits.
        {"name": "adamw_large_8bit", "kind": "adamw", "layers": 24, "width": 1024, "vocab": 30522, "bits": 8, "grad": "bf16", "copy": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "logp", "logp", "logp_grad", "loss", "adamw", "adamw"])
    most = {c["kind"]: work(c)["bytes"] for c in listed()}  # of each kind the last, its largest
    most["logp"] = max(work(c)["bytes"] for c in listed() if c["kind"] == "logp")
    most["logp_grad"] = most["loss"]
    while True:
        if kind == "embed":
            t = rng.choice(["f32", "bf16", "f16"])
            c = {"kind": kind, "tokens": _log_int(rng, 1, 65536), "vocab": _log_int(rng, 100, 131072), "dim": _log_int(rng, 16, 4096), "table": t,
                 "out": rng.choice(["f32", t]), "scale": rng.choice([1.0, 8.5])}
        elif kind == "embed_grad":
            c = {"kind": kind, "tokens": _log_int(rng, 1, 65536), "vocab": _log_int(rng, 100, 131072), "dim": _log_int(rng, 16, 4096),
                 "grad": rng.choice(["f32", "bf16", "f16"]), "scale": rng.choice([1.0, 8.5]), "add": rng.random() < 0.4}
            if 4 * c["vocab"] * c["dim"] > 1 << 30:
                continue
        elif kind == "adamw":
            c = {"kind": kind, "layers": rng.randint(1, 24), "width": _log_int(rng, 32, 1024), "vocab": _log_int(rng, 100, 65536), "bits": rng.choice([8, 32]),
                 "grad": rng.choice(["f32", "bf16", "f16"]), "copy": rng.random() < 0.3}
        else:
            c = {"kind": kind, "rows": _log_int(rng, 1, 16384), "vocab": _log_int(rng, 100, 262144), "logits": rng.choice(["f32", "bf16", "f16"]),
                 "scale": rng.choice([1.0, 0.7, 1.25]), "masked": rng.random() < 0.4}
            if kind == "logp":
                c["top"] = rng.choice([0, 1, 5, 20, 32])
        if kind in ("embed", "embed_grad") and rng.random() < 0.5:  # widths are round as often as not
            c["dim"] = (c["dim"] + 63) // 64 * 64
        # int64 keys of the plain form's selection take four to eight times the logits' memory
        if work(c)["bytes"] <= most[kind] * (0.25 if c.get("top") else 1.0):
            return c


def shapes(case):
    """The tensors of an encoder of so many layers: embeddings, then per layer four projections, two norms and a feed-forward."""
    w, v = case["width"], case["vocab"]
    one = [(w, w), (w,)] * 4 + [(w,), (w,)] + [(w, 4 * w), (4 * w,), (4 * w, w), (w,)] + [(w,), (w,)]
    return [(v, w), (512, w), (w,), (w,)] + one * case["layers"] + [(w, 2), (2,)]


def _starts(case):
    at, found = 0, []
    for s in shapes(case):
        n = math.prod(s)
        found.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return found, at


# ------------------------------------------------------------------------------------------ inputs
def _tokens(g, n, vocab, none):
    """Token numbers whose frequencies fall with their number as words' do; a share `none` of them stands for no token."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().clamp(0, vocab - 1).to(torch.int32)
    if none:
        ids[torch.rand(n, generator=g, device="cuda") < none] = -1
    return ids


def _logits(case, g):
    r, v, t = case["rows"], case["vocab"], F[case["logits"]]
    x = torch.randn((r, v), generator=g, device="cuda", dtype=t) * 2.5
    ids = _tokens(g, r, v, 0.0)
    x[torch.arange(r, device="cuda"), ids.long()] += 8.0  # a trained model gives its tokens weight
    if case["masked"]:  # a grammar's mask: half of the vocabulary in every other row, and one row with nothing allowed
        closed = torch.rand((v,), generator=g, device="cuda") < 0.5
        x[::2].masked_fill_(closed, float("-inf"))
        if r > 8:
            x[5] = float("-inf")
    ids[torch.rand(r, generator=g, device="cuda") < (0.1 if r > 1 else 0.0)] = -1  # tokens that are not scored
    return x, ids


def prepare(case, seed):
    g, kind, dev = torch.Generator(device="cuda").manual_seed(seed), case["kind"], {"device": "cuda"}
    s = {"case": case, "kind": kind, "handles": None}
    if kind == "embed":
        t, d = case["tokens"], case["dim"]
        s["table"] = (torch.randn((case["vocab"], d), generator=g, device="cuda") * 0.02).to(F[case["table"]])
        s["ids"] = _tokens(g, t, case["vocab"], 0.05)
        s["y"] = torch.empty((t, d), dtype=F[case["out"]], **dev)
    elif kind == "embed_grad":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        s["ids"] = _tokens(g, t, v, 0.05)
        s["g"] = (torch.randn((t, d), generator=g, device="cuda") * 1e-2).to(F[case["grad"]])
        s["y"] = torch.randn((v, d), generator=g, device="cuda") * 1e-2 if case["add"] else torch.empty((v, d), **dev)
    elif kind in ("logp", "logp_grad", "loss"):
        r, v = case["rows"], case["vocab"]
        s["x"], s["ids"] = _logits(case, g)
        s["logp"], s["entropy"] = torch.empty(r, **dev), torch.empty(r, **dev)
        if kind == "logp":
            s["top_ids"], s["top_logp"] = torch.empty((r, case["top"]), dtype=torch.int32, **dev), torch.empty((r, case["top"]), **dev)
        else:
            s["gl"] = -torch.rand(r, generator=g, device="cuda") / r
            s["ge"] = -torch.rand(r, generator=g, device="cuda") * (0.01 / r)
            s["stats"], s["dx"] = torch.empty((r, 2), **dev), torch.empty((r, v), dtype=s["x"].dtype, **dev)
    else:
        places, n = _starts(case)
        there = torch.zeros(n, dtype=torch.bool, **dev)
        for at, m in places:
            there[at:at + m] = True
        s["places"], s["step"] = places, 10
        normal = lambda std: torch.randn(n, generator=g, device="cuda") * std  # noqa: E731
        s["p"] = torch.where(there, normal(0.02), 0.0)
        size = torch.exp(normal(1.0))  # some directions have larger gradients than others
        s["g"] = torch.where(there, normal(1e-3) * size, 0.0).to(F[case["grad"]])
        m, v = torch.where(there, normal(3e-4) * size, 0.0), torch.where(there, torch.square(1e-3 * size), 0.0)
        if case["bits"] == 8:
            s["m"], s["m_scale"] = _encode(m, 127)
            s["v"], s["v_scale"] = _encode(torch.sqrt(v), 255)
            s["m_values"], s["v_values"] = torch.empty(n, **dev), torch.empty(n, **dev)
        else:
            s["m"], s["v"] = m, v
        s["w"] = torch.zeros(n, dtype=torch.bfloat16, **dev) if case["copy"] else None
    return s


# ------------------------------------------------------------------------------------------ 8-bit states
def _encode(x, top):
    """Codes of a square law and a scale for each block: |x| = scale * code^2, the block's largest at code `top`; what is not zero
    in unsigned codes (second moments) does not become zero.  A block with a value that is not finite has a scale that is not a
    number; one below 2^-100 throughout is zero."""
    x = x.reshape(-1, BLOCK)
    largest = x.abs().amax(1, keepdim=True)
    some, fine = largest >= 2.0 ** -100, torch.isfinite(largest)
    r = torch.where(some & fine, float(top * top) / largest, 0.0)
    code = torch.round(torch.sqrt(torch.where(fine, x.abs(), 0.0) * r))
    if top == 255:
        code = torch.where((x > 0) & some & fine, code.clamp(1, 255), code).to(torch.uint8)
    else:
        code = (torch.sign(torch.where(fine, x, 0.0)) * code.clamp(max=127)).to(torch.int8)
    scale = torch.where(fine, torch.where(some, largest / float(top * top), 0.0), float("nan"))
    return code.reshape(-1), scale.reshape(-1)


def _decode(code, scale, dtype=torch.float32):
    c = code.to(dtype).reshape(-1, BLOCK)
    return (scale.to(dtype).reshape(-1, 1) * (c * c.abs())).reshape(-1)


LR, BETA1, BETA2, EPS, DECAY, GRAD_SCALE = 1e-3, 0.9, 0.999, 1e-8, 0.01, 0.5


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
        if kind == "adamw":
            part = lambda k, at, n: ctx.borrow(s[k][at:at + n]) if s.get(k) is not None else None  # noqa: E731
            blocks = lambda k, at, n: part(k, at // BLOCK, (n + BLOCK - 1) // BLOCK)  # noqa: E731
            h["tensors"] = L.AdamWTensors(ctx, [
                L.adamw_tensor(part("p", at, n), part("g", at, n), part("m", at, n), part("v", at, n), blocks("m_scale", at, n), blocks("v_scale", at, n), part("w", at, n))
                for at, n in s["places"]])
        s["handles"] = h
    if kind == "embed":
        L.embedding(h["table"], h["ids"], h["y"], scale=case["scale"])
        return s["y"]
    if kind == "embed_grad":
        L.embedding_grad(h["g"], h["ids"], h["y"], scale=case["scale"], add=case["add"])
        return s["y"]
    if kind == "logp":
        if not case["top"]:
            L.token_log_probs(h["x"], h["ids"], h["logp"], h["entropy"], scale=case["scale"])
            return s["logp"], s["entropy"]
        L.token_log_probs(h["x"], h["ids"], h["logp"], h["entropy"], top_ids=h["top_ids"], top_log_probs=h["top_logp"], scale=case["scale"])
        return s["logp"], s["entropy"], s["top_ids"], s["top_logp"]
    if kind == "logp_grad":
        L.token_log_probs(h["x"], h["ids"], h["logp"], h["entropy"], stats=h["stats"], scale=case["scale"])
        L.token_log_probs_grad(h["x"], h["ids"], h["stats"], h["entropy"], h["gl"], h["ge"], h["dx"], scale=case["scale"])
        return s["logp"], s["entropy"], s["dx"]
    if kind == "loss":
        L.token_log_probs_and_grad(h["x"], h["ids"], h["gl"], h["ge"], h["logp"], h["entropy"], h["dx"], scale=case["scale"])
        return s["logp"], s["entropy"], s["dx"]
    s["step"] += 1
    L.adamw_step(h["tensors"], step=s["step"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY, grad_scale=GRAD_SCALE)
    if case["bits"] == 8:
        L.adamw_states(h["m"], h["m_scale"], h["v"], h["v_scale"], h["m_values"], h["v_values"])
        return [s["p"], s["m_values"], s["v_values"]] + ([s["w"]] if case["copy"] else [])
    return [s["p"], s["m"], s["v"]] + ([s["w"]] if case["copy"] else [])


def _run_plain(s):
    kind, case = s["kind"], s["case"]
    if kind == "embed":
        there = (s["ids"] >= 0) & (s["ids"] < case["vocab"])
        rows = s["table"][s["ids"].clamp(0, case["vocab"] - 1)].float() * case["scale"]
        return torch.where(there[:, None], rows, 0.0).to(s["y"].dtype)
    if kind == "embed_grad":
        there = (s["ids"] >= 0) & (s["ids"] < case["vocab"])
        rows = torch.where(there[:, None], s["g"].float() * case["scale"], 0.0)
        if case["add"]:
            return s["y"].index_add_(0, s["ids"].clamp(0, case["vocab"] - 1), rows)
        return torch.zeros_like(s["y"]).index_add_(0, s["ids"].clamp(0, case["vocab"] - 1), rows)
    if kind in ("logp", "logp_grad", "loss"):
        x = s["x"].float() * case["scale"]
        return _log_probs(x, s["x"], s["ids"], case.get("top", 0), s.get("gl"), s.get("ge"), case["scale"])
    s["step"] += 1
    b1, b2, t = BETA1, BETA2, s["step"]
    g = s["g"].float() * GRAD_SCALE
    if case["bits"] == 8:
        m, root = _decode(s["m"], s["m_scale"]), _decode(s["v"], s["v_scale"])
        v = root * root
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g * g * (1.0 - b2)
    root = torch.sqrt(v)
    size, spread = LR / (1.0 - b1 ** t), 1.0 / math.sqrt(1.0 - b2 ** t)
    s["p"] = s["p"] * (1.0 - LR * DECAY) - (m * size) / (root * spread + EPS)
    copy = [s["p"].to(torch.bfloat16)] if case["copy"] else []
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode(m, 127)
        s["v"], s["v_scale"] = _encode(root, 255)
        m, root = _decode(s["m"], s["m_scale"]), _decode(s["v"], s["v_scale"])
        return [s["p"], m, root * root] + copy
    s["m"], s["v"] = m, v
    return [s["p"], m, v] + copy


def _log_probs(x, logits, ids, top, gl, ge, scale):
    """From scaled logits: log probabilities, entropy, and the alternatives (by the logits as they came) or the gradient."""
    v = x.shape[1]
    m = x.amax(1, keepdim=True)
    some = m > float("-inf")  # rows in which anything is allowed
    d = x - torch.where(some, m, 0.0)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    there = (ids >= 0) & (ids < v)
    own_d = d.gather(1, ids.clamp(0, v - 1).long()[:, None])
    logp = torch.where(there, torch.where(some, own_d - log_z, float("-inf"))[:, 0], 0.0)
    ed = torch.where(e > 0, e * d, 0.0)
    entropy = torch.where(some, log_z - ed.sum(1, keepdim=True) / z, 0.0)
    if gl is not None:
        gl, ge = torch.where(there, gl, 0.0)[:, None], ge[:, None]
        p = e / z
        dx = -gl * p - ge * (torch.where(p > 0, p * (d - log_z), 0.0) + p * entropy)
        dx.scatter_add_(1, ids.clamp(0, v - 1).long()[:, None], gl)
        return logp, entropy[:, 0], torch.where(some, dx * scale, 0.0).to(logits.dtype)
    if not top:
        return logp, entropy[:, 0]
    # unique whole-number keys: larger logits first, then lower tokens
    bits = (logits.float() + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -2147483648 - bits) * (1 << 32) + (v - torch.arange(v, device=x.device))
    best = v - (key.topk(top, 1).values & 0xFFFFFFFF)
    return logp, entropy[:, 0], best.to(torch.int32), torch.where(some, d.gather(1, best) - log_z, float("-inf"))


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s, kind, D = prepare(case, seed), case["kind"], torch.float64
    if kind in ("embed", "embed_grad"):
        keep = ((s["ids"] >= 0) & (s["ids"] < case["vocab"])).nonzero()[:, 0]
        token = s["ids"][keep].long()
        if kind == "embed":
            y = torch.zeros((case["tokens"], case["dim"]), dtype=D, device="cuda")
            y[keep] = s["table"].to(D)[token] * case["scale"]
            return y
        y = s["y"].to(D) if case["add"] else torch.zeros(s["y"].shape, dtype=D, device="cuda")
        return y.index_add_(0, token, s["g"].to(D)[keep] * case["scale"])
    if kind in ("logp", "logp_grad", "loss"):
        parts, r = [], case["rows"]
        for at in range(0, r, 512):
            rows = slice(at, min(r, at + 512))
            x, ids = s["x"][rows].to(D) * case["scale"], s["ids"][rows].long()
            lse = torch.logsumexp(x, 1, keepdim=True)
            open_row = lse > float("-inf")
            logq = torch.where(open_row, x - lse, float("-inf"))
            q = torch.exp(logq)
            qlogq = torch.nan_to_num(q * logq, nan=0.0)
            h = -qlogq.sum(1, keepdim=True)
            scored = (ids >= 0) & (ids < case["vocab"])
            at_id = torch.nn.functional.one_hot(ids.clamp(0, case["vocab"] - 1), case["vocab"]).to(D) if kind != "logp" else None
            logp = torch.where(scored, logq.gather(1, ids.clamp(0, case["vocab"] - 1)[:, None])[:, 0], 0.0)
            if kind == "logp":
                top = torch.sort(logq, 1, descending=True).values[:, :case["top"]] if case["top"] else None
                parts.append((logp, h[:, 0], top))
            else:
                gl, ge = torch.where(scored, s["gl"][rows].to(D), 0.0)[:, None], s["ge"][rows].to(D)[:, None]
                dx = case["scale"] * (gl * (at_id - q) - ge * (qlogq + q * h))
                parts.append((logp, h[:, 0], torch.where(open_row, dx, 0.0)))
        joined = [torch.cat(p) if p[0] is not None else None for p in zip(*parts)]
        if kind == "logp":
            return joined[:2] if not case["top"] else [joined[0], joined[1], None, joined[2]]
        return joined
    t, g = s["step"] + 1, s["g"].to(D) * GRAD_SCALE
    m = _decode(s["m"], s["m_scale"], D) if case["bits"] == 8 else s["m"].to(D)
    v = torch.square(_decode(s["v"], s["v_scale"], D)) if case["bits"] == 8 else s["v"].to(D)
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = s["p"].to(D) * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    if case["bits"] == 8:
        def stored(x, top):
            x = x.reshape(-1, BLOCK)
            largest = x.abs().amax(1, keepdim=True)
            share = torch.where(largest > 0, x.abs() / largest, 0.0)
            c = torch.round(top * torch.sqrt(share))
            c = torch.where((share > 0) & (c < 1) & (top == 255), 1.0, c)
            return (torch.sign(x) * largest * torch.square(c / top)).reshape(-1)
        m, v = stored(m, 127), torch.square(stored(torch.sqrt(v), 255))
    return [p, m, v] + ([p] if case["copy"] else [])


# ------------------------------------------------------------------------------------------ bounds
def work(case):
    kind = case["kind"]
    if kind == "embed":
        n = case["tokens"] * case["dim"]
        return {"bytes": 4 * case["tokens"] + n * (SIZE[case["table"]] + SIZE[case["out"]]), "flops": n}
    if kind == "embed_grad":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        rows = v
        if case["add"]:  # the rows that some token reaches, expected: frequencies fall as 1 / (number + 1)
            rows = int(sum(1.0 - math.exp(-0.95 * t * math.log((k + 2) / (k + 1)) / math.log(v + 1)) for k in range(v)))
        return {"bytes": 4 * t + t * d * SIZE[case["grad"]] + 4 * rows * d * (2 if case["add"] else 1), "flops": 2 * t * d}
    if kind == "logp":
        r, v = case["rows"], case["vocab"]
        return {"bytes": r * v * SIZE[case["logits"]] + r * (12 + 8 * case["top"]), "flops": 6 * r * v}
    if kind in ("logp_grad", "loss"):
        r, v = case["rows"], case["vocab"]
        return {"bytes": 2 * r * v * SIZE[case["logits"]] + 20 * r, "flops": 14 * r * v}
    n = sum(math.prod(x) for x in shapes(case))
    states = 16 * n if case["bits"] == 32 else 4 * n + 16 * n // BLOCK + 8 * n  # read and written; in 8 bits also given back as values
    return {"bytes": n * (8 + SIZE[case["grad"]] + (2 if case["copy"] else 0)) + states, "flops": 16 * n}
