"""How much of the pool log probabilities from hidden states take at most, on a planning context: what the header says."""
import pytest

import sage_b200 as S
from sage_b200 import language as L

MB = 1 << 20


def most(rows, vocab, dim, kind, out, pitch):
    """Bytes of segments that a gradient adds to those of its operands."""
    ctx = S.Context(-1)
    e = lambda *s, d=S.F32: ctx.empty(s, d)  # noqa: E731
    r = lambda n, d: e(n, pitch, d=d).view((n, dim), (pitch, 1))  # noqa: E731
    b = r(rows, kind), r(vocab, kind), e(rows, d=S.I32), e(rows, 2), e(rows), e(rows), e(rows), r(rows, out), r(vocab, out)
    before = ctx.mem_stats()["mem_total"]
    L.head_log_probs_grad(*b)
    found = ctx.mem_stats()
    ctx.close()
    return found["mem_peak"] - before


@pytest.mark.parametrize("rows,vocab,dim,kind,out,pitch", [
    (8192, 131072, 4095, "bf16", "bf16", 4095),   # every row off its boundary, eight pieces
    (8192, 131072, 4095, "bf16", "f32", 4095),
    (8192, 131072, 4096, "bf16", "bf16", 4096),
    (4096, 60001, 1001, "f32", "f32", 1001),
    (600000, 2000, 64, "f16", "f16", 64),          # a piece of one tile is more than 256 MB
    (700, 30000, 72, "f16", "f32", 75)])
def test_memory_of_the_gradient(rows, vocab, dim, kind, out, pitch):
    t = {"bf16": S.BF16, "f16": S.F16, "f32": S.F32}
    size, aligned = 4 if out == "f32" else 2, (dim + 7) // 8 * 8
    planes = 3 if kind == "f32" else 1
    q = max(256 * MB, 512 * planes * (rows + 255))
    piece = max(256, q // (2 * planes * rows))  # tokens
    sums = (rows + 255) * aligned * 4 if q < rows * vocab * 2 * planes or pitch * size % 16 else 0
    if pitch * size % 16:
        sums += (min(piece, vocab) + 255) * aligned * 4
    copies = (rows + vocab) * aligned * (6 if kind == "f32" else 2 if pitch * 2 % 16 else 0)
    # (segments are rounded up to 2 MB, small ones to 20; what each row needs is 24 bytes and less)
    assert most(rows, vocab, dim, t[kind], t[out], pitch) <= q + sums + copies + 20 * MB + 24 * rows + 60 * MB
