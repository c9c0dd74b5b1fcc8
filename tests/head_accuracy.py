"""How far logits summed as the kernels sum them may be from 64 bits, for inputs on which that is narrow enough to tell the sums that are made from poorer ones.

The tensor cores add 16 products at a time to a sum in f32 and cut what lies below its last place, 2U of it at most each time (U = 2^-24); chains of such additions (16-bit
operands: 512 k at most; f32 operands, in pieces: 64 k) are added up to nearest."""
import numpy as np

from language_oracle import U, bf16_bits, bf16_values

KEPT = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]  # of the nine products of pieces, those that are made


def pieces(x):
    """f32 -> its three bf16 pieces, each to nearest."""
    found, rest = [], np.asarray(x, np.float32)
    for _ in range(3):
        found.append(bf16_values(bf16_bits(rest)).reshape(rest.shape))
        rest = rest - found[-1]
    return [p.astype(np.float64) for p in found]


def products(h, w, kept):
    a, b = pieces(h), pieces(w)
    return sum(a[i] @ b[j].T for i, j in kept)


def log_p(x, ids):
    m = x.max(1, keepdims=True)
    return (x - m - np.log(np.exp(x - m).sum(1, keepdims=True)))[np.arange(len(ids)), ids]


def positive_sums(terms, kind):
    """The bound of sums of positive terms [rows, K] of like size, which every cut makes smaller: cut by cut and addition by addition.

    A product of bf16 numbers has 16 bits.  In a chain of 512 k and less such a term is 2^-9 of the sum and more, so that it ends at 2^-24 of it and a cut takes what the sum itself has below its last
    place, 2U at most.  A product of f16 numbers has 22 bits, six of them below that, so that each of the 16 that are added at a time is cut as well.  With three places kept under the sum's
    last, 2^-26 of it, they lose half of that on average, 16 x 2^-27 = 2U together: with the sum's own cut, the two cuts of 2U that head_oracle.py counts for 16 products."""
    f32, chain, cut = kind == "f32", 64 if kind == "f32" else 512, 4 * U if kind == "f16" else 2 * U
    rows, k = terms.shape
    blocks = -(-k // 64)
    per = -(-blocks // -(-blocks // (chain // 64))) * 64  # chains of equal length, whole blocks of 64
    total, running = np.zeros(rows), np.zeros(rows)
    for at in range(0, k, per):
        t = terms[:, at:at + per]
        sums = np.stack([t[:, :j].sum(1) for j in range(16, t.shape[1] + 16, 16)], 1)
        total += cut * sums.sum(1)
        if f32:  # the five small products' sums are 2^-8 of the block's and less: 20 cuts of them; what is not made is 2^-26 of it
            total += 2 * U * 20 / 256 * sums[:, -1] + 2.0 ** -26 * 1.01 * sums[:, -1]
        running += sums[:, -1]
        total += U * running
    return total


def rms_limit(h, w, ids):
    """The root mean square of the error of log p from f32 operands, K = 512, terms of random signs with size s = sqrt(sum of the terms' squares).  Of a block of 64 k four cuts count, 2U of a
    partial sum each at most, which behind the j-th is 0.8 sqrt(16 j / K) s on average: 0.8 x 4 (1 + 1.42 + 1.74 + 2) / sqrt(K) = 19.7 / sqrt(K) of s together; K / 64 blocks of independent
    signs: 19.7 / 8 x 2U s = 4.9 U s.  Additions to nearest: U / sqrt(3) of sums that grow to s: U s sqrt((K / 64) / 6) = 1.2 U s.  Together 5.1 U s; of the logit asked for and of the mean of the others
    under p: sqrt(2).  Then the difference from the largest, the logarithm and the last difference: 2U |log p| and 4U."""
    assert h.shape[1] == 512
    s = np.sqrt(((h.astype(np.float64) ** 2) @ (w.astype(np.float64) ** 2).T).mean())
    want = log_p(h.astype(np.float64) @ w.astype(np.float64).T, ids)
    return np.sqrt(2) * 5.1 * U * s + 2 * U * np.sqrt((want ** 2).mean()) + 4 * U


def random_signs(seed):
    rng = np.random.default_rng(seed)
    h, w = rng.standard_normal((256, 512)).astype(np.float32), (8 / np.sqrt(512) * rng.standard_normal((128, 512))).astype(np.float32)
    return h, w, rng.integers(0, 128, 256).astype(np.int32)
