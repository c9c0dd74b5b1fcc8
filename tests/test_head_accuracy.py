"""The limit that f32 hidden states' log probabilities are held against on a GPU tells six products of pieces from any five: computed here, in 64 bits."""
import numpy as np
import pytest

import head_accuracy as A


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_the_limit_tells_poorer_sums(seed):
    h, w, ids = A.random_signs(seed)
    want = A.log_p(h.astype(np.float64) @ w.astype(np.float64).T, ids)
    rms = lambda kept: np.sqrt(((A.log_p(A.products(h, w, kept), ids) - want) ** 2).mean())  # noqa: E731
    limit = A.rms_limit(h, w, ids)
    assert rms(A.KEPT) < 0.1 * limit
    for i in range(len(A.KEPT)):
        assert rms(A.KEPT[:i] + A.KEPT[i + 1:]) > 1.2 * limit, A.KEPT[i]


def test_pieces_are_the_whole_number():
    x = np.random.default_rng(3).standard_normal(10000).astype(np.float32)
    assert np.array_equal(sum(A.pieces(x)), x.astype(np.float64))
