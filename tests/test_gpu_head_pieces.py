"""Log probabilities from hidden states whose results are not where the tensor memory can be written to, in several pieces of the vocabulary, against 64 bits."""
import numpy as np
import pytest

import sage_b200 as S

from test_gpu_head import check
from test_gpu_language import Held

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = S.Context(0)
    yield c
    assert c.status_word() == 0
    c.close()


@pytest.mark.parametrize("kind,rows,out", [("bf16", 4100, "bf16"), ("bf16", 4100, "f32"), ("f32", 2100, "f32")])
def test_pieces_of_an_odd_width(ctx, kind, rows, out):
    """Sums of each piece of the weight lie in the same memory, one after the other."""
    with Held(ctx) as d:
        check(ctx, d, np.random.default_rng(6), rows, 40001, 37, kind, out=out)
