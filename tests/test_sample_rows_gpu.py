"""A row's token is its own: the same whichever rows are drawn beside it."""
import numpy as np
import pytest

from oracle import sequence as s
from tests.test_inference_ops_gpu import _logits, _sample, lib  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [s.F32, s.F16, s.BF16])
@pytest.mark.parametrize("vocab", [300, 5003, 70001])
def test_rows_drawn_alone_and_together(lib, dtype, vocab):  # noqa: F811
    l, u = _logits(24, vocab, vocab)
    cuts = {"temperature": 0.9, "top_k": 200, "top_p": 0.95, "min_p": 0.01}
    tokens, logp = _sample(lib, l, u, dtype, **cuts)
    for rows in (np.s_[:1], np.s_[5:8], np.s_[::-1]):
        some, some_logp = _sample(lib, l[rows], u[rows], dtype, **cuts)
        assert np.array_equal(some, tokens[rows]) and np.array_equal(some_logp, logp[rows])
