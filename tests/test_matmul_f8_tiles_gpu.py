"""Products of operands in 8 bits whose workgroups take several tiles one after
another, at sizes where each of the large tiles is chosen."""
import numpy as np
import pytest

from oracle import sequence as s
from tests.test_inference_ops_gpu import _matmul, _operands, lib  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [np.nan, np.inf])
@pytest.mark.parametrize("dtype,m,n,k", [(s.BF16, 2300, 4300, 640), (s.F16, 4100, 4300, 640), (s.F32, 4100, 4300, 640), (s.BF16, 5000, 5000, 1024)])
def test_a_tile_leaves_nothing_to_the_next(lib, dtype, m, n, k, scale):  # noqa: F811
    """Scales that are not finite in the last block of K, of 128 of A's rows or of 128 of W's, change the
    results of those alone: all others have the same bits as without them."""
    (a, sa, w, sw), _ = _operands(m, n, k, 7, False)
    clean = _matmul(lib, (a, sa, w, sw), n, k, None, dtype)
    assert np.isfinite(clean).all()
    for at in (0, 5 * 128, m // 128 * 128):
        bad = sa.copy()
        bad[at:at + 128, -1] = scale
        got = _matmul(lib, (a, bad, w, sw), n, k, None, dtype)
        assert not np.isfinite(got[at:at + 128]).any()
        rest = np.r_[0:at, min(at + 128, m):m]
        assert np.array_equal(got[rest], clean[rest]), "A"
    for block in (0, 9, n // 128):
        bad = sw.copy()
        bad[block, -1] = scale
        got = _matmul(lib, (a, sa, w, bad), n, k, None, dtype)
        assert not np.isfinite(got[:, block * 128:(block + 1) * 128]).any()
        rest = np.r_[0:block * 128, min((block + 1) * 128, n):n]
        assert np.array_equal(got[:, rest], clean[:, rest]), "W"
