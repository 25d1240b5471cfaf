"""Products of operands in 8 bits at sizes where each way of computing them is chosen, the large tiles with
several for each workgroup, one after another."""
import numpy as np
import pytest

from ml_framework_amd import capi
from oracle import inference as q
from oracle import sequence as s
from tests.matmul_f8_ways import WAYS
from tests.test_inference_ops_gpu import Bytes, _matmul, _operands, lib  # noqa: F401 (a fixture)
from tests.test_sequence_ops_gpu import Rows, _close

pytestmark = pytest.mark.gpu

# a way's 16-bit code serves both types: every other size has one
SIZES = [(s.F32 if f32 else (s.BF16, s.F16)[i % 2], m, n, k) for i, (f32, m, n, k, _) in enumerate(WAYS)]


def _stored(ops, n, k, bias, dtype, gap, shift):
    """C as it is stored, of operands on the host."""
    m = ops[0].shape[0]
    dev = [Bytes(x.shape, x.dtype, x) for x in ops]
    b = Bytes(bias.shape, np.float32, bias)
    c = Rows((m, n), dtype, n + gap, shift)
    capi.call("seera_hip_matmul_f8", *[x.ptr for x in dev], b.ptr, c.ptr, m, n, k, n + gap, dtype)
    return c.raw()


def _parts(ops, bias, some=True):
    """(where in C, operands and bias of that part): a few rows of each 64, with the first and the last, and four
    blocks of 128 columns, the last one among them; or all of it."""
    a, sa, w, sw = ops
    m, n = a.shape[0], w.shape[0]
    if not some:
        yield np.s_[:, :], ops, bias
        return
    r = np.random.default_rng(m)
    rows = np.unique(np.r_[0, m - 1, np.arange(m)[r.random(m) < 3 / 64]])
    yield np.s_[rows], (a[rows], sa[rows], w, sw), bias
    for block in sorted({0, 1, n // 256, (n - 1) // 128}):
        cols = np.s_[block * 128:(block + 1) * 128]
        yield np.s_[:, cols], (a, sa, w[cols], sw[block:block + 1]), bias[cols]


@pytest.mark.parametrize("dtype,m,n,k", SIZES)
def test_every_way(lib, dtype, m, n, k):  # noqa: F811
    (a, sa, w, sw), bias = _operands(m, n, k, k, True)
    ops = a, sa / 16, w, sw  # inside fp16's range
    got = _stored(ops, n, k, bias, dtype, 3, 1)
    for at, part, b in _parts(ops, bias):
        want, bound = q.matmul(*part, b, fp32=dtype == s.F32)
        _close(s.load(got[at], dtype), want, bound, dtype, "C")


@pytest.mark.parametrize("dtype,m,n,k", SIZES)
def test_every_way_is_exact_on_whole_numbers(lib, dtype, m, n, k):  # noqa: F811
    """Small whole numbers with scales of powers of two: every sum is a whole number below 2^24 and no product is
    cut, so that the one rounding is the result's, and a term in a wrong place shows."""
    r = np.random.default_rng(m)
    kp = q.padded(k)
    a, w = np.zeros((m, kp), np.int8), np.zeros((n, kp), np.int8)
    a[:, :k], w[:, :k] = r.integers(-8, 9, (m, k), np.int8), r.integers(-8, 9, (n, k), np.int8)
    codes = q.encode(np.arange(-8, 9))
    sa, sw = 2.0 ** r.integers(0, 3, (m, kp // 128)), 2.0 ** r.integers(0, 3, (q.padded(n) // 128, kp // 128))
    bias = r.integers(-1000, 1001, n).astype(np.float32)
    ops = codes[a + 8], sa.astype(np.float32), codes[w + 8], sw.astype(np.float32)
    got = _stored(ops, n, k, bias, dtype, 0, 0)
    # numbers that fp16 cannot hold are infinite
    for at, part, b in _parts(ops, bias, m * n > 3e7):
        want, _ = q.matmul(*part, b)
        assert np.abs(want).max() < 2**24
        assert np.array_equal(got[at], s.store(want, dtype)), "C"


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


@pytest.mark.parametrize("dtype,m,n,k", [next(c for c, w in zip(SIZES, WAYS) if w[0] == f32 and w[4] == way) for f32, way in sorted({(w[0], w[4]) for w in WAYS})])
def test_scales_whose_product_leaves_the_range(lib, dtype, m, n, k):  # noqa: F811
    """Scales of 2^70 and 2^-62 (times ordinary ones), whose products fp32 holds no longer or with few
    bits, where their products with the sums are ordinary numbers: 0, sums of the smallest codes, sums of large ones.
    What has ordinary scales has the same bits as without them."""
    (a, sa, w, sw), bias = _operands(m, n, k, 5, True)
    clean = _stored((a, sa, w, sw), n, k, bias, dtype, 1, 0)
    a, sa, w, sw = a.copy(), sa.copy(), w.copy(), sw.copy()
    r = np.random.default_rng(n)
    few = lambda shape: np.where(r.random(shape) < 0.02, r.choice(np.array([1, 2, 3, 129], np.uint8), shape), 0).astype(np.uint8)  # noqa: E731
    high, low = np.unique(np.r_[0, r.integers(0, m, 9)]), np.unique(np.r_[m // 2, m - 1, r.integers(0, m, 9)])
    low = np.setdiff1d(low, high)
    a[high, :k], sa[high] = few((len(high), k)), sa[high] * np.float32(2.0**70)
    sa[low] *= np.float32(2.0**-62)
    w[128:256, :k], sw[1] = few((128, k)), sw[1] * np.float32(2.0**70)
    blocks = np.unique([2, n // 128])
    sw[blocks] *= np.float32(2.0**-62)
    changed = np.unique(np.r_[high, low])
    ordinary_rows = np.setdiff1d(np.arange(m), changed)
    ordinary = np.ones(n, bool)
    ordinary[128:256] = False
    for b in blocks:
        ordinary[b * 128:(b + 1) * 128] = False
    zero = np.zeros(n, np.float32)
    for bias in (bias, zero):
        got = _stored((a, sa, w, sw), n, k, bias, dtype, 1, 0)
        want, bound = q.matmul(a[changed], sa[changed], w, sw, bias, fp32=dtype == s.F32)
        if dtype == s.F16:  # beyond its range the results are infinite, and near its end they may be
            near = np.abs(np.abs(want) - 65520) <= bound
            values = np.where(near, 0, s.load(got[changed], dtype))
            over = (np.abs(want) > 65520) & ~near
            assert np.array_equal(values[over], np.copysign(np.inf, want[over]))
            keep = ~over & ~near
            _close(values[keep], want[keep], bound[keep], dtype, "C")
        else:
            _close(s.load(got[changed], dtype), want, bound, dtype, "C")
        if bias is not zero:
            at = np.ix_(ordinary_rows, ordinary)
            assert np.array_equal(got[at], clean[at])


@pytest.mark.parametrize("m,n", [(66000, 33000), (1, (1 << 27) + 5)])
def test_no_k_of_any_size(lib, m, n):  # noqa: F811
    """K == 0 gives the bias at sizes beyond 2^31 results, and of rows beyond 2^27."""
    bias = np.random.default_rng(n).integers(-128, 129, n).astype(np.float32)
    want = s.store(bias, s.BF16)
    b, c = Bytes((n,), np.float32, bias), capi.DeviceBuffer(m * n * 2)
    capi.call("seera_hip_matmul_f8", None, None, None, None, b.ptr, c.ptr, m, n, 0, n, s.BF16)
    for i in sorted({0, 1, 127, 128, m // 2, m - 1} & set(range(m))):
        row = np.empty(n, np.uint16)
        capi.check(lib.seera_hip_memcpy_d2h(row.ctypes.data, c.ptr + i * n * 2, row.nbytes))
        assert np.array_equal(row, want), i
    c.close()
    b.buf.close()
    capi.check(lib.seera_hip_empty_cache())
