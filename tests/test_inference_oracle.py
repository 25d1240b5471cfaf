"""Pins oracle/inference.py on the CPU before it checks the HIP kernels, with
planted mistakes that its checks must reject, and the argument checks of the entry
points, which run before any device work."""
import numpy as np
import pytest

from ml_framework_amd import capi
from oracle import inference as q
from oracle.sequence import BF16, load, store


def test_every_code():
    """The 254 finite codes against their definition, and back."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    v = q.decode(codes)
    for c, x in zip(codes, v):
        e, m = int(c) >> 3 & 15, int(c) & 7
        want = (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0**-6
        assert x == (-want if c & 128 else want)
    assert np.array_equal(q.encode(v), codes)
    assert v.max() == 448 and np.isnan(q.decode([0x7F, 0xFF])).all()


def test_encoding_rounds_to_nearest_even():
    v = q.decode(np.arange(127))
    middle = (v[1:] + v[:-1]) / 2
    assert np.array_equal(q.encode(middle), [c if c % 2 == 0 else c + 1 for c in range(126)])
    assert np.array_equal(q.encode(np.nextafter(middle, 1e9)), np.arange(1, 127))
    assert np.array_equal(q.encode(np.nextafter(middle, 0)), np.arange(126))
    assert np.array_equal(q.encode([449.0, 463.9, -463.9]), [0x7E, 0x7E, 0xFE])


def test_quantized_values_are_near():
    """Each within half a step, 2^-4 of itself or 2^-10 of the scale, of the value."""
    r = np.random.default_rng(1)
    v = (r.standard_normal((5, 300)) * np.exp(3 * r.standard_normal((5, 300)))).astype(np.float32)
    v[2] = 0
    v[3, :128] *= np.float32(1e-42)
    for codes, scales in (q.quantize_rows(v), (lambda c, s: (c, np.repeat(s, 5, 0)))(*q.quantize_weights(v))):
        assert codes.shape == (5, 384) and not codes[:, 300:].any()
        s = np.repeat(scales, 128, 1)[:, :300].astype(np.float64)
        off = np.abs(q.decode(codes)[:, :300] * s - v)
        assert np.all(off <= np.maximum(np.abs(v) * 2.0**-4, s * 2.0**-10) * (1 + 1e-6) + 2.0**-140)
    _, scales = q.quantize_rows(np.array([[np.inf, 1.0], [np.nan, 1.0], [0.0, 0.0]], np.float32))
    assert np.isnan(scales[:2]).all() and scales[2, 0] == 0


def test_check_codes_rejects_mistakes():
    r = np.random.default_rng(2)
    n = r.standard_normal((3, 200)).astype(np.float32)
    codes, scales = q.quantize_rows(n)
    exact = np.zeros_like(n, np.float64)
    q.check_codes(codes, scales, n.astype(np.float64), exact)
    for at, by in (((0, 5), 1), ((2, 199), -1), ((1, 130), 128)):
        bad = codes.copy()
        bad[at] = (int(bad[at]) + by) % 256
        with pytest.raises(AssertionError, match="codes"):
            q.check_codes(bad, scales, n.astype(np.float64), exact)
    bad = codes.copy()
    bad[1, 200] = 1
    with pytest.raises(AssertionError, match="padding"):
        q.check_codes(bad, scales, n.astype(np.float64), exact)
    with pytest.raises(AssertionError, match="scales"):
        q.check_codes(codes, scales * np.float32(1 + 1e-6), n.astype(np.float64), exact)


def test_product_of_codes_is_the_product_of_values():
    r = np.random.default_rng(3)
    a, w = r.standard_normal((4, 300)).astype(np.float32), r.standard_normal((150, 300)).astype(np.float32)
    (ac, sa), (wc, sw) = q.quantize_rows(a), q.quantize_weights(w)
    c, bound = q.matmul(ac, sa, wc, sw)
    A = q.decode(ac) * np.repeat(sa, 128, 1)
    W = q.decode(wc) * np.repeat(np.repeat(sw, 128, 1), 128, 0)[:150]
    assert np.allclose(c, A @ W.T, rtol=0, atol=1e-12)
    # and near the product of the values before they were rounded (2^-4 each, and both)
    assert np.all(np.abs(c - a.astype(float) @ w.T) <= 0.13 * (np.abs(a.astype(float)) @ np.abs(w.T)))
    # a term that is left out is seen
    ac[1, 7] = 0
    assert np.abs(q.matmul(ac, sa, wc, sw)[0] - c)[1].max() > 3 * bound[1].max()


# ---- sampling: the distribution that a grid of u draws ----


def _shares(l, n=20000, **kw):
    got = np.bincount([q.sample_row(l, (i + 0.5) / n, **kw)[0] for i in range(n)], minlength=l.size)
    return got / n


@pytest.mark.parametrize("kw,want", [
    ({}, [0.4, 0.1, 0.3, 0.2]),
    ({"temperature": 0.5}, [0.16 / 0.3, 0.01 / 0.3, 0.09 / 0.3, 0.04 / 0.3]),
    ({"top_k": 2}, [4 / 7, 0, 3 / 7, 0]),
    ({"top_k": 1}, [1, 0, 0, 0]),
    ({"top_p": 0.75}, [4 / 9, 0, 3 / 9, 2 / 9]),
    ({"top_p": 0.0}, [1, 0, 0, 0]),
    ({"top_p": 0.65}, [4 / 7, 0, 3 / 7, 0]),
    ({"top_k": 3, "top_p": 0.7}, [4 / 7, 0, 3 / 7, 0]),  # 0.7 of 0.9: reached by the first two
    ({"min_p": 0.45}, [4 / 9, 0, 3 / 9, 2 / 9]),
    ({"min_p": 2.0}, [1, 0, 0, 0]),
    ({"temperature": 0.0}, [1, 0, 0, 0])])
def test_shares(kw, want):
    assert np.abs(_shares(np.log([0.4, 0.1, 0.3, 0.2]), **kw) - want).max() < 1e-3


def test_ties_keep_the_lowest_index():
    l = np.array([0.0, 1.0, 0.0, 1.0, 0.0])
    assert [np.flatnonzero(_shares(l, 500, top_k=k)).tolist() for k in (1, 2, 3, 4)] == [[1], [1, 3], [0, 1, 3], [0, 1, 2, 3]]
    assert q.sample_row(l, 0.9, temperature=0)[0] == 1
    e = np.e
    assert np.flatnonzero(_shares(l, 500, top_p=(2 * e + 1.5) / (2 * e + 3))).tolist() == [0, 1, 2, 3]


def test_rows_with_nothing_or_something_odd():
    inf, nan = np.inf, np.nan
    assert q.sample_row(np.array([-inf, nan]), 0.5)[:2] == (-1, -inf)
    assert q.sample_row(np.array([]), 0.5)[:2] == (-1, -inf)
    assert np.allclose(_shares(np.array([nan, 0.0, -inf, 0.0]), 500), [0, 0.5, 0, 0.5])
    assert np.allclose(_shares(np.array([inf, 0.0, inf, 0.0]), 500), [0.5, 0, 0.5, 0])
    assert np.allclose(_shares(np.array([3.0, -inf, 1.0]), 500, temperature=np.inf), [0.5, 0, 0.5])
    assert q.sample_row(np.array([1.0, 2.0]), nan)[0] == 0 and q.sample_row(np.array([1.0, 2.0]), 1.0)[0] == 1
    assert q.sample_row(np.array([-0.0, 0.0]), 0.2, top_k=1)[0] == 0


def test_logp_of_the_cut_distribution():
    l = np.log([0.4, 0.1, 0.3, 0.2])
    token, logp, _ = q.sample_row(l, 0.99, top_k=2)
    assert token == 2 and abs(logp - np.log(3 / 7)) < 1e-10
    l = load(store(np.linspace(-3, 3, 50), BF16), BF16)
    token, logp, _ = q.sample_row(l, 0.3, temperature=0.7)
    p = np.exp(l / 0.7) / np.exp(l / 0.7).sum()
    assert np.cumsum(p)[token - 1] <= 0.3 < np.cumsum(p)[token] and abs(logp - np.log(p[token])) < 1e-10


# ---- refusals ----

P = 0x10000  # an address that no call reaches


def _refused(name, args, what):
    lib = capi.load()
    assert getattr(lib, name)(*args) == capi.SEERA_ERR_INVALID_ARGUMENT
    assert what in lib.seera_hip_last_error().decode(), lib.seera_hip_last_error()


@pytest.mark.parametrize("change,what", [
    ({"rows": -1}, "dims"), ({"cols": -1}, "dims"), ({"cols": 16385, "ldy": 20000, "ldg": 20000}, "above"), ({"act": 2}, "activation"), ({"dtype": 3}, "dtype"),
    ({"ldy": 7}, "row distance"), ({"ldg": 7}, "row distance"), ({"ldy": 1 << 31}, "row distance"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"y": None}, "null"), ({"codes": None}, "null"), ({"scales": None}, "null"), ({"g": P + 2}, "aligned"), ({"codes": P + 8}, "aligned"), ({"scales": P + 2}, "aligned"),
    ({"w2": P + 1}, "aligned")])
def test_norm_refusals(change, what):
    base = dict(y=P, g=P, r=P, w1=P, s=P, w2=P, r_out=P, codes=P, scales=P, rows=2, cols=8, ldy=8, ldg=8, eps=1e-6, act=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_block_norm_fwd_f8", args, what)
    _refused("seera_hip_block_norm_fwd_f8_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"n": -1}, "dims"), ({"k": -1}, "dims"), ({"dtype": 3}, "dtype"), ({"transposed": 2}, "transposed"), ({"ldw": 7}, "ldw"), ({"transposed": 1, "ldw": 8}, "ldw"),
    ({"ldw": 1 << 60}, "ldw"), ({"n": 0x7FFFFFFF, "ldw": 1 << 31}, "too large"), ({"k": 0x7FFFFFFF}, "too large"), ({"n": 1 << 30, "k": 1 << 30, "ldw": 1 << 30}, "too large"),
    ({"w": None}, "null"), ({"codes": None}, "null"), ({"scales": None}, "null"), ({"w": P + 2}, "aligned"), ({"codes": P + 4}, "aligned")])
def test_quantize_refusals(change, what):
    base = dict(w=P, codes=P, scales=P, n=8, k=9, ldw=8, transposed=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_quantize_weights_f8", args, what)
    _refused("seera_hip_quantize_weights_f8_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"M": -1}, "dims"), ({"N": -1}, "dims"), ({"K": -1}, "dims"), ({"dtype": -1}, "dtype"), ({"ldc": 7}, "ldc"), ({"ldc": 1 << 60}, "ldc"),
    ({"M": 0x7FFFFFFF}, "too large"), ({"K": 0x7FFFFFFF}, "too large"), ({"M": 0x7FFFFF00, "N": 1 << 20, "ldc": 1 << 20}, "too large"),
    ({"a": None}, "null"), ({"a_scales": None}, "null"), ({"w": None}, "null"), ({"w_scales": None}, "null"), ({"C": None}, "null"),
    ({"a": P + 8}, "aligned"), ({"w": P + 1}, "aligned"), ({"bias": P + 2}, "aligned"), ({"C": P + 2}, "aligned")])
def test_matmul_refusals(change, what):
    base = dict(a=P, a_scales=P, w=P, w_scales=P, bias=P, C=P, M=4, N=8, K=16, ldc=8, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_matmul_f8", args, what)
    _refused("seera_hip_matmul_f8_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"rows": -1}, "dims"), ({"vocab": -1}, "dims"), ({"vocab": (1 << 22) + 1, "ld": 1 << 23}, "above"), ({"dtype": 5}, "dtype"), ({"ld": 7}, "row distance"),
    ({"ld": 1 << 61}, "too large"), ({"logits": None}, "null"), ({"uniform": None}, "null"), ({"tokens": None}, "null"), ({"logits": P + 1}, "aligned"),
    ({"top_k": P + 2}, "aligned"), ({"logp": P + 2}, "aligned")])
def test_sample_refusals(change, what):
    base = dict(logits=P, uniform=P, temperature=P, top_k=P, top_p=P, min_p=P, tokens=P, logp=P, rows=2, vocab=8, ld=8, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_sample", args, what)
    _refused("seera_hip_sample_async", args + [None], what)


def test_nothing_to_do_needs_no_pointers():
    lib = capi.load()
    for dims in ((0, 8), (2, 0)):
        assert lib.seera_hip_block_norm_fwd_f8_async(*[None] * 9, *dims, 8, 8, 1e-6, 0, 0, None) == capi.SEERA_OK
        assert lib.seera_hip_quantize_weights_f8_async(None, None, None, *dims, 8, 0, 0, None) == capi.SEERA_OK
        assert lib.seera_hip_matmul_f8_async(*[None] * 6, *dims, 16, 8, 0, None) == capi.SEERA_OK
    assert lib.seera_hip_sample_async(*[None] * 8, 0, 8, 8, 0, None) == capi.SEERA_OK
