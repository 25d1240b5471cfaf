"""The operators that a model answers with (block norm in 8 bits, weights in 8
bits, their product, sampling) from their formulas, in 64 bits but for what is
defined by fp32 operations (a scale and a code's quotient, which are compared bit
by bit).

Bounds count roundings as in oracle/sequence.py. An e4m3 code is nearest to its
quotient: off by at most 2^-4 of it, or by 2^-10 below the smallest normal value.
"""
from __future__ import annotations

import math

import numpy as np

from .sequence import U, norm_next

BLOCK, LARGEST = 128, 448.0


def padded(k):
    return -(-k // BLOCK) * BLOCK


def decode(codes):
    """e4m3 codes as 64-bit values: s eeee mmm, bias 7, denormals, 0x7f is NaN."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, np.ldexp(8.0 + m, e - 10), np.ldexp(1.0 * m, -9))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


_VALUES = decode(np.arange(127))


def encode(v):
    """The nearest code, ties to the even one; |v| is at most 464."""
    a = np.abs(np.asarray(v, np.float64))
    hi = np.clip(np.searchsorted(_VALUES, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _VALUES[hi] - a, a - _VALUES[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def scales_of(largest):
    """fp32, from blocks' largest magnitudes."""
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(np.isfinite(largest), np.float32(largest) / np.float32(LARGEST), np.float32(np.nan)).astype(np.float32)


def _codes(v, scale):
    """v, scale: fp32. The quotient is rounded to fp32, then to a code."""
    with np.errstate(divide="ignore", invalid="ignore"):
        quotient = np.where(scale > 0, v / scale, np.float32(0) * v)
    return encode(quotient)


def quantize_rows(v):
    """Codes [rows][kp] and scales [rows][kp / 128] of fp32 values (finite ones: codes
    under a scale of NaN stand for nothing)."""
    rows, k = v.shape
    whole = np.zeros((rows, padded(k)), np.float32)
    whole[:, :k] = v
    blocks = whole.reshape(rows, -1, BLOCK)
    scales = scales_of(np.abs(blocks).max(2))
    return _codes(blocks, scales[..., None]).reshape(rows, -1), scales


def quantize_weights(w):
    """The same with a scale for each 128 x 128; w [n, k] fp32."""
    n, k = w.shape
    whole = np.zeros((padded(n), padded(k)), np.float32)
    whole[:n, :k] = w
    blocks = whole.reshape(padded(n) // BLOCK, BLOCK, -1, BLOCK)
    scales = scales_of(np.abs(blocks).max((1, 3)))
    return _codes(blocks, scales[:, None, :, None]).reshape(padded(n), -1)[:n], scales


def norm_values(kept, w2, eps):
    """n and its bound, from r_out as it was stored."""
    if w2 is None:
        return kept, np.zeros_like(kept)
    out, bound = norm_next(kept, w2, eps)
    return out["n_out"], bound["n_out"]


def check_codes(codes, scales, n, bound):
    """That codes and scales are those of values within `bound` of n (rows of k)."""
    rows, k = n.shape
    kp = padded(k)
    assert codes.shape == (rows, kp) and scales.shape == (rows, kp // BLOCK)
    assert not np.any(codes[:, k:]), "padding"
    v, b = np.zeros((rows, kp)), np.zeros((rows, kp))
    v[:, :k], b[:, :k] = n, bound
    v, b, got = (x.reshape(rows, -1, BLOCK) for x in (v, b, decode(codes)))
    largest, off = np.abs(v).max(2), b.max(2)
    # a maximum moves by no more than its candidates; the division rounds once
    assert np.all(np.abs(scales * LARGEST - largest) <= off + 2 * U * largest + 2.0**-140), "scales"
    s = np.where(scales > 0, scales, 1.0)[..., None].astype(np.float64)
    quotient = v / s
    slack = b / s + 4 * U * np.abs(quotient)
    half = np.maximum(2.0**-4 * (np.abs(quotient) + slack), 2.0**-10)
    assert np.all(np.abs(got - quotient) <= half * (1 + 2.0**-20) + slack), "codes"


def matmul(a, a_scales, w, w_scales, bias=None, fp32=True):
    """C and its bound, from codes and scales. A block's 128 products are exact; their
    sum is taken as 127 additions off by at most a unit in the last place (2 U) of
    the sum of their magnitudes, then two products and a sum for each block, the sums
    of all blocks, and the bias. Results that are kept in 16 bits (fp32 False) come
    from an instruction that cuts each product below 2^-13 of the largest of its group of 8
    along K: seven of them by less than that, with the largest at most the
    product of the groups' largest factors. (Lanes hold 16 consecutive codes twice, so
    that its groups of 8 are consecutive here.)"""
    m, kp = a.shape
    n = w.shape[0]
    A, W = decode(a), decode(w)
    blocks = kp // BLOCK
    c, size, cut = np.zeros((m, n)), np.zeros((m, n)), np.zeros((m, n))
    for b in range(blocks):
        x, y = A[:, b * BLOCK:(b + 1) * BLOCK], W[:, b * BLOCK:(b + 1) * BLOCK]
        s = a_scales[:, b].astype(np.float64)[:, None] * np.repeat(w_scales[:, b].astype(np.float64), BLOCK)[None, :n]
        c += (x @ y.T) * s
        size += (np.abs(x) @ np.abs(y).T) * s
        if not fp32:
            cut += np.abs(x).reshape(m, -1, 8).max(2) @ np.abs(y).reshape(n, -1, 8).max(2).T * s
    bound = size * (2 * BLOCK + 2 + blocks) * U + 7 * 2.0**-13 * cut
    if bias is not None:
        c = c + bias
        bound = bound + np.abs(c) * U
    return c, bound


ONE = 1 << 40


def weights(l, temperature):
    """Whole multiples of 2^-40, as Python integers in an object array."""
    top = l.max()
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l == top, 0.0, (l - top) / temperature)
        w = np.rint(np.exp(z) * ONE)
    return np.where(np.isnan(w) | (l == -np.inf), 0, w).astype(np.int64)


def sample_row(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logp, how near u of the total is to the nearest border, as a share of the
    total) of one row of 64-bit logits."""
    l = np.where(np.isnan(l), -np.inf, l) + 0.0
    if l.size == 0 or l.max() == -np.inf:
        return -1, -np.inf, 1.0
    if not temperature > 0:
        return int(l.argmax()), 0.0, 1.0
    w = weights(l, temperature)
    order = np.argsort(-l, kind="stable")
    ranked = w[order]
    if 0 < top_k < l.size:
        ranked = ranked[:top_k]
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(ranked)[:-1]])  # sums of at most 2^22 weights of 2^40: inside 2^63
        share = max(1, math.ceil(max(float(top_p), 0.0) * float(ranked.sum())))
        ranked = ranked[:int((before < share).sum())]
    keep = np.zeros(l.size, bool)
    keep[order[:len(ranked)]] = True
    if min_p > 0:
        with np.errstate(invalid="ignore"):
            d = np.where(l == l.max(), 0.0, l - l.max())
            keep &= np.exp(d / temperature) >= min(min_p, 1.0)
    kept = np.where(keep, w, 0)
    mass = np.cumsum(kept)
    total = int(mass[-1])
    u = 0.0 if not u > 0 else min(float(u), 1.0)
    at = min(total - 1, int(u * float(total)))
    token = int(np.searchsorted(mass, at, side="right"))
    near = np.abs(mass.astype(np.float64) - u * total).min() / total
    logp = (0.0 if l[token] == l.max() else (l[token] - l.max()) / temperature) - math.log(total / ONE)
    return token, logp, near
