"""The sequence model's operators (gated scan, block norm, AdamW) in 64 bits,
from their formulas, with bounds on what 32-bit arithmetic may differ by.

Every array is numpy. ``u`` is fp32's unit roundoff. The bounds count
roundings: a term that passes through k of them is off by at most k u of
itself, so a bound is the same sum over magnitudes, each term weighted by its
count. A gate from a 32-bit sigmoid is off by (4 + 2 |f|) u of itself: the
exponential's argument is rounded (|f| u), then exponential, sum, reciprocal
and product.
"""
from __future__ import annotations

import numpy as np

U = 2.0**-24
F32, F16, BF16 = 0, 1, 2
HALF_ULP = {F32: U, F16: 2.0**-11, BF16: 2.0**-8}  # of 24, 11 and 8 significant bits
TINY = {F32: 2.0**-149, F16: 2.0**-25, BF16: 2.0**-134}  # the smallest spacing, halved for the 16-bit types


def store(a, dtype):
    """Values as their bytes in memory."""
    a = np.asarray(a, np.float32)
    if dtype == F32:
        return a
    if dtype == F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    bits = a.view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), out)


def load(a, dtype):
    """Bytes in memory as 64-bit values."""
    if dtype == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(dtype):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[dtype]


def rounding(ref, dtype):
    """What storing a value in `dtype` may add to its error."""
    return HALF_ULP[dtype] * np.abs(ref) * 1.01 + TINY[dtype]


# ---- gated scan: x, f, h ... [batch, time, channels] ----


def gates(f, sigmoid):
    """a, 1 - a, and how many u of itself each may be off."""
    if not sigmoid:
        return f, np.ones_like(f), np.zeros_like(f)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-f)), 1 / (1 + np.exp(f)), 4 + 2 * np.minimum(np.abs(f), 104)


def _lengths(lengths, batch, time):
    return np.full(batch, time) if lengths is None else np.clip(lengths, 0, time)


def scan_fwd(x, f, h0=None, lengths=None, sigmoid=True):
    """h, hT and their bounds."""
    batch, time, channels = x.shape
    n = _lengths(lengths, batch, time)
    h, bound = np.zeros_like(x), np.zeros_like(x)
    state = np.zeros((batch, channels)) if h0 is None else h0.astype(np.float64)
    size, weighed = np.abs(state), np.zeros_like(state)  # sum of |terms|; the same, each by its roundings
    for t in range(time):
        live = (n > t)[:, None]
        xt, ft = np.where(live, x[:, t], 0.0), np.where(live, f[:, t], 0.0)
        a, rest, off = gates(ft, sigmoid)
        b = rest * xt
        new = a * state + b
        # a product with a, then a sum; the span's gates may be multiplied first
        w = np.abs(a) * (weighed + (2 + off) * size) + (3 + off) * np.abs(b)
        z = np.abs(a) * size + np.abs(b)
        state, size, weighed = np.where(live, new, state), np.where(live, z, size), np.where(live, w, weighed)
        h[:, t], bound[:, t] = np.where(live, state, 0.0), np.where(live, weighed, 0.0)
    return h, state, bound * U, weighed * U


def scan_bwd(x, f, h, dh, h0=None, dhT=None, lengths=None, sigmoid=True):
    """{dx, df, dh0} and their bounds."""
    batch, time, channels = f.shape
    n = _lengths(lengths, batch, time)
    out = {k: np.zeros_like(f) for k in ("dx", "df")}
    bound = {k: np.zeros_like(f) for k in ("dx", "df")}
    first = np.zeros((batch, channels)) if h0 is None else h0.astype(np.float64)
    carry = np.zeros((batch, channels)) if dhT is None else dhT.astype(np.float64)
    size, weighed = np.abs(carry), np.zeros_like(carry)
    for t in reversed(range(time)):
        live = (n > t)[:, None]
        ft, dt = np.where(live, f[:, t], 0.0), np.where(live, dh[:, t], 0.0)
        before = h[:, t - 1] if t else first
        a, rest, off = gates(ft, sigmoid)
        g = dt + carry
        gw = weighed + size + np.abs(dt)
        gz = size + np.abs(dt)
        if sigmoid:
            other = before - np.where(live, x[:, t], 0.0)
            dx, df = g * rest, g * rest * other * a
            bx, bf = rest * (gw + (2 + off) * gz), rest * np.abs(other) * a * (gw + (6 + 2 * off) * gz)
        else:
            dx, df = g, g * before
            bx, bf = gw, np.abs(before) * (gw + 2 * gz)
        for k, v, w in (("dx", dx, bx), ("df", df, bf)):
            out[k][:, t], bound[k][:, t] = np.where(live, v, 0.0), np.where(live, w, 0.0) * U
        carry = np.where(live, a * g, carry)
        weighed = np.where(live, np.abs(a) * (gw + (2 + off) * gz), weighed)
        size = np.where(live, np.abs(a) * gz, size)
    out["dh0"], bound["dh0"] = carry, weighed * U
    return out, bound


# ---- block norm: rows of cols ----


def act(g, silu):
    """The activation, its slope, and how many u of their magnitudes they may be off."""
    with np.errstate(over="ignore"):
        q = 1 / (1 + np.exp(-g))
    off = 8 + 2 * np.minimum(np.abs(g), 104)
    if silu:
        return g * q, q * (1 + g * (1 - q)), off, q * (1 + np.abs(g))
    return q, q * (1 - q), off, q


def _sum_roundings(cols):
    """Roundings that a value passes in a sum over a row or over rows: at most
    64 in a thread's own chain, then a tree and the mean's division."""
    return 64 + 32


def norm_fwd(y, g=None, r=None, w1=None, s=None, eps=1e-6, silu=True):
    """{r_out, rstd1} and their bounds (before a 16-bit output's own rounding)."""
    k = _sum_roundings(y.shape[1])
    out, bound = {}, {}
    u, off = y, np.zeros_like(y)
    if w1 is not None:
        rstd = 1 / np.sqrt((y * y).mean(1) + eps)
        out["rstd1"], bound["rstd1"] = rstd, rstd * (k / 2 + 4) * U
        u, off = y * rstd[:, None] * w1, off + k / 2 + 6
    if g is not None:
        a, _, more, _ = act(g, silu)
        u, off = u * a, off + more + 1
    if s is not None:
        u, off = u * s, off + 1
    out["r_out"] = u if r is None else u + r
    bound["r_out"] = (np.abs(u) * off + np.abs(out["r_out"])) * U
    return out, bound


def norm_next(kept, w2, eps=1e-6):
    """{n_out, rstd2} and their bounds, of the residual stream as it was stored."""
    k = _sum_roundings(kept.shape[1])
    rstd = 1 / np.sqrt((kept * kept).mean(1) + eps)
    n = kept * rstd[:, None] * w2
    return {"n_out": n, "rstd2": rstd}, {"n_out": np.abs(n) * (k / 2 + 8) * U, "rstd2": rstd * (k / 2 + 4) * U}


def norm_bwd(y, g=None, r_out=None, w1=None, s=None, w2=None, rstd1=None, rstd2=None, dr_out=None, dn=None, silu=True):
    """{dy, dg, dr, dw1, ds, dw2} and their bounds (before a 16-bit output's own
    rounding), from the statistics that the forward saved."""
    shape = y.shape
    k = _sum_roundings(shape[1])
    out, bound = {}, {}
    d = np.zeros(shape) if dr_out is None else dr_out
    off = np.zeros(shape)  # bound of d, in u
    if w2 is not None:
        hat = r_out * rstd2[:, None]
        q = dn * w2
        mean, size = (q * hat).mean(1, keepdims=True), np.abs(q * hat).mean(1, keepdims=True)
        out["dw2"] = (dn * hat).sum(0)
        bound["dw2"] = np.abs(dn * hat).sum(0) * (k + 4)
        term = rstd2[:, None] * (q - hat * mean)
        off = rstd2[:, None] * (4 * np.abs(q) + np.abs(hat) * size * (k + 8)) + np.abs(d + term)
        d = d + term
    out["dr"], bound["dr"] = d, off
    hat = y if w1 is None else y * rstd1[:, None]
    z = hat if w1 is None else hat * w1
    a, slope, more, slope_size = act(g, silu) if g is not None else (np.ones(shape), None, np.zeros(shape), None)
    if s is not None:
        out["ds"] = (d * z * a).sum(0)
        bound["ds"] = (np.abs(z * a) * (off + np.abs(d) * (k + 6 + more))).sum(0)
        d, off = d * s, np.abs(s) * (off + np.abs(d))
    if g is not None:
        out["dg"] = d * z * slope
        bound["dg"] = np.abs(z) * slope_size * (off + np.abs(d) * (8 + more))
        d, off = d * a, np.abs(a) * (off + np.abs(d) * (1 + more))
    if w1 is not None:
        out["dw1"] = (d * hat).sum(0)
        bound["dw1"] = (np.abs(hat) * (off + np.abs(d) * (k + 4))).sum(0)
        q, qoff = d * w1, np.abs(w1) * (off + np.abs(d))
        mean = (q * hat).mean(1, keepdims=True)
        moff = (np.abs(hat) * (qoff + np.abs(q) * (k + 4))).mean(1, keepdims=True)
        r1 = rstd1[:, None]
        d, off = r1 * (q - hat * mean), r1 * (qoff + 3 * np.abs(q) + np.abs(hat) * (moff + 5 * np.abs(mean)))
    out["dy"], bound["dy"] = d, off
    return out, {name: b * U for name, b in bound.items()}


# ---- AdamW ----

BLOCK = 128


def mix(x):
    x = np.asarray(x, np.uint32)
    x = x ^ (x >> np.uint32(16))
    x = x * np.uint32(0x6A09E667)
    x = x ^ (x >> np.uint32(15))
    x = x * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def rounding_bits(seed, tensor, count):
    """The 32 random bits of each of a tensor's values: the low half rounds m,
    the high half v."""
    with np.errstate(over="ignore"):
        key = mix(np.uint32(tensor) * np.uint32(0x9E3779B9) + np.uint32(seed))
        return mix(np.arange(count, dtype=np.uint32) * np.uint32(0x9E3779B9) + key)


def _blocks(a):
    pad = -len(a) % BLOCK
    return np.concatenate([a, np.zeros(pad, a.dtype)]).reshape(-1, BLOCK)


def encode(value, random16, top):
    """Codes and block exponents of fp32 values: the definition, in whole numbers
    (ticks of the code's last place, 2^20 to one) and Python's exact powers."""
    value = np.asarray(value, np.float32)
    a = _blocks(np.abs(value)).astype(np.float64)
    finite = np.isfinite(a).all(1)
    a = np.where(finite[:, None], a, 0.0)
    largest = a.max(1)
    e = np.where(largest > 0, np.frexp(largest)[1] - 1, -127)
    e = np.where(largest > 1.875 * np.exp2(e), e + 1, e)
    e = np.maximum(e, -127)
    own = np.where(a > 0, np.frexp(a)[1] - 1, -2000)
    low = (e + 1 - top)[:, None]
    power = np.maximum(own, low)
    ticks = np.rint(np.ldexp(a, 23 - power))  # of 2^(power - 23): exact but below the smallest power
    n = (ticks.astype(np.int64) + 16 * _blocks(random16.astype(np.int64))) >> 20
    code = (power - low) * 8 + n
    if top == 31:
        code = np.where(a > 0, np.maximum(code, 1), code)
    code = np.minimum(code, 127 if top == 15 else 255).reshape(-1)[:len(value)]
    if top == 15:
        code = code + np.where(value < 0, 128, 0)
    return code.astype(np.uint8), np.where(finite, e + 127, 255).astype(np.uint8)


def decode(codes, exponents, top):
    c = codes.astype(np.int64)
    size = c & 127 if top == 15 else c
    field = size >> 3
    value = np.ldexp(((size & 7) + np.where(field > 0, 8, 0)).astype(np.float64), np.maximum(field, 1) - top - 3)
    e = np.repeat(exponents.astype(np.int64), BLOCK)[:len(codes)]
    value = np.where(e == 255, np.nan, np.ldexp(value, e - 127))
    return np.where((c >= 128) & (top == 15), -value, value).astype(np.float32)


def adamw_moments(m, v, grad, scale, beta1, beta2):
    """The moments in fp32, one rounding an operation, as they are rounded to codes."""
    one = np.float32
    g = grad.astype(np.float32) * one(scale)
    m = m * one(beta1) + g * one(1 - beta1)
    v = v * one(beta2) + (g * g) * one(1 - beta2)
    return m, v


def adamw(p, m, v, grad, scale, lr, beta1, beta2, eps, weight_decay, step):
    """p, m, v after the step in 64 bits, and p's bound."""
    g = grad.astype(np.float64) * np.float64(np.float32(scale))
    m = beta1 * m.astype(np.float64) + (1 - beta1) * g
    v = beta2 * v.astype(np.float64) + (1 - beta2) * g * g
    update = lr * (m / (1 - beta1**step)) / (np.sqrt(v / (1 - beta2**step)) + eps)
    p64 = p.astype(np.float64) * (1 - lr * weight_decay) - update
    # m: three roundings over magnitudes that may cancel; v has no cancellation
    size = lr * (np.abs(beta1 * m) + np.abs(g)) / (1 - beta1**step) / (np.sqrt(v / (1 - beta2**step)) + eps)
    return p64, m, v, (3 * np.abs(p.astype(np.float64)) + 16 * (np.abs(update) + size)) * U
