"""Pins oracle/sequence.py on the CPU before it checks the HIP kernels: the
gradients against central differences of the forward in 64 bits, the recurrence
against its closed form, the 8-bit codes against a table of every code's value,
and planted mistakes that these checks must reject. And the argument checks of
the entry points, which run before any device work."""
import ctypes

import numpy as np
import pytest

from ml_framework_amd import capi
from oracle import sequence as q


def _difference(f, x, direction, step=1e-5):
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


# ---- gated scan ----


def test_scan_closed_form():
    """A constant gate and input: a geometric series."""
    a, n = 0.75, 20
    h, hT, _, _ = q.scan_fwd(np.full((1, n, 1), 2.0), np.full((1, n, 1), a), np.full((1, 1), 5.0), sigmoid=False)
    t = np.arange(1, n + 1)
    assert np.allclose(h[0, :, 0], a**t * 5 + 2 * (1 - a**t) / (1 - a), rtol=1e-14)
    assert hT[0, 0] == h[0, -1, 0]
    f = np.log(a / (1 - a))
    h, _, _, _ = q.scan_fwd(np.full((1, n, 1), 2.0), np.full((1, n, 1), f), np.full((1, 1), 5.0))
    assert np.allclose(h[0, :, 0], a**t * 5 + 2 * (1 - a**t), rtol=1e-14)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("lengths", [None, [5, 0, 3]])
def test_scan_gradients_against_differences(sigmoid, lengths):
    r = np.random.default_rng(3)
    shape = (3, 5, 4)
    x, f, dh = r.standard_normal(shape), r.standard_normal(shape), r.standard_normal(shape)
    h0, dhT = r.standard_normal((3, 4)), r.standard_normal((3, 4))
    n = None if lengths is None else np.array(lengths)
    inside = np.ones(shape, bool) if n is None else np.arange(5)[None, :, None] < n[:, None, None]
    dh = np.where(inside, dh, 0.0)

    def loss(x, f, h0):
        h, hT, _, _ = q.scan_fwd(x, f, h0, n, sigmoid)
        return (h * dh).sum() + (hT * dhT).sum()

    h, _, _, _ = q.scan_fwd(x, f, h0, n, sigmoid)
    got, _ = q.scan_bwd(x, f, h, dh, h0, dhT, n, sigmoid)
    for name, at in (("dx", 0), ("df", 1), ("dh0", 2)):
        args = [x, f, h0]
        d = r.standard_normal(args[at].shape)

        def along(v):
            return loss(*[v if i == at else a for i, a in enumerate(args)])

        want = _difference(along, args[at], d)
        # a central difference of a smooth loss of order 10: h^2 terms and 1e-16 / h
        assert abs((got[name] * d).sum() - want) <= 1e-7 * max(1.0, abs(want)), name
        assert abs((1.01 * got[name] * d).sum() - want) > 1e-7 * max(1.0, abs(want)), "a planted 1% is seen"


# ---- block norm ----


@pytest.mark.parametrize("parts", ["g r w1 s w2", "w2", "r w2", "g w1", "s r", "g s w1 w2"])
@pytest.mark.parametrize("silu", [True, False])
def test_norm_gradients_against_differences(parts, silu):
    r = np.random.default_rng(5)
    rows, cols = 3, 6
    parts = parts.split()
    v = {"y": r.standard_normal((rows, cols))}
    for k in parts:
        v[k] = r.standard_normal((rows, cols) if k in "gr" else cols)
    d_r, d_n = r.standard_normal((rows, cols)), r.standard_normal((rows, cols))

    def fwd(v):
        first = {k: a for k, a in v.items() if k != "w2"}
        out, _ = q.norm_fwd(**first, silu=silu)
        if "w2" in v:
            out.update(q.norm_next(out["r_out"], v["w2"])[0])
        return out

    def loss(v):
        out = fwd(v)
        return (out["r_out"] * d_r).sum() + ((out["n_out"] * d_n).sum() if "w2" in v else 0.0)

    kept = fwd(v)
    got, _ = q.norm_bwd(v["y"], v.get("g"), kept["r_out"], v.get("w1"), v.get("s"), v.get("w2"), kept.get("rstd1"), kept.get("rstd2"),
                        d_r, d_n if "w2" in v else None, silu)
    for k in v:
        d = r.standard_normal(v[k].shape)
        want = _difference(lambda a: loss({**v, k: a}), v[k], d)
        assert abs((got["d" + k] * d).sum() - want) <= 1e-7 * max(1.0, abs(want)), k


# ---- AdamW's codes ----


@pytest.mark.parametrize("top", [15, 31])
def test_codes_keep_their_values(top):
    """Every code's value, in one block with the largest: encoded to itself,
    whatever the random bits, and between two neighbours up or down by them."""
    n = 128 if top == 15 else 256
    every = q.decode(np.arange(n).astype(np.uint8), np.full(-(-n // 128), 127, np.uint8), top)
    assert np.all(np.diff(every) > 0) and every[0] == 0 and every[-1] == 1.875
    for random in (0, 1, 40000, 65535):
        for half in range(n // 128):
            block = every[half * 128:half * 128 + 128].copy()
            if half == 0 and n > 128:
                block[0] = 1.875  # keeps the exponent
            codes, e = q.encode(block, np.full(128, random), top)
            assert e[0] == 127
            want = np.arange(half * 128, half * 128 + 128)
            if half == 0 and n > 128:
                want[0] = n - 1
            assert np.array_equal(codes, want)
    low, high = every[20], every[21]
    block = np.full(128, low + 0.25 * (high - low), np.float32)
    block[0] = 1.875
    codes, _ = q.encode(block, np.arange(128) * 512, top)
    assert np.array_equal(codes[1:] == 21, (np.arange(1, 128) * 512) >= 0.75 * 65536)


def test_codes_refuse_to_lose_a_positive_v_and_mark_what_is_not_finite():
    v = np.full(128, 1e-30, np.float32)
    v[0] = 1.0
    codes, e = q.encode(v, np.zeros(128, np.int64), 31)
    assert codes[0] > 200 and np.all(codes[1:] == 1)
    for planted in (np.inf, np.nan):
        v[5] = planted
        codes, e = q.encode(v, np.zeros(128, np.int64), 31)
        assert e[0] == 255 and np.all(np.isnan(q.decode(codes, e, 31)))


def test_rounding_bits_are_even():
    """The mean and the neighbours' correlation of a million 16-bit draws, to five
    standard deviations."""
    bits = q.rounding_bits(7, 3, 1 << 20)
    for part in (bits & 0xFFFF, bits >> 16):
        u = part / 65536 - 0.5
        assert abs(u.mean()) < 5 / np.sqrt(12 * len(u))
        assert abs((u[1:] * u[:-1]).mean() * 12) < 5 / np.sqrt(len(u))
    assert not np.array_equal(bits, q.rounding_bits(8, 3, 1 << 20))
    assert not np.array_equal(bits, q.rounding_bits(7, 4, 1 << 20))


def test_codes_need_another_seed_in_each_step():
    """A second moment that falls by a thousandth of itself a step, 2000 times: with a
    seed of its own for each step the codes follow, with one for all they stay where
    they are (each value meets the same threshold again and again). The header says so."""
    n, steps = 1280, 2000
    r = np.random.default_rng(5)
    start = (0.5 + r.random(n)).astype(np.float32)
    left = {}
    for fresh in (True, False):
        codes, e = q.encode(start, r.integers(0, 65536, n), 31)
        first = q.decode(codes, e, 31)
        for step in range(steps):
            v = q.decode(codes, e, 31) * np.float32(0.999)
            codes, e = q.encode(v, q.rounding_bits(step if fresh else 7, 0, n) >> 16, 31)
        left[fresh] = (q.decode(codes, e, 31).astype(np.float64) / first).mean()
    # a step moves a code of 8 to 15 places down by one with a chance of a thousandth of them: its
    # value varies by at most 0.001 / 8 of its square, in 2000 steps by exp(0.25) - 1, so that a value
    # deviates by 0.54 of the mean 0.999^2000, and the mean over n by a root of n less
    assert abs(left[True] - 0.999**steps) < 5 * 0.54 * 0.999**steps / np.sqrt(n), left
    assert left[False] > 0.9, left
    header = " ".join(open(capi.HEADER).read().replace(" * ", " ").split())
    assert "as long as each step has another seed" in header


# ---- argument checks ----


def _refused(name, args, what):
    lib = capi.load()
    assert getattr(lib, name)(*args) == capi.SEERA_ERR_INVALID_ARGUMENT, (name, args)
    assert what in lib.seera_hip_last_error().decode(), lib.seera_hip_last_error()


P = 4096  # an aligned address that no check reads


@pytest.mark.parametrize("change,what", [
    ({"batch": -1}, "dims"), ({"time": -1}, "dims"), ({"channels": -2}, "dims"), ({"gate": 2}, "gate"), ({"time_major": 2}, "time_major"),
    ({"dtype": 3}, "dtype"), ({"ldx": 7}, "row distance"), ({"ldf": 7}, "row distance"), ({"ldx": 1 << 41}, "too large"), ({"x": None}, "null"), ({"f": None}, "null"),
    ({"h": None}, "null"), ({"x": P + 1, "dtype": 1}, "aligned"), ({"f": P + 2}, "aligned"), ({"h0": P + 2}, "aligned"), ({"lengths": P + 1}, "aligned")])
def test_scan_refusals(change, what):
    base = dict(x=P, f=P, h0=P, lengths=None, h=P, hT=P, batch=2, time=3, channels=8, ldx=8, ldf=8, gate=1, time_major=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_gated_scan_fwd", args, what)
    _refused("seera_hip_gated_scan_fwd_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"batch": -1}, "dims"), ({"gate": -1}, "gate"), ({"dtype": 9}, "dtype"), ({"lddx": 7}, "row distance"), ({"lddf": 7}, "row distance"),
    ({"x": None}, "null"), ({"h": None}, "null"), ({"dh": None}, "null"), ({"dx": None}, "null"), ({"df": None}, "null"), ({"dx": P + 2}, "aligned")])
def test_scan_bwd_refusals(change, what):
    base = dict(x=P, f=P, h0=P, lengths=None, h=P, dh=P, dhT=P, dx=P, df=P, dh0=P, batch=2, time=3, channels=8, ldx=8, ldf=8, lddx=8, lddf=8,
                gate=1, time_major=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_gated_scan_bwd", args, what)
    _refused("seera_hip_gated_scan_bwd_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"rows": -1}, "dims"), ({"cols": -1}, "dims"), ({"cols": 16385, "ldy": 20000, "ldg": 20000}, "above"), ({"act": 2}, "activation"), ({"dtype": 3}, "dtype"),
    ({"ldy": 7}, "row distance"), ({"ldg": 7}, "row distance"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"y": None}, "null"),
    ({"n_out": None}, "null"), ({"w2": None}, "n_out needs w2"), ({"w2": None, "n_out": None, "r_out": None}, "null"), ({"g": P + 2}, "aligned")])
def test_norm_refusals(change, what):
    base = dict(y=P, g=P, r=P, w1=P, s=P, w2=P, r_out=P, n_out=P, rstd1=P, rstd2=P, rows=2, cols=8, ldy=8, ldg=8, eps=1e-6, act=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_block_norm_fwd", args, what)
    _refused("seera_hip_block_norm_fwd_async", args + [None], what)


@pytest.mark.parametrize("change,what", [
    ({"rows": -1}, "dims"), ({"cols": 16385}, "above"), ({"act": 2}, "activation"), ({"lddy": 7}, "row distance"), ({"lddg": 7}, "row distance"),
    ({"y": None}, "null"), ({"r_out": None}, "null"), ({"rstd1": None}, "null"), ({"rstd2": None}, "null"), ({"dn": None}, "null"), ({"w2": None}, "dn needs w2"),
    ({"w2": None, "dn": None, "dr_out": None}, "null"), ({"dy": None}, "null"), ({"dg": None}, "null"), ({"dw1": None}, "null"), ({"ds": None}, "null"),
    ({"dw2": None}, "null")])
def test_norm_bwd_refusals(change, what):
    base = dict(y=P, g=P, r_out=P, w1=P, s=P, w2=P, rstd1=P, rstd2=P, dr_out=P, dn=P, dy=P, dg=P, dr=P, dw1=P, ds=P, dw2=P, rows=2, cols=8,
                ldy=8, ldg=8, lddy=8, lddg=8, act=0, dtype=0)
    args = list({**base, **change}.values())
    _refused("seera_hip_block_norm_bwd", args, what)
    _refused("seera_hip_block_norm_bwd_async", args + [None], what)


def _tensor(**change):
    base = dict(param=P, grad=P, m=P, v=P, m_exp=P, v_exp=P, count=5, state_bits=32)
    return (capi.AdamwTensor * 1)(capi.AdamwTensor(**{**base, **change}))


@pytest.mark.parametrize("change,what", [
    ({"count": -1}, "negative count"), ({"state_bits": 16}, "state_bits"), ({"grad_dtype": 4}, "grad_dtype"), ({"param16": P, "param16_dtype": 0}, "param16_dtype"),
    ({"weight_decay": float("inf")}, "weight_decay"), ({"param": None}, "null"), ({"grad": None}, "null"), ({"m": None}, "null"), ({"v": None}, "null"),
    ({"state_bits": 8, "m_exp": None}, "null"), ({"state_bits": 8, "v_exp": None}, "null"), ({"param": P + 2}, "aligned"), ({"m": P + 1}, "aligned")])
def test_adamw_refuses_tensors(change, what):
    _refused("seera_hip_adamw_step", (_tensor(**change), 1, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None), what)


@pytest.mark.parametrize("change,what", [
    ({"n": -1}, "number of tensors"), ({"tensors": None}, "null array"), ({"lr": float("nan")}, "lr"), ({"beta1": 1.0}, "betas"), ({"beta2": -0.1}, "betas"),
    ({"eps": -1e-8}, "eps"), ({"step": 0}, "counts from 1"), ({"scale": P + 1}, "aligned")])
def test_adamw_refuses_constants(change, what):
    base = dict(tensors=_tensor(), n=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, seed=0, scale=None)
    _refused("seera_hip_adamw_step", list({**base, **change}.values()), what)
    _refused("seera_hip_adamw_step_async", list({**base, **change}.values()) + [None], what)


def test_adamw_tensor_layout():
    """The ctypes structure, field by field, against the header's (natural alignment,
    no padding): a host buffer of the same layout may stand for an array of them."""
    names = ["param", "grad", "m", "v", "m_exp", "v_exp", "param16", "count", "weight_decay", "grad_dtype", "param16_dtype", "state_bits", "reserved"]
    offsets = [8 * i for i in range(9)] + [72, 76, 80, 84]
    assert [getattr(capi.AdamwTensor, n).offset for n in names] == offsets and ctypes.sizeof(capi.AdamwTensor) == 88
    body = open(capi.HEADER).read().split("typedef struct seera_adamw_tensor {")[1].split("}")[0]
    assert [line.split()[-1].strip("*;") for line in body.strip().splitlines()] == names


def test_adamw_values_refusals():
    two = (ctypes.c_void_p * 1)(P)
    _refused("seera_hip_adamw_state_values", (_tensor(), 1, None, two), "null array")
    _refused("seera_hip_adamw_state_values", (_tensor(), 1, two, (ctypes.c_void_p * 1)(P + 2)), "aligned")


def test_sizes_that_no_launch_reaches_are_refused():
    for time in (1, 20, 500):
        _refused("seera_hip_gated_scan_fwd_async", (P, P, P, None, P, P, 1 << 30, time, 2048, 2048, 2048, 1, 0, 0, None), "too large")
        _refused("seera_hip_gated_scan_bwd_async", (P, P, P, None, P, P, P, P, P, P, 1 << 30, time, 2048, *[2048] * 4, 1, 0, 0, None), "too large")
    _refused("seera_hip_gated_scan_fwd_async", (P, P, P, None, P, P, 2, (1 << 30) + 1, 8, 8, 8, 1, 0, 0, None), "time")
    _refused("seera_hip_adamw_step_async", (_tensor(count=1 << 50), 1, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None, None), "too large")


def test_a_grid_that_rounds_up_to_the_limit_is_refused():
    """A scan's grid is a multiple of eight blocks: the last few counts below a
    launch's limit round up to it."""
    for batch in ((1 << 25) - 1, (1 << 25) - 7):
        _refused("seera_hip_gated_scan_fwd_async", (P, P, P, None, P, P, batch, 20, 2, 2, 2, 1, 0, 2, None), "too large")


def test_a_refused_step_has_moved_no_tensor():
    """The last of more tensors than one launch takes is too large: the call is
    refused before any launch (here, without a device, a launch is another error)."""
    many = (capi.AdamwTensor * 60)(*[_tensor()[0]] * 59, _tensor(count=1 << 50)[0])
    _refused("seera_hip_adamw_step_async", (many, 60, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None, None), "tensor 59 is too large")
    outs = (ctypes.c_void_p * 60)(*[P] * 60)
    _refused("seera_hip_adamw_state_values_async", (many, 60, outs, outs, None), "tensor 59 is too large")


def test_a_linear_scans_backward_asks_nothing_of_x():
    """x is not read there, so that its row distance is not looked at either."""
    for ldx in (0, -1, 1 << 62):
        args = (None, P, None, None, P, P, None, P, P, None, 0, 3, 8, ldx, 8, 8, 8)
        assert capi.load().seera_hip_gated_scan_bwd_async(*args, capi.SEERA_GATE_LINEAR, 0, 0, None) == capi.SEERA_OK
        _refused("seera_hip_gated_scan_bwd_async", (*args, capi.SEERA_GATE_SIGMOID, 0, 0, None), "row distance")


def test_nothing_to_do_needs_no_pointers():
    lib = capi.load()
    for dims in ((0, 3, 8), (2, 3, 0)):
        assert lib.seera_hip_gated_scan_fwd_async(None, None, None, None, None, None, *dims, 8, 8, 1, 0, 0, None) == capi.SEERA_OK
    assert lib.seera_hip_block_norm_fwd_async(*[None] * 10, 0, 8, 8, 8, 1e-6, 0, 0, None) == capi.SEERA_OK
    assert lib.seera_hip_adamw_step_async(None, 0, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None, None) == capi.SEERA_OK
