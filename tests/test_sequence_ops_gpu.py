"""The gated scan, the block norm and the AdamW step on the GPU against
oracle/sequence.py (64 bits), at the sizes, layouts and values where they can go
wrong. Tolerances are the oracle's bounds, which count roundings; they were
derived before the first run. Outputs lie in buffers of a byte pattern with room
after each row and at the end, which has to be intact afterwards."""
import ctypes

import numpy as np
import pytest

from ml_framework_amd import capi
from ml_framework_amd.capi import DeviceBuffer
from oracle import sequence as q

pytestmark = pytest.mark.gpu

DTYPES = [q.F32, q.F16, q.BF16]
FILL = 0xA5


@pytest.fixture(scope="module")
def lib():
    assert capi.gpu_available(), "no HIP device visible"
    return capi.load()


@pytest.fixture
def stream(lib):
    st = ctypes.c_void_p()
    capi.check(lib.seera_hip_stream_create(ctypes.byref(st)))
    yield st.value
    lib.seera_hip_stream_destroy(st.value)


class Rows:
    """A device matrix of `dtype` with rows `ld` apart from element `shift` on."""

    def __init__(self, shape, dtype, ld=None, shift=0, data=None, hole=None):
        self.rows, self.cols, self.dtype, self.shift = int(np.prod(shape[:-1])), shape[-1], dtype, shift
        self.shape, self.ld = shape, ld or shape[-1]
        self.size = np.dtype(q.storage(dtype)).itemsize
        whole = np.full((shift + self.rows * self.ld + 64) * self.size, FILL, np.uint8).view(q.storage(dtype))
        if hole is not None:
            whole[:] = q.store(np.full(1, hole), dtype)[0]
        if data is not None:
            self._view(whole)[:] = q.store(data, dtype).reshape(self.rows, self.cols)
        self.buf = DeviceBuffer.from_array(whole)
        self.ptr = self.buf.ptr + shift * self.size

    def _view(self, whole):
        return whole[self.shift:self.shift + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def raw(self):
        """The stored values; everything around them must be untouched."""
        whole = self.buf.to_array(self.buf.nbytes // self.size, q.storage(self.dtype))
        got = self._view(whole).copy()
        self._view(whole)[:] = np.full(self.cols * self.size, FILL, np.uint8).view(q.storage(self.dtype))
        assert np.all(whole.view(np.uint8) == FILL), "written outside of the matrix"
        return got.reshape(self.shape)

    def values(self):
        return q.load(self.raw(), self.dtype)


def _seen(data, dtype):
    """Values as the device has them."""
    return q.load(q.store(data, dtype), dtype)


def _close(got, ref, bound, dtype, what):
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what + ": NaN in other places"
    ok = np.isfinite(ref)
    assert np.array_equal(got[~ok & ~np.isnan(ref)], ref[~ok & ~np.isnan(ref)]), what + ": infinities"
    off = np.abs(got[ok] - ref[ok])
    tol = bound[ok] + (q.rounding(ref, dtype)[ok] if dtype != q.F32 else q.TINY[q.F32])
    worst = np.argmax(off - tol) if off.size else 0
    assert np.all(off <= tol), f"{what}: off by {off[worst]:.3e}, bound {tol[worst]:.3e}, value {ref[ok][worst]:.3e}"


# ---- gated scan ----


def _scan_data(batch, time, channels, dtype, sigmoid, seed, dead=None):
    r = np.random.default_rng(seed)
    shape = (batch, time, channels)
    f = r.standard_normal(shape) + np.linspace(-2, 5, channels)
    if not sigmoid:
        f = np.tanh(f) * 0.999
    start = r.random((batch, time, 1)) < 0.02
    f = np.where(start, -np.inf if sigmoid else 0.0, f)
    d = {"x": _seen(r.standard_normal(shape), dtype), "f": _seen(f, dtype), "dh": _seen(r.standard_normal(shape), dtype),
         "h0": r.standard_normal((batch, channels)).astype(np.float32), "dhT": r.standard_normal((batch, channels)).astype(np.float32)}
    return d


def _order(a, time_major):
    return np.ascontiguousarray(a.transpose(1, 0, 2)) if time_major else a


def _scan_forward(lib, d, dtype, sigmoid, lengths=None, time_major=False, gap=0, shift=0, h0=True, hT=True, stream=None, in_place=False):
    batch, time, channels = d["x"].shape
    shape = (time, batch, channels) if time_major else (batch, time, channels)
    x, f = (Rows(shape, dtype, channels + gap, shift, _order(d[k], time_major), hole=np.nan) for k in ("x", "f"))
    h = Rows(shape, dtype, shift=shift)
    first = DeviceBuffer.from_array(d["h0"])
    n = DeviceBuffer.from_array(np.asarray(lengths, np.int32)) if lengths is not None else None
    last = first if in_place else DeviceBuffer(d["h0"].nbytes)
    args = (x.ptr, f.ptr, first.ptr if h0 else None, n.ptr if n else None, h.ptr, last.ptr if hT else None, batch, time, channels,
            channels + gap, channels + gap, int(sigmoid), int(time_major), dtype)
    if stream is None:
        capi.call("seera_hip_gated_scan_fwd", *args)
    else:
        capi.call("seera_hip_gated_scan_fwd_async", *args, stream)
        capi.check(lib.seera_hip_stream_synchronize(stream))
    return _order(h.values(), time_major), last.to_array(d["h0"].shape) if hT else None


def _scan_backward(lib, d, h, dtype, sigmoid, lengths=None, time_major=False, gap=0, shift=0, h0=True, dhT=True, stream=None):
    batch, time, channels = d["x"].shape
    shape = (time, batch, channels) if time_major else (batch, time, channels)
    x, f = (Rows(shape, dtype, channels + gap, shift, _order(d[k], time_major), hole=np.nan) for k in ("x", "f"))
    kept, dh = Rows(shape, dtype, None, shift, _order(h, time_major)), Rows(shape, dtype, None, shift, _order(d["dh"], time_major))
    dx, df = (Rows(shape, dtype, channels + gap, shift) for _ in range(2))
    first, last, dh0 = DeviceBuffer.from_array(d["h0"]), DeviceBuffer.from_array(d["dhT"]), DeviceBuffer(d["h0"].nbytes)
    n = DeviceBuffer.from_array(np.asarray(lengths, np.int32)) if lengths is not None else None
    ld = channels + gap
    args = (x.ptr if sigmoid else None, f.ptr, first.ptr if h0 else None, n.ptr if n else None, kept.ptr, dh.ptr, last.ptr if dhT else None, dx.ptr, df.ptr,
            dh0.ptr, batch, time, channels, ld, ld, ld, ld, int(sigmoid), int(time_major), dtype)
    if stream is None:
        capi.call("seera_hip_gated_scan_bwd", *args)
    else:
        capi.call("seera_hip_gated_scan_bwd_async", *args, stream)
        capi.check(lib.seera_hip_stream_synchronize(stream))
    return {"dx": _order(dx.values(), time_major), "df": _order(df.values(), time_major), "dh0": dh0.to_array(d["h0"].shape).astype(np.float64)}


def _check_scan(lib, batch, time, channels, dtype, sigmoid, seed=1, lengths=None, poison=False, **kw):
    d = _scan_data(batch, time, channels, dtype, sigmoid, seed)
    if poison:  # rows that a length leaves out hold anything
        out = np.arange(time)[None, :, None] >= np.clip(lengths, 0, time)[:, None, None]
        for k, v in (("x", np.nan), ("f", np.inf), ("dh", np.nan)):
            d[k] = np.where(out, v, d[k])
    n = None if lengths is None else np.asarray(lengths)
    first = d["h0"].astype(np.float64) if kw.get("h0", True) else None
    ref, last, bound, last_bound = q.scan_fwd(d["x"], d["f"], first, n, sigmoid)
    got, got_last = _scan_forward(lib, d, dtype, sigmoid, lengths, **{k: v for k, v in kw.items() if k != "dhT"})
    _close(got, ref, bound, dtype, "h")
    if got_last is not None:
        _close(got_last.astype(np.float64), last, last_bound + 1e-7 * np.abs(last), q.F32, "hT")
    back = {k: v for k, v in kw.items() if k not in ("hT", "in_place")}
    kept = _seen(np.where(np.isnan(ref), 0, ref), dtype)
    if poison:
        kept = np.where(out, np.nan, kept)
    refs, bounds = q.scan_bwd(d["x"], d["f"], kept, d["dh"], first, d["dhT"] if kw.get("dhT", True) else None, n, sigmoid)
    gots = _scan_backward(lib, d, kept, dtype, sigmoid, lengths, **back)
    for k in refs:
        _close(gots[k], refs[k], bounds[k], q.F32 if k == "dh0" else dtype, k)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,time,channels", [(1, 1, 1), (3, 1, 64), (2, 2, 33), (1, 7, 130), (2, 31, 64), (3, 129, 65), (2, 300, 96), (1, 1025, 40), (5, 640, 8),
                                                 (2, 8, 34), (2, 9, 34), (3, 32, 200), (1, 33, 200), (2, 128, 36), (2, 256, 20), (1, 511, 70)])
def test_scan_sizes(lib, batch, time, channels, dtype, sigmoid):
    _check_scan(lib, batch, time, channels, dtype, sigmoid)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,time,channels", [(1, 9000, 64), (2, 4097, 70), (8, 2048, 256), (300, 33, 64), (40, 260, 512)])
def test_scan_split_and_wide(lib, batch, time, channels, dtype):
    """Long sequences of few channels (time is split) and many channels."""
    _check_scan(lib, batch, time, channels, dtype, True, seed=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap,shift", [(0, 1), (1, 0), (2, 2), (3, 5), (64, 8)])
@pytest.mark.parametrize("time_major", [False, True])
def test_scan_layouts(lib, dtype, gap, shift, time_major):
    """Rows that no wide load fits, slices of wider matrices, both row orders."""
    _check_scan(lib, 3, 140, 66, dtype, True, gap=gap, shift=shift, time_major=time_major)
    _check_scan(lib, 2, 1, 70, dtype, False, gap=gap, shift=shift, time_major=time_major)


@pytest.mark.parametrize("time_major", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("time,lengths", [(1, [0, 1, -3, 5]), (9, [9, 0, 1, 8]), (260, [260, 0, 1, 129]), (5000, [17, 4999, 2500, 0])])
def test_scan_lengths(lib, time, lengths, sigmoid, time_major):
    """Sequences that end inside a tile, empty ones, lengths out of range; NaN and
    infinities in the rows left out."""
    _check_scan(lib, 4, time, 66, q.BF16, sigmoid, lengths=lengths, poison=True, time_major=time_major)
    _check_scan(lib, 4, time, 35, q.F32, sigmoid, lengths=lengths, poison=True, time_major=time_major)


@pytest.mark.parametrize("time", [1, 50, 3000])
def test_scan_without_optional_parts(lib, time):
    _check_scan(lib, 2, time, 64, q.F32, True, h0=False, dhT=False)
    _check_scan(lib, 2, time, 64, q.F32, True, hT=False)
    _check_scan(lib, 2, time, 64, q.BF16, False, in_place=True)


def test_scan_without_steps_copies_the_state(lib):
    d = _scan_data(2, 0, 10, q.F32, True, 1)
    assert np.array_equal(_scan_forward(lib, d, q.F32, True)[1], d["h0"])
    assert np.all(_scan_forward(lib, d, q.F32, True, h0=False)[1] == 0)
    assert np.array_equal(_scan_backward(lib, d, d["x"], q.F32, True)["dh0"], d["dhT"].astype(np.float64))


@pytest.mark.parametrize("time", [40, 2500])
def test_scan_values_stay_in_their_chain(lib, time):
    """Infinity and NaN in one channel reach no other, and nothing before them."""
    d = _scan_data(2, time, 64, q.F32, True, 4)
    d["x"][0, 30, 3], d["x"][1, 20, 7] = np.inf, np.nan
    ref, last, bound, _ = q.scan_fwd(d["x"], d["f"], d["h0"].astype(np.float64))
    got, got_last = _scan_forward(lib, d, q.F32, True)
    clean = np.ones(ref.shape, bool)
    clean[0, 30:, 3] = clean[1, 20:, 7] = False
    assert np.all(np.isfinite(got[clean]))
    _close(np.where(clean, got, 0), np.where(clean, ref, 0), np.where(clean, bound, 0), q.F32, "h")
    assert not np.isfinite(got[0, 30, 3]) and np.isnan(got[1, 20, 7])


def test_scan_steps_equal_the_whole(lib, stream):
    """A sequence token by token, the state carried in one buffer, gives the states
    of the whole sequence within the bound."""
    batch, time, channels = 2, 37, 96
    d = _scan_data(batch, time, channels, q.F32, True, 6)
    ref, last, bound, last_bound = q.scan_fwd(d["x"], d["f"], d["h0"].astype(np.float64))
    state = DeviceBuffer.from_array(d["h0"])
    x, f = (DeviceBuffer.from_array(_order(d[k], True).astype(np.float32)) for k in ("x", "f"))
    h = DeviceBuffer(batch * time * channels * 4)
    for t in range(time):
        at = t * batch * channels * 4
        capi.call("seera_hip_gated_scan_fwd_async", x.ptr + at, f.ptr + at, state.ptr, None, h.ptr + at, state.ptr, batch, 1, channels, channels, channels,
                  1, 0, q.F32, stream)
    capi.check(lib.seera_hip_stream_synchronize(stream))
    _close(h.to_array((time, batch, channels)).transpose(1, 0, 2).astype(np.float64), ref, bound, q.F32, "h")
    _close(state.to_array((batch, channels)).astype(np.float64), last, last_bound, q.F32, "state")


@pytest.mark.parametrize("time,channels", [(60, 64), (4000, 32)])
def test_scan_gradient_against_differences(lib, time, channels):
    """The backward's gradient along a direction against a difference of the GPU's
    own forward. The loss is linear in h, and x enters linearly: a step of any size
    gives the slope, so a step of one loses nothing to rounding."""
    d = _scan_data(1, time, channels, q.F32, True, 9)
    v = np.random.default_rng(10).standard_normal(d["x"].shape)
    h, last = _scan_forward(lib, d, q.F32, True)
    got = _scan_backward(lib, d, h, q.F32, True)

    def loss(x):
        h, last = _scan_forward(lib, {**d, "x": x.astype(np.float32).astype(np.float64)}, q.F32, True)
        return (h * d["dh"]).sum() + (last.astype(np.float64) * d["dhT"]).sum(), np.abs(h * d["dh"]).sum()

    (up, size), (down, _) = loss(d["x"] + v), loss(d["x"] - v)
    assert abs((up - down) / 2 - (got["dx"] * v).sum()) <= 64 * q.U * size * np.sqrt(time)
    # f enters smoothly: the second difference's error is step^2 times a third derivative of order one
    step = 2.0**-7
    w = v * np.isfinite(d["f"])
    def loss_f(s):
        g = np.where(np.isfinite(d["f"]), d["f"] + s * w, d["f"])
        h, last = _scan_forward(lib, {**d, "f": g.astype(np.float32).astype(np.float64)}, q.F32, True)
        return (h * d["dh"]).sum() + (last.astype(np.float64) * d["dhT"]).sum()
    slope = (loss_f(step) - loss_f(-step)) / (2 * step)
    want = (got["df"] * w).sum()
    assert abs(slope - want) <= step**2 * np.abs(got["df"] * w).sum() * 8 + 64 * q.U * size * np.sqrt(time) / step


@pytest.mark.parametrize("time", [3, 100, 2500])
def test_scan_linear_backward_without_x(lib, time):
    """No x and no row distance of one: the result of a call that gives both."""
    batch, c = 2, 40
    d = _scan_data(batch, time, c, q.F32, False, 13)
    h, _ = _scan_forward(lib, d, q.F32, False)
    want = _scan_backward(lib, d, h, q.F32, False)
    f, kept, dh = (Rows((batch, time, c), q.F32, data=a) for a in (d["f"], h, d["dh"]))
    dx, df = (Rows((batch, time, c), q.F32) for _ in range(2))
    h0, dhT, dh0 = DeviceBuffer.from_array(d["h0"]), DeviceBuffer.from_array(d["dhT"]), DeviceBuffer(d["h0"].nbytes)
    capi.call("seera_hip_gated_scan_bwd", None, f.ptr, h0.ptr, None, kept.ptr, dh.ptr, dhT.ptr, dx.ptr, df.ptr, dh0.ptr, batch, time, c, 0, c, c, c,
              capi.SEERA_GATE_LINEAR, 0, q.F32)
    assert np.array_equal(dx.values(), want["dx"]) and np.array_equal(df.values(), want["df"])
    assert np.array_equal(dh0.to_array(d["h0"].shape).astype(np.float64), want["dh0"])


def test_scan_rows_far_apart(lib):
    """Rows 8 MiB and more apart: a tile's rows would lie further from each other
    than 32 bits of address reach. x and f are two slices of the same wide rows."""
    time, c, ld = 40, 24, (1 << 21) + 3
    d = _scan_data(1, time, c, q.F32, True, 12)
    whole = np.zeros(time * ld, np.float32)
    rows = whole.reshape(time, ld)
    rows[:, :c], rows[:, c:2 * c] = d["x"][0], d["f"][0]
    xf, h0, h = DeviceBuffer.from_array(whole), DeviceBuffer.from_array(d["h0"]), Rows((1, time, c), q.F32)
    capi.call("seera_hip_gated_scan_fwd", xf.ptr, xf.ptr + 4 * c, h0.ptr, None, h.ptr, None, 1, time, c, ld, ld, 1, 0, 0)
    ref, _, bound, _ = q.scan_fwd(d["x"], d["f"], d["h0"].astype(np.float64))
    got = h.values()
    _close(got, ref, bound, q.F32, "h")
    kept, dh = Rows((1, time, c), q.F32, data=ref), Rows((1, time, c), q.F32, data=d["dh"])
    refs, bounds = q.scan_bwd(d["x"], d["f"], _seen(ref, q.F32), d["dh"], d["h0"].astype(np.float64))
    dx, df = (Rows((1, time, c), q.F32) for _ in range(2))
    capi.call("seera_hip_gated_scan_bwd", xf.ptr, xf.ptr + 4 * c, h0.ptr, None, kept.ptr, dh.ptr, None, dx.ptr, df.ptr, None, 1, time, c, ld, ld, c, c, 1, 0, 0)
    _close(dx.values(), refs["dx"], bounds["dx"], q.F32, "dx")
    _close(df.values(), refs["df"], bounds["df"], q.F32, "df")


# ---- block norm ----

NORM_PARTS = ["g r w1 s w2", "w2", "r w2", "g w1", "s r", "g", "g r s w2", ""]


def _norm_data(rows, cols, dtype, parts, seed):
    r = np.random.default_rng(seed)
    d = {"y": _seen(r.standard_normal((rows, cols)) * np.exp(r.standard_normal((rows, 1))), dtype)}
    for k in parts.split():
        if k in "gr":
            d[k] = _seen(r.standard_normal((rows, cols)) * 2, dtype)
        else:
            d[k] = (1 + 0.3 * r.standard_normal(cols)).astype(np.float32).astype(np.float64)
    d["dr_out"], d["dn"] = (_seen(r.standard_normal((rows, cols)), dtype) for _ in range(2))
    return d


def _norm_forward(lib, d, dtype, silu, gap=0, shift=0, stats=True, r_out=True, stream=None, eps=1e-6):
    rows, cols = d["y"].shape
    y = Rows((rows, cols), dtype, cols + gap, shift, d["y"], hole=np.nan)
    g = Rows((rows, cols), dtype, cols + gap, shift, d["g"], hole=np.nan) if "g" in d else None
    r = Rows((rows, cols), dtype, None, shift, d["r"]) if "r" in d else None
    w = {k: Rows((1, cols), q.F32, None, shift, d[k][None]) if k in d else None for k in ("w1", "s", "w2")}
    out, nxt = Rows((rows, cols), dtype, None, shift), Rows((rows, cols), dtype, None, shift)
    s1, s2 = Rows((1, rows), q.F32), Rows((1, rows), q.F32)
    p = lambda m, on=True: m.ptr if m is not None and on else None  # noqa: E731
    args = (y.ptr, p(g), p(r), p(w["w1"]), p(w["s"]), p(w["w2"]), p(out, r_out), p(nxt, "w2" in d), p(s1, stats), p(s2, stats), rows, cols, cols + gap, cols + gap,
            eps, 0 if silu else 1, dtype)
    if stream is None:
        capi.call("seera_hip_block_norm_fwd", *args)
    else:
        capi.call("seera_hip_block_norm_fwd_async", *args, stream)
        capi.check(lib.seera_hip_stream_synchronize(stream))
    got = {}
    if r_out:
        got["r_out"] = out.values()
    if "w2" in d:
        got["n_out"] = nxt.values()
        if stats:
            got["rstd2"] = s2.values()[0]
    if "w1" in d and stats:
        got["rstd1"] = s1.values()[0]
    return got


def _norm_backward(lib, d, kept, dtype, silu, gap=0, shift=0, dr=True, dr_out=True):
    rows, cols = d["y"].shape
    inner = any(k in d for k in ("w1", "g", "s"))
    y = Rows((rows, cols), dtype, cols + gap, shift, d["y"], hole=np.nan) if inner else None
    g = Rows((rows, cols), dtype, cols + gap, shift, d["g"], hole=np.nan) if "g" in d else None
    w = {k: Rows((1, cols), q.F32, None, shift, d[k][None]) if k in d else None for k in ("w1", "s", "w2")}
    dw = {k: Rows((1, cols), q.F32, None, shift) if k in d else None for k in ("w1", "s", "w2")}
    r = Rows((rows, cols), dtype, None, shift, kept["r_out"]) if "w2" in d else None
    s1 = Rows((1, rows), q.F32, data=kept["rstd1"][None]) if "w1" in d else None
    s2 = Rows((1, rows), q.F32, data=kept["rstd2"][None]) if "w2" in d else None
    d_r = Rows((rows, cols), dtype, None, shift, d["dr_out"]) if dr_out else None
    d_n = Rows((rows, cols), dtype, None, shift, d["dn"]) if "w2" in d else None
    dy, dg = (Rows((rows, cols), dtype, cols + gap, shift) for _ in range(2))
    d_x = Rows((rows, cols), dtype, None, shift)
    p = lambda m, on=True: m.ptr if m is not None and on else None  # noqa: E731
    capi.call("seera_hip_block_norm_bwd", p(y), p(g), p(r), p(w["w1"]), p(w["s"]), p(w["w2"]), p(s1), p(s2), p(d_r), p(d_n), dy.ptr, p(dg, "g" in d), p(d_x, dr),
              p(dw["w1"]), p(dw["s"]), p(dw["w2"]), rows, cols, cols + gap, cols + gap, cols + gap, cols + gap, 0 if silu else 1, dtype)
    got = {"dy": dy.values()}
    if "g" in d:
        got["dg"] = dg.values()
    if dr:
        got["dr"] = d_x.values()
    for k, m in dw.items():
        if m is not None:
            got["d" + k] = m.values()[0]
    return got


def _check_norm(lib, rows, cols, dtype, parts, silu=True, seed=1, d=None, **kw):
    d = d or _norm_data(rows, cols, dtype, parts, seed)
    names = ("y", "g", "r", "w1", "s")
    ref, bound = q.norm_fwd(**{k: d[k] for k in names if k in d}, silu=silu)
    got = _norm_forward(lib, d, dtype, silu, **kw)
    if "w2" in d:
        more, more_bound = q.norm_next(got["r_out"], d["w2"])  # of what was stored
        ref.update(more)
        bound.update(more_bound)
    for k in got:
        _close(got[k], ref[k], bound[k], dtype if k in ("r_out", "n_out") else q.F32, k)
    kept = {k: _seen(ref[k], dtype if k == "r_out" else q.F32) for k in ("r_out", "rstd1", "rstd2") if k in ref}
    refs, bounds = q.norm_bwd(d["y"], d.get("g"), kept["r_out"], d.get("w1"), d.get("s"), d.get("w2"), kept.get("rstd1"), kept.get("rstd2"),
                              d["dr_out"], d["dn"] if "w2" in d else None, silu)
    gots = _norm_backward(lib, d, kept, dtype, silu, **kw)
    for k in gots:
        _close(gots[k], refs[k], bounds[k], q.F32 if k[1:] in ("w1", "s", "w2") else dtype, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", NORM_PARTS)
def test_norm_parts(lib, dtype, parts):
    _check_norm(lib, 9, 200, dtype, parts, silu=True)
    _check_norm(lib, 5, 77, dtype, parts, silu=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (2, 63), (3, 512), (1, 1024), (700, 66), (4, 2048), (3, 2050), (2, 4096), (5, 4098), (2, 8192), (3, 8001), (2, 16384),
                                       (1, 16383), (1500, 256), (2100, 1000)])
def test_norm_sizes(lib, dtype, rows, cols):
    _check_norm(lib, rows, cols, dtype, "g r w1 s w2", seed=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", ["w2", "r w2", "g w1", "s r", "g r s w2"])
@pytest.mark.parametrize("rows,cols", [(1500, 2048), (700, 1024), (700, 1502), (600, 5002)])
def test_norm_parts_over_many_rows(lib, dtype, parts, rows, cols):
    """Several rows a block and several waves a row, with one of the two norms or
    none: the sums of consecutive rows share memory."""
    _check_norm(lib, rows, cols, dtype, parts, silu=cols != 1024, seed=cols)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap,shift", [(0, 1), (1, 0), (2, 2), (8, 0), (64, 4)])
def test_norm_layouts(lib, dtype, gap, shift):
    _check_norm(lib, 6, 264, dtype, "g r w1 s w2", gap=gap, shift=shift)
    _check_norm(lib, 6, 1200, dtype, "g w1", gap=gap, shift=shift, silu=False)


def test_norm_optional_outputs(lib, stream):
    d = _norm_data(4, 300, q.BF16, "g r w1 s w2", 3)
    full = _norm_forward(lib, d, q.BF16, True)
    less = _norm_forward(lib, d, q.BF16, True, stats=False, r_out=False, stream=stream)
    assert np.array_equal(full["n_out"], less["n_out"])
    kept = {k: full[k] for k in ("r_out", "rstd1", "rstd2")}
    whole = _norm_backward(lib, d, kept, q.BF16, True)
    less = _norm_backward(lib, d, kept, q.BF16, True, dr=False)
    assert all(np.array_equal(whole[k], less[k]) for k in less)
    refs, bounds = q.norm_bwd(d["y"], d["g"], kept["r_out"], d["w1"], d["s"], d["w2"], kept["rstd1"], kept["rstd2"], None, d["dn"])
    alone = _norm_backward(lib, d, kept, q.BF16, True, dr_out=False)
    for k in alone:
        _close(alone[k], refs[k], bounds[k], q.F32 if k[1:] in ("w1", "s", "w2") else q.BF16, k)


@pytest.mark.parametrize("cols", [200, 1501, 9000])
def test_norm_slope_of_a_saturated_gate(lib, cols):
    """The gradient of a sigmoid gate far from 0, against sigma(g) sigma(-g): each of
    the two by an exponential whose argument is rounded (|g| u), a sum, a reciprocal
    and products, so that the relative error stays (16 + 2 |g|) u where 1 - sigma(g)
    has no digit left."""
    rows = 3
    d = _norm_data(rows, cols, q.F32, "g", 31)
    d["g"] = _seen(np.linspace(-80, 80, rows * cols).reshape(rows, cols), q.F32)
    got = _norm_backward(lib, d, {}, q.F32, False)
    with np.errstate(over="ignore"):
        slope = 1 / (1 + np.exp(d["g"])) / (1 + np.exp(-d["g"]))
    want = d["dr_out"] * d["y"] * slope
    assert np.all(np.abs(got["dg"] - want) <= np.abs(want) * (16 + 2 * np.abs(d["g"])) * q.U + 2.0**-126)


def test_norm_of_no_rows(lib):
    """No rows: the sums over them are zero."""
    w, out = DeviceBuffer.from_array(np.ones(40, np.float32)), [DeviceBuffer.from_array(np.full(40, 7, np.float32)) for _ in range(3)]
    capi.call("seera_hip_block_norm_bwd", None, None, None, w.ptr, w.ptr, w.ptr, None, None, None, None, None, None, None, *[o.ptr for o in out], 0, 40, 40, 40, 40, 40, 0, 0)
    assert all(np.all(o.to_array(40) == 0) for o in out)


def test_norm_rows_of_zeros_and_of_large_values(lib):
    """A zero row has 1 / sqrt(eps); large gates saturate without a NaN."""
    d = _norm_data(6, 128, q.F32, "g r w1 s w2", 8)
    d["y"][1], d["r"][1] = 0, 0
    d["g"][2] = np.where(np.arange(128) % 2, 300.0, -300.0)
    d["y"][3] *= 1e15
    got = _norm_forward(lib, d, q.F32, True)
    ref, bound = q.norm_fwd(**{k: d[k] for k in ("y", "g", "r", "w1", "s")})
    assert got["rstd1"][1] == pytest.approx(1000, rel=1e-6) and np.all(got["n_out"][1] == 0)
    for k in ("r_out", "rstd1"):
        _close(got[k], ref[k], bound[k] + 1e-30, q.F32, k)
    kept = {**{k: _seen(ref[k], q.F32) for k in ("r_out", "rstd1")}, "rstd2": _seen(q.norm_next(_seen(ref["r_out"], q.F32), d["w2"])[0]["rstd2"], q.F32)}
    refs, bounds = q.norm_bwd(d["y"], d["g"], kept["r_out"], d["w1"], d["s"], d["w2"], kept["rstd1"], kept["rstd2"], d["dr_out"], d["dn"])
    gots = _norm_backward(lib, d, kept, q.F32, True)
    for k in gots:
        _close(gots[k], refs[k], bounds[k] + 1e-30, q.F32, k)


def test_norm_nan_stays_in_its_row(lib):
    d = _norm_data(5, 96, q.BF16, "g r w1 s w2", 8)
    d["y"][2, 7] = np.nan
    got = _norm_forward(lib, d, q.BF16, True)
    for k in ("r_out", "n_out"):
        assert np.all(np.isnan(got[k][2])) and np.all(np.isfinite(np.delete(got[k], 2, 0)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [8, 9, 77, 203, 1501, 2051, 5001, 9003])
def test_norm_infinities_at_a_rows_end(lib, dtype, cols):
    """An infinity in one of the last columns, where a row's last loads reach into
    each other at an odd width: the row's norm is 1 / infinity, so that its other
    values are 0; backward its mean is infinite and the row's gradients with it."""
    rows = 12
    at = [cols - 1 - min(i, cols - 1) for i in range(rows - 3)]  # three rows without
    for parts, forward, backward in (("r w2", "y", "dn"), ("g w1", "y", "dr_out")):
        d = _norm_data(rows, cols, dtype, parts, cols)
        for row, c in enumerate(at):
            d[forward][row, c] = np.inf if row % 2 else -np.inf
        with np.errstate(invalid="ignore"):
            ref, bound = q.norm_fwd(**{k: d[k] for k in ("y", "g", "r", "w1") if k in d})
            got = _norm_forward(lib, d, dtype, True)
            if "w2" in d:
                more, more_bound = q.norm_next(got["r_out"], d["w2"])
                ref.update(more)
                bound.update(more_bound)
        for k in got:
            _close(got[k], ref[k], bound[k], dtype if k in ("r_out", "n_out") else q.F32, k)
        d = _norm_data(rows, cols, dtype, parts, cols)
        kept = _norm_forward(lib, d, dtype, True)
        for row, c in enumerate(at):
            d[backward][row, c] = np.inf if row % 2 else -np.inf
        with np.errstate(invalid="ignore"):
            refs, bounds = q.norm_bwd(d["y"], d.get("g"), kept["r_out"], d.get("w1"), None, d.get("w2"), kept.get("rstd1"), kept.get("rstd2"),
                                      d["dr_out"], d["dn"] if "w2" in d else None)
        gots = _norm_backward(lib, d, kept, dtype, True)
        for k in gots:
            _close(gots[k], refs[k], bounds[k], q.F32 if k[1:] in ("w1", "s", "w2") else dtype, k)


def test_norm_in_place(lib):
    """r_out over r, dr over dr_out: the results of separate buffers."""
    rows, cols = 40, 512
    d = _norm_data(rows, cols, q.BF16, "g r w1 s w2", 3)
    want = _norm_forward(lib, d, q.BF16, True)
    m = {k: Rows((rows, cols), q.BF16, data=d[k]) for k in ("y", "g", "r", "dr_out", "dn")}
    w = {k: Rows((1, cols), q.F32, data=d[k][None]) for k in ("w1", "s", "w2")}
    dw = {k: Rows((1, cols), q.F32) for k in w}
    nxt, s1, s2 = Rows((rows, cols), q.BF16), Rows((1, rows), q.F32), Rows((1, rows), q.F32)
    capi.call("seera_hip_block_norm_fwd", m["y"].ptr, m["g"].ptr, m["r"].ptr, *[w[k].ptr for k in ("w1", "s", "w2")], m["r"].ptr, nxt.ptr, s1.ptr, s2.ptr, rows, cols,
              cols, cols, 1e-6, 0, q.BF16)
    assert np.array_equal(m["r"].values(), want["r_out"]) and np.array_equal(nxt.values(), want["n_out"])
    back = _norm_backward(lib, d, want, q.BF16, True)
    capi.call("seera_hip_block_norm_bwd", m["y"].ptr, m["g"].ptr, m["r"].ptr, *[w[k].ptr for k in ("w1", "s", "w2")], s1.ptr, s2.ptr, m["dr_out"].ptr, m["dn"].ptr,
              m["y"].ptr, m["g"].ptr, m["dr_out"].ptr, *[dw[k].ptr for k in ("w1", "s", "w2")], rows, cols, cols, cols, cols, cols, 0, q.BF16)
    for k, v in (("dy", m["y"]), ("dg", m["g"]), ("dr", m["dr_out"])):
        assert np.array_equal(v.values(), back[k]), k
    for k in dw:
        assert np.array_equal(dw[k].values()[0], back["d" + k]), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", ["g r w1 s w2", "w2", "r w2", "g w1", "s r", "g r s w2"])
@pytest.mark.parametrize("rows,cols", [(300, 1501), (40, 1500), (270, 5003), (300, 9001)])
def test_norm_in_place_over_several_waves(lib, dtype, parts, rows, cols):
    """Every overlap that is allowed, at widths of several waves whose last loads
    reach into the pack before them: the results of separate buffers, bit for bit."""
    d = _norm_data(rows, cols, dtype, parts, rows + cols)
    want = _norm_forward(lib, d, dtype, True)
    w = {k: Rows((1, cols), q.F32, data=d[k][None]) if k in d else None for k in ("w1", "s", "w2")}
    p = lambda m: m.ptr if m is not None else None  # noqa: E731
    weights = [p(w[k]) for k in ("w1", "s", "w2")]
    for r_over, n_over in (("r", "y"), ("y", "r"), ("g", "y"), ("r", "g"), ("y", None), (None, "y")):
        names = {r_over, n_over} - {None}
        if not names <= set(d) or (n_over and "w2" not in d):
            continue
        m = {k: Rows((rows, cols), dtype, data=d[k]) if k in d else None for k in ("y", "g", "r")}
        r_out = m[r_over] if r_over else Rows((rows, cols), dtype)
        n_out = (m[n_over] if n_over else Rows((rows, cols), dtype)) if "w2" in d else None
        capi.call("seera_hip_block_norm_fwd", m["y"].ptr, p(m["g"]), p(m["r"]), *weights, r_out.ptr, p(n_out), None, None, rows, cols, cols, cols, 1e-6, 0, dtype)
        assert np.array_equal(r_out.values(), want["r_out"]), (r_over, n_over)
        assert n_out is None or np.array_equal(n_out.values(), want["n_out"]), (r_over, n_over)
    back = _norm_backward(lib, d, want, dtype, True)
    inner = any(k in d for k in ("w1", "g", "s"))
    for dr_over in ("dr_out", "dn"):
        if dr_over == "dn" and "w2" not in d:
            continue
        m = {k: Rows((rows, cols), dtype, data=d[k]) if k in d else None for k in ("y", "g", "dr_out")}
        m["dn"] = Rows((rows, cols), dtype, data=d["dn"]) if "w2" in d else None
        kept = Rows((rows, cols), dtype, data=want["r_out"]) if "w2" in d else None
        s1, s2 = (Rows((1, rows), q.F32, data=want[k][None]) if k in want else None for k in ("rstd1", "rstd2"))
        dw = {k: Rows((1, cols), q.F32) if k in d else None for k in w}
        capi.call("seera_hip_block_norm_bwd", m["y"].ptr if inner else None, p(m["g"]), p(kept), *weights, p(s1), p(s2), m["dr_out"].ptr, p(m["dn"]),
                  m["y"].ptr, p(m["g"]), m[dr_over].ptr, *[p(dw[k]) for k in w], rows, cols, cols, cols, cols, cols, 0, dtype)
        for k, v in (("dy", m["y"]), ("dg", m["g"]), ("dr", m[dr_over])):
            assert v is None or np.array_equal(v.values(), back[k]), (k, dr_over)
        for k in dw:
            assert dw[k] is None or np.array_equal(dw[k].values()[0], back["d" + k]), (k, dr_over)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", ["g r w1 s w2", "w2", "g w1"])
def test_norm_wide_rows_over_many_rows(lib, dtype, parts):
    """Rows beyond the widths whose backward stays in registers, several a block."""
    _check_norm(lib, 520, 9002, dtype, parts, seed=77)


# ---- AdamW ----


class Tensors:
    """A list of tensors on the device and their descriptors."""

    def __init__(self, sizes, bits, grad_dtype, copy, seed, shift=0, decay=0.01, step=10):
        r = np.random.default_rng(seed)
        self.host, self.dev, self.table = [], [], (capi.AdamwTensor * max(len(sizes), 1))()
        bits = bits if isinstance(bits, list) else [bits] * len(sizes)
        for i, (n, b) in enumerate(zip(sizes, bits)):
            spread = np.exp(2 * r.standard_normal(n)) * 1e-3
            h = {"p": (r.standard_normal(n) * 0.1).astype(np.float32), "g": q.store(r.standard_normal(n) * spread, grad_dtype),
                 "m": (r.standard_normal(n) * spread * 0.3).astype(np.float32), "v": (spread * spread * r.random(n)).astype(np.float32), "bits": b,
                 "decay": decay if i % 2 == 0 else 0.0}
            d = {"p": Rows((1, n), q.F32, None, shift, h["p"][None]), "g": Rows((1, n), grad_dtype, None, shift, q.load(h["g"], grad_dtype)[None])}
            if b == 8:
                for k, top in (("m", 15), ("v", 31)):
                    codes, e = q.encode(h[k], r.integers(0, 65536, n), top)
                    h[k + "_codes"], h[k + "_exp"], h[k] = codes, e, q.decode(codes, e, top)
                    d[k] = DeviceBuffer.from_array(np.concatenate([np.full(shift, 0x5A, np.uint8), codes, np.full(64, 0x5A, np.uint8)]))
                    d[k + "_exp"] = DeviceBuffer.from_array(np.concatenate([e, np.full(64, 0x5A, np.uint8)]))
            else:
                d["m"], d["v"] = (Rows((1, n), q.F32, None, shift, h[k][None]) for k in ("m", "v"))
            at = shift if b == 8 else 0
            t = self.table[i]
            t.param, t.grad, t.m, t.v, t.count, t.state_bits = d["p"].ptr, d["g"].ptr, d["m"].ptr + at, d["v"].ptr + at, n, b
            t.grad_dtype, t.weight_decay = grad_dtype, h["decay"]
            if b == 8:
                t.m_exp, t.v_exp = d["m_exp"].ptr, d["v_exp"].ptr
            if copy:
                d["p16"] = Rows((1, n), copy, None, shift)
                t.param16, t.param16_dtype = d["p16"].ptr, copy
            self.host.append(h)
            self.dev.append(d)
        self.shift, self.grad_dtype, self.copy = shift, grad_dtype, copy

    def check(self, scale, lr, beta1, beta2, eps, step, seed):
        for i, (h, d) in enumerate(zip(self.host, self.dev)):
            n, g = len(h["p"]), q.load(h["g"], self.grad_dtype)
            p, m, v, bound = q.adamw(h["p"], h["m"], h["v"], g, scale, lr, beta1, beta2, eps, h["decay"], step)
            got = d["p"].values()[0]
            _close(got, p, bound, q.F32, f"p of tensor {i}")
            if self.copy:
                assert np.array_equal(d["p16"].raw()[0], q.store(got, self.copy)), f"copy of tensor {i}"
            with np.errstate(over="ignore", invalid="ignore"):
                m32, v32 = q.adamw_moments(h["m"], h["v"], g, scale, beta1, beta2)
            if h["bits"] == 32:
                assert np.array_equal(d["m"].raw()[0], m32) and np.array_equal(d["v"].raw()[0], v32), f"moments of tensor {i}"
                h["m"], h["v"] = m32, v32
            else:
                random = q.rounding_bits(seed, i, n)
                for k, top, value, part in (("m", 15, m32, random & 0xFFFF), ("v", 31, v32, random >> 16)):
                    codes, e = q.encode(value, part, top)
                    whole = d[k].to_array(d[k].nbytes, np.uint8)
                    assert np.all(whole[:self.shift] == 0x5A) and np.all(whole[self.shift + n:] == 0x5A), "written outside of the codes"
                    exps = d[k + "_exp"].to_array(d[k + "_exp"].nbytes, np.uint8)
                    assert np.array_equal(exps[:len(e)], e) and np.all(exps[len(e):] == 0x5A), f"exponents of tensor {i}.{k}"
                    fine = np.repeat(e != 255, q.BLOCK)[:n]
                    assert np.array_equal(whole[self.shift:self.shift + n][fine], codes[fine]), f"codes of tensor {i}.{k}"
                    h[k] = q.decode(whole[self.shift:self.shift + n], e, top)
            h["p"] = got.astype(np.float32)


CONSTANTS = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad_dtype", DTYPES)
@pytest.mark.parametrize("copy", [0, q.F16, q.BF16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_adamw_tensors(lib, bits, grad_dtype, copy, shift):
    """Sizes around the vectors, the blocks and a thread block's share; aligned or not."""
    t = Tensors([1, 5, 127, 128, 129, 2048, 4097, 20000, 0, 3], bits, grad_dtype, copy, 1, shift)
    scale = DeviceBuffer.from_array(np.array([0.37], np.float32))
    for step in (1, 2, 3):
        capi.call("seera_hip_adamw_step", t.table, len(t.host), *CONSTANTS.values(), step, 77 + step, scale.ptr)
        t.check(0.37, **CONSTANTS, step=step, seed=77 + step)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad_dtype", DTYPES)
@pytest.mark.parametrize("eps", [1e-8, 1e-30])
@pytest.mark.parametrize("decay", [0.0, 0.01])
def test_adamw_rounds_correctly(lib, bits, grad_dtype, eps, decay):
    """The parameter is that of fp32 operations, each rounded correctly, bit for bit,
    with states of either kind."""
    one = np.float32
    n, lr, beta1, beta2, scale = 20000, 3e-3, 0.9, 0.999, one(0.37)
    t = Tensors([n], bits, grad_dtype, 0, 21, decay=decay)
    device_scale = DeviceBuffer.from_array(np.array([scale], np.float32))
    for step in (1, 2, 50):
        h, d = t.host[0], t.dev[0]
        g = q.load(h["g"], grad_dtype).astype(np.float32)
        capi.call("seera_hip_adamw_step", t.table, 1, lr, beta1, beta2, eps, step, step, device_scale.ptr)
        m, v = q.adamw_moments(h["m"], h["v"], g, scale, beta1, beta2)
        size, root = one(lr / (1 - beta1**step)), one(1 / np.sqrt(1 - beta2**step))
        want = h["p"] * one(1 - lr * h["decay"]) - size * m / (np.sqrt(v) * root + one(eps))
        assert want.dtype == np.float32
        assert np.array_equal(d["p"].raw()[0].view(np.uint32), want.view(np.uint32))
        h["p"], h["m"], h["v"] = want, m, v
        if bits == 8:  # the next step starts from what the codes hold
            for k, top in (("m", 15), ("v", 31)):
                h[k] = q.decode(d[k].to_array(n, np.uint8), d[k + "_exp"].to_array(-(-n // q.BLOCK), np.uint8), top)


def test_adamw_many_tensors_of_both_kinds(lib, stream):
    """More tensors than one launch describes, 8 and 32 bits mixed, no gradient scale."""
    r = np.random.default_rng(2)
    sizes = [int(n) for n in np.exp(r.uniform(0, 8, 210))]
    t = Tensors(sizes, [8 if i % 3 else 32 for i in range(210)], q.F32, 0, 3)
    capi.call("seera_hip_adamw_step_async", t.table, len(sizes), *CONSTANTS.values(), 5, 9, None, stream)
    capi.check(lib.seera_hip_stream_synchronize(stream))
    t.check(1.0, **CONSTANTS, step=5, seed=9)


def test_adamw_from_nothing(lib):
    """All-zero states are zeros in both forms; the first step of both is the same."""
    n = 1000
    r = np.random.default_rng(4)
    p, g = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)
    g[::7] = 0
    out = []
    for bits in (32, 8):
        dp, dg = DeviceBuffer.from_array(p), DeviceBuffer.from_array(g)
        zero = [DeviceBuffer.from_array(np.zeros(4 * n, np.uint8)) for _ in range(4)]
        t = capi.AdamwTensor(param=dp.ptr, grad=dg.ptr, m=zero[0].ptr, v=zero[1].ptr, m_exp=zero[2].ptr, v_exp=zero[3].ptr, count=n, state_bits=bits)
        capi.call("seera_hip_adamw_step", ctypes.byref(t), 1, *CONSTANTS.values(), 1, 0, None)
        out.append(dp.to_array(n))
    assert np.array_equal(*out) and np.all(np.isfinite(out[0])) and np.array_equal(out[0][::7], p[::7])


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-12, 1e-6])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_small_eps(lib, eps, bits):
    """Gradients down to where their squares are denormal, with an eps that keeps them
    from mattering and without one."""
    n = 512
    r = np.random.default_rng(14)
    size = np.repeat(10.0 ** np.array([-19.5, -18, -12, -3]), 128)
    p, g = (0.1 * r.standard_normal(n)).astype(np.float32), (size * (0.5 + r.random(n)) * np.sign(r.standard_normal(n))).astype(np.float32)
    dp, dg = DeviceBuffer.from_array(p), DeviceBuffer.from_array(g)
    zero = [DeviceBuffer.from_array(np.zeros(4 * n, np.uint8)) for _ in range(4)]
    t = capi.AdamwTensor(param=dp.ptr, grad=dg.ptr, m=zero[0].ptr, v=zero[1].ptr, m_exp=zero[2].ptr, v_exp=zero[3].ptr, count=n, state_bits=bits)
    capi.call("seera_hip_adamw_step", ctypes.byref(t), 1, 1e-3, 0.9, 0.999, eps, 1, 0, None)
    # v as fp32 holds it: a denormal has fewer bits, which the reference follows
    m32, v32 = q.adamw_moments(np.zeros(n, np.float32), np.zeros(n, np.float32), g, 1.0, 0.9, 0.999)
    update = 1e-3 * (m32.astype(np.float64) / (1 - 0.9)) / (np.sqrt(v32.astype(np.float64) / (1 - 0.999)) + eps)
    got = dp.to_array(n).astype(np.float64)
    assert np.all(np.abs(got - (p - update)) <= 16 * q.U * (np.abs(p) + np.abs(update)))


def test_adamw_not_finite_gradients(lib):
    """Infinity and NaN reach their own parameter at once; an 8-bit block that held
    one is NaN from then on, other blocks are untouched."""
    t = Tensors([600], 8, q.F32, 0, 5)
    g = t.host[0]["g"].copy()
    g[10], g[300] = np.nan, np.inf
    buf = DeviceBuffer.from_array(g)
    t.table[0].grad = buf.ptr
    capi.call("seera_hip_adamw_step", t.table, 1, *CONSTANTS.values(), 1, 1, None)
    p = t.dev[0]["p"].values()[0]
    assert np.array_equal(np.flatnonzero(~np.isfinite(p)), [10, 300])
    values = [DeviceBuffer(600 * 4) for _ in range(2)]
    capi.call("seera_hip_adamw_state_values", t.table, 1, (ctypes.c_void_p * 1)(values[0].ptr), (ctypes.c_void_p * 1)(values[1].ptr))
    block = np.arange(600) // 128
    for b in values:
        assert np.array_equal(np.isnan(b.to_array(600)), (block == 0) | (block == 2))


@pytest.mark.parametrize("shift", [0, 3])
def test_adamw_state_values(lib, shift):
    sizes = [1, 127, 128, 1000, 5000, 0]
    t = Tensors(sizes, [8, 8, 32, 8, 32, 8], q.F32, 0, 6, shift)
    out = {k: [Rows((1, n), q.F32, None, shift) for n in sizes] for k in "mv"}
    ptrs = {k: (ctypes.c_void_p * len(sizes))(*[b.ptr for b in out[k]]) for k in "mv"}
    capi.call("seera_hip_adamw_state_values", t.table, len(sizes), ptrs["m"], ptrs["v"])
    for k in "mv":
        for h, b in zip(t.host, out[k]):
            assert np.array_equal(b.raw()[0], h[k]), k
    skipped = (ctypes.c_void_p * len(sizes))()
    fresh = [Rows((1, n), q.F32, None, shift) for n in sizes]
    capi.call("seera_hip_adamw_state_values", t.table, len(sizes), skipped, (ctypes.c_void_p * len(sizes))(*[b.ptr for b in fresh]))
    for h, b in zip(t.host, fresh):
        assert np.array_equal(b.raw()[0], h["v"])


def test_adamw_8_bits_learn_like_32(lib):
    """A noisy quadratic whose coordinates have curvatures over orders of magnitude:
    after 1500 steps the 8-bit states leave no more than 1.3 times the 32-bit ones'
    distance (rounding to nearest leaves v at a quarter of its value)."""
    n, steps = 4096, 1500
    r = np.random.default_rng(7)
    scale, start = np.exp(2 * r.standard_normal(n)), r.standard_normal(n).astype(np.float32)
    left = []
    for bits in (32, 8):
        noise = np.random.default_rng(8)
        dp, dg = DeviceBuffer.from_array(start), DeviceBuffer(4 * n)
        zero = [DeviceBuffer.from_array(np.zeros(4 * n, np.uint8)) for _ in range(4)]
        t = capi.AdamwTensor(param=dp.ptr, grad=dg.ptr, m=zero[0].ptr, v=zero[1].ptr, m_exp=zero[2].ptr, v_exp=zero[3].ptr, count=n, state_bits=bits)
        x = start
        for step in range(1, steps + 1):
            g = (scale * (x + 0.5 * noise.standard_normal(n))).astype(np.float32)
            capi.check(lib.seera_hip_memcpy_h2d(dg.ptr, g.ctypes.data, g.nbytes))
            capi.call("seera_hip_adamw_step", ctypes.byref(t), 1, 1e-2 * (1 - step / steps), 0.9, 0.999, 1e-8, step, step, None)
            x = dp.to_array(n)
        left.append(np.sqrt((x.astype(np.float64)**2).mean()))
    assert left[1] <= 1.3 * left[0] and left[0] < 0.1, left


# ---- streams and graphs ----


def test_graph_replays(lib, stream):
    """One training step's calls in a graph, replayed with new inputs between eager
    work: every replay equals the eager result bit for bit."""
    batch, time, c = 3, 2100, 64
    rows = batch * time
    r = np.random.default_rng(11)
    mats = {k: DeviceBuffer(rows * c * 4) for k in ("x", "f", "g", "r", "h", "ro", "no", "dro", "dn", "dy", "dg", "dr", "dx", "df")}
    vec = {k: DeviceBuffer.from_array(np.ones(c, np.float32)) for k in ("w1", "s", "w2", "dw1", "ds", "dw2", "m", "v")}
    st = {k: DeviceBuffer(rows * 4) for k in ("s1", "s2")}
    zero = DeviceBuffer.from_array(np.zeros(c, np.float32))
    t = capi.AdamwTensor(param=vec["w1"].ptr, grad=vec["dw1"].ptr, m=vec["m"].ptr, v=vec["v"].ptr, count=c, state_bits=32)

    def seq():
        capi.call("seera_hip_gated_scan_fwd_async", mats["x"].ptr, mats["f"].ptr, None, None, mats["h"].ptr, None, batch, time, c, c, c, 1, 0, 0, stream)
        capi.call("seera_hip_block_norm_fwd_async", mats["h"].ptr, mats["g"].ptr, mats["r"].ptr, vec["w1"].ptr, vec["s"].ptr, vec["w2"].ptr, mats["ro"].ptr, mats["no"].ptr,
                  st["s1"].ptr, st["s2"].ptr, rows, c, c, c, 1e-6, 0, 0, stream)
        capi.call("seera_hip_block_norm_bwd_async", mats["h"].ptr, mats["g"].ptr, mats["ro"].ptr, vec["w1"].ptr, vec["s"].ptr, vec["w2"].ptr, st["s1"].ptr, st["s2"].ptr,
                  mats["dro"].ptr, mats["dn"].ptr, mats["dy"].ptr, mats["dg"].ptr, mats["dr"].ptr, vec["dw1"].ptr, vec["ds"].ptr, vec["dw2"].ptr, rows, c, c, c, c, c, 0, 0, stream)
        capi.call("seera_hip_gated_scan_bwd_async", mats["x"].ptr, mats["f"].ptr, None, None, mats["h"].ptr, mats["dy"].ptr, None, mats["dx"].ptr, mats["df"].ptr, None,
                  batch, time, c, c, c, c, c, 1, 0, 0, stream)
        capi.call("seera_hip_adamw_step_async", ctypes.byref(t), 1, *CONSTANTS.values(), 3, 4, None, stream)

    ones = np.ones(c, np.float32)

    def reset(values):
        for k, v in values.items():
            capi.check(lib.seera_hip_memcpy_h2d(mats[k].ptr, v.ctypes.data, v.nbytes))
        for k, v in (("w1", ones), ("m", 0 * ones), ("v", 0 * ones)):
            capi.check(lib.seera_hip_memcpy_h2d(vec[k].ptr, v.ctypes.data, v.nbytes))

    def results():
        capi.check(lib.seera_hip_stream_synchronize(stream))
        return {**{k: mats[k].to_array(rows * c) for k in ("h", "ro", "no", "dy", "dg", "dr", "dx", "df")}, **{k: vec[k].to_array(c) for k in vec}}

    def fresh():
        return {k: r.standard_normal(rows * c).astype(np.float32) for k in ("x", "f", "g", "r", "dro", "dn")}

    reset(fresh())
    seq()
    results()
    capi.check(lib.seera_hip_graph_capture_begin(stream))
    try:
        seq()
    finally:
        graph = ctypes.c_void_p()
        status = lib.seera_hip_graph_capture_end(stream, ctypes.byref(graph))
    capi.check(status)
    try:
        for _ in range(4):
            values = fresh()
            reset(values)
            capi.check(lib.seera_hip_graph_launch(graph.value, stream))
            replayed = results()
            reset(values)
            seq()
            eager = results()
            for k in eager:
                assert np.array_equal(replayed[k].view(np.uint32), eager[k].view(np.uint32)), k
            assert np.any(eager["w1"] != 1)
    finally:
        capi.check(lib.seera_hip_graph_destroy(graph.value))
    del zero


def test_two_streams(lib):
    """Calls that use workspaces on two streams at once give each its own result."""
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        capi.check(lib.seera_hip_stream_create(ctypes.byref(s)))
        streams.append(s.value)
    try:
        time, c = 6000, 64
        want, bufs = [], []
        for i in range(2):
            d = _scan_data(1, time, c, q.F32, True, 20 + i)
            want.append(_scan_forward(lib, d, q.F32, True)[0])
            bufs.append([DeviceBuffer.from_array(d[k].astype(np.float32)) for k in ("x", "f", "h0")] + [DeviceBuffer(time * c * 4)])
        for _ in range(3):
            for s, (x, f, h0, h) in zip(streams, bufs):
                capi.call("seera_hip_gated_scan_fwd_async", x.ptr, f.ptr, h0.ptr, None, h.ptr, None, 1, time, c, c, c, 1, 0, 0, s)
        for s in streams:
            capi.check(lib.seera_hip_stream_synchronize(s))
        for w, b in zip(want, bufs):
            assert np.array_equal(b[3].to_array((1, time, c)).astype(np.float64), w)
    finally:
        for s in streams:
            lib.seera_hip_stream_destroy(s)
