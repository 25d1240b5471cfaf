"""The operators of a recurrent language model's block and of its training
step, as a program that holds tensors on the GPU calls them, and the same in
elementary operations.

Kinds of case (``case["kind"]``):
  scan    the gated linear recurrence over time, forward or backward; with
          ``time`` 1 the step of a model that generates token by token
  norm    the norms after and before a block with the gate, the residual scale
          and the residual between them, forward or backward
  adamw   an AdamW step over all tensors of a model, states in 32 or 8 bits

Activations are in the case's ``dtype``; weights, states, statistics and the
gradients of weights are fp32.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain form

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # the library's numbers for the types
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GATES = {"linear": 0, "sigmoid": 1}
ACTS = {"silu": 0, "sigmoid": 1}


def listed():
    return [
        # One token for each of 64 sequences: the smallest call of generation.
        {"name": "scan_step_64x1024", "kind": "scan", "backward": False, "batch": 64, "time": 1, "channels": 1024, "dtype": "bf16",
         "gate": "sigmoid", "packed": True, "ragged": False, "time_major": False},
        # A training batch: inputs and gates are two halves of one projection.
        {"name": "scan_fwd_8x2048x1024", "kind": "scan", "backward": False, "batch": 8, "time": 2048, "channels": 1024, "dtype": "bf16",
         "gate": "sigmoid", "packed": True, "ragged": False, "time_major": False},
        {"name": "scan_bwd_8x2048x1024", "kind": "scan", "backward": True, "batch": 8, "time": 2048, "channels": 1024, "dtype": "bf16",
         "gate": "sigmoid", "packed": True, "ragged": False, "time_major": False},
        # One long document: few channels, all of the work along time.
        {"name": "scan_fwd_1x65536x512", "kind": "scan", "backward": False, "batch": 1, "time": 65536, "channels": 512, "dtype": "f32",
         "gate": "linear", "packed": False, "ragged": False, "time_major": False},
        # Sequences of several lengths in one padded batch, odd in every size.
        {"name": "scan_bwd_ragged", "kind": "scan", "backward": True, "batch": 5, "time": 1537, "channels": 777, "dtype": "f32",
         "gate": "sigmoid", "packed": False, "ragged": True, "time_major": True},
        # The rows of one decoding step.
        {"name": "norm_fwd_16x1024", "kind": "norm", "backward": False, "rows": 16, "cols": 1024, "dtype": "bf16", "act": "silu", "parts": "full"},
        # A training batch, forward and backward, with every part.
        {"name": "norm_fwd_16384x2048", "kind": "norm", "backward": False, "rows": 16384, "cols": 2048, "dtype": "bf16", "act": "silu", "parts": "full"},
        {"name": "norm_bwd_16384x2048", "kind": "norm", "backward": True, "rows": 16384, "cols": 2048, "dtype": "bf16", "act": "silu", "parts": "full"},
        # Rows that no vector load fits, in the type of the framework's tensors.
        {"name": "norm_bwd_odd", "kind": "norm", "backward": True, "rows": 3001, "cols": 1501, "dtype": "f32", "act": "sigmoid", "parts": "full"},
        # The parameters of the 784-512-256-10 classifier.
        {"name": "adamw_mlp", "kind": "adamw", "sizes": "401408,131072,2560,512,256,10", "bits": 32, "grad": "f32", "copy": "none"},
        # Sixteen blocks of width 1024 (projections, norms) and an embedding of
        # 32768 rows; states in 32 bits, then in 8 beside 16-bit gradients.
        {"name": "adamw_model_32", "kind": "adamw", "sizes": "33554432,2097152*16,1048576*32,1024*48", "bits": 32, "grad": "f32", "copy": "none"},
        {"name": "adamw_model_8", "kind": "adamw", "sizes": "33554432,2097152*16,1048576*32,1024*48", "bits": 8, "grad": "bf16", "copy": "bf16"},
    ]


# A drawn case is no larger than the largest listed one of its kind.
MOST_SCAN, MOST_NORM, MOST_ADAMW = 33554432, 33554432, 100000000
NOT_SIZES = (1536, 3072)


def _log(rng, low, high):
    """A size spread evenly over the logarithm of [low, high]."""
    v = max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))
    return v + 1 if v in NOT_SIZES else v


def _round(rng, v, low):
    """Most sizes of real models are multiples of a power of two; half of the drawn ones are."""
    step = rng.choice([1, 1, 1, 8, 64, 128])
    v = max(low, v // step * step if v >= step else v)
    return v + step if v in NOT_SIZES else v


def draw(rng):
    """One more case of the same kinds and ranges."""
    kind = rng.choice(["scan", "scan", "norm", "norm", "adamw"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "scan":
        while True:
            case = {"kind": kind, "backward": rng.random() < 0.5, "batch": _log(rng, 1, 64), "time": rng.choice([1, _log(rng, 2, 65536), _log(rng, 128, 8192)]),
                    "channels": _round(rng, _log(rng, 32, 4096), 32), "dtype": dtype, "gate": rng.choice(["linear", "sigmoid"]),
                    "packed": rng.random() < 0.5, "ragged": rng.random() < 0.3, "time_major": rng.random() < 0.3}
            if case["batch"] * case["time"] * case["channels"] <= MOST_SCAN // (2 if case["backward"] else 1):
                return case
    if kind == "norm":
        while True:
            case = {"kind": kind, "backward": rng.random() < 0.5, "rows": _log(rng, 1, 32768), "cols": _round(rng, _log(rng, 64, 8192), 64), "dtype": dtype,
                    "act": rng.choice(["silu", "sigmoid"]), "parts": rng.choice(["full", "full", "pre", "gated"])}
            if case["rows"] * case["cols"] <= MOST_NORM:
                return case
    while True:
        sizes = [_log(rng, 1, rng.choice([1000, 100000, 4000000])) for _ in range(_log(rng, 1, 150))]
        if sum(sizes) <= MOST_ADAMW:
            break
    return {"kind": kind, "sizes": ",".join(str(s) for s in sorted(sizes, reverse=True)), "bits": rng.choice([8, 32]), "grad": dtype,
            "copy": rng.choice(["none", "f16", "bf16"])}


def _sizes(case):
    out = []
    for part in case["sizes"].split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def work(case):
    """Each input read once, each output written once."""
    if case["kind"] == "scan":
        b, t, c, e = case["batch"], case["time"], case["channels"], BYTES[case["dtype"]]
        share = 0.75 if case["ragged"] and t > 1 else 1.0  # lengths lie evenly between a half and all of the time
        n, linear = b * t * c, case["gate"] == "linear"
        if not case["backward"]:
            return {"bytes": int(n * e * (2 * share + 1) + 8 * b * c), "flops": int(n * share * (2 if linear else 8))}
        return {"bytes": int(n * e * ((3 if linear else 4) * share + 2) + 12 * b * c), "flops": int(n * share * (4 if linear else 14))}
    if case["kind"] == "norm":
        r, c, e = case["rows"], case["cols"], BYTES[case["dtype"]]
        y, g, res, w1, s, w2 = _parts(case)
        weights = sum((w1, s, w2))
        if not case["backward"]:
            return {"bytes": r * c * e * (1 + g + res + 1 + w2) + 4 * c * weights + 4 * r * (w1 + w2), "flops": r * c * 16}
        return {"bytes": r * c * e * ((w1 or g or s) + g + w2 + 1 + w2 + 1 + g + res) + 8 * c * weights + 4 * r * (w1 + w2), "flops": r * c * 40}
    n, g = sum(_sizes(case)), BYTES[case["grad"]]
    copy = 0 if case["copy"] == "none" else 2
    if case["bits"] == 32:
        return {"bytes": n * (24 + g + copy), "flops": n * 15}
    # codes in and out, a block's exponents, and the values written for the reader
    return {"bytes": int(n * (12 + g + copy + 8 + 4 / 128)), "flops": n * 50}


# ---- inputs ----


class _Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, seed, dtype=torch.float32):
        self.device, self.dtype = torch.device("cuda"), dtype
        self.gen = torch.Generator(device=self.device).manual_seed(int(seed) * 6007 + 29)

    def normal(self, *shape, scale=1.0, shift=0.0, dtype=None):
        return torch.randn(*shape, generator=self.gen, device=self.device).mul_(scale).add_(shift).to(dtype or self.dtype)

    def chance(self, *shape):
        return torch.rand(*shape, generator=self.gen, device=self.device)


def _scan_inputs(case, seed):
    b, t, c, dtype = case["batch"], case["time"], case["channels"], DTYPES[case["dtype"]]
    r = _Inputs(seed, dtype)
    rows = (t, b) if case["time_major"] else (b, t)
    # forget gates of a trained model: mostly open, some channels for thousands of steps
    gate = r.normal(*rows, c, scale=1.0, dtype=torch.float32) + torch.linspace(0.0, 6.0, c, device=r.device)
    start = r.chance(*rows, 1) < 1 / 512  # a new document begins: nothing is kept
    if case["gate"] == "linear":
        a = torch.sigmoid(gate)
        x, f = r.normal(*rows, c, dtype=torch.float32) * (1 - a), torch.where(start, 0.0, a)
    else:
        x, f = r.normal(*rows, c, dtype=torch.float32), torch.where(start, -math.inf, gate)
    st = {}
    if case["packed"]:
        st["xf"] = torch.cat([x, f], -1).to(dtype)
        st["x"], st["f"] = st["xf"][..., :c], st["xf"][..., c:]
    else:
        st["x"], st["f"] = x.to(dtype), f.to(dtype)
    del x, f, gate
    st["h0"] = r.normal(b, c, scale=0.3, dtype=torch.float32)
    if case["ragged"]:
        st["lengths"] = (t - (r.chance(b) * (t // 2 + 1)).int()).clamp_(0, t).int()
    if case["backward"]:
        st["dh"] = r.normal(*rows, c)
        st["dhT"] = r.normal(b, c, scale=0.3, dtype=torch.float32)
    return st


def _parts(case):
    """Which of y, g, r, w1, s, w2 a norm case has."""
    return {"full": (1, 1, 1, 1, 1, 1),  # after the block and before the next
            "gated": (1, 1, 0, 1, 0, 0),  # the gated norm inside a block
            "pre": (1, 0, 1, 0, 0, 1)}[case["parts"]]  # the residual, then the next block's norm


def _norm_inputs(case, seed):
    n, c, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
    r = _Inputs(seed, dtype)
    _, g, res, w1, s, w2 = _parts(case)
    st = {"y": r.normal(n, c, scale=0.7)}
    if g:
        st["g"] = r.normal(n, c)
    if res:
        st["r"] = r.normal(n, c, scale=2.0)
    if w1:
        st["w1"] = r.normal(c, scale=0.1, shift=1.0, dtype=torch.float32)
    if s:
        st["s"] = r.normal(c, scale=0.05, shift=0.3, dtype=torch.float32)
    if w2:
        st["w2"] = r.normal(c, scale=0.1, shift=1.0, dtype=torch.float32)
    if case["backward"]:
        st["dr_out"] = r.normal(n, c)
        if w2:
            st["dn"] = r.normal(n, c)
    return st


EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 128  # values of an 8-bit state that share an exponent
DECAYED = 8192  # tensors from this size on are products' weights, which decay


def _arena(case):
    """Where each tensor lies in the flat buffers (each starts a block)."""
    sizes = _sizes(case)
    starts = np.concatenate([[0], np.cumsum([-(-s // BLOCK) * BLOCK for s in sizes])])
    return sizes, [int(s) for s in starts[:-1]], int(starts[-1])


def _adamw_inputs(case, seed):
    sizes, starts, total = _arena(case)
    r = _Inputs(seed)
    inside = torch.zeros(total, dtype=torch.bool, device=r.device)
    if total == sum(sizes):
        inside[:] = True
    else:
        for n, at in zip(sizes, starts):
            inside[at:at + n] = True
    spread = torch.exp(r.normal(total)) * 1e-3  # gradients of one tensor differ by orders of magnitude
    grad = torch.where(inside, r.normal(total) * spread, 0.0)
    m = torch.where(inside, r.normal(total) * spread * 0.3, 0.0)
    v = torch.where(inside, (0.5 + r.chance(total)) * spread * spread, 0.0)
    p = torch.where(inside, r.normal(total) * 0.05, 0.0)
    return {"p": p, "grad": grad.to(DTYPES[case["grad"]]), "m": m, "v": v, "scale": torch.full((1,), 0.7, device=r.device)}


# What the library's step reads for each tensor (seera_adamw_tensor).
TENSOR = np.dtype([("param", "u8"), ("grad", "u8"), ("m", "u8"), ("v", "u8"), ("m_exp", "u8"), ("v_exp", "u8"), ("param16", "u8"), ("count", "i8"),
                   ("weight_decay", "f8"), ("grad_dtype", "i4"), ("param16_dtype", "i4"), ("state_bits", "i4"), ("reserved", "i4")])


def _prepare_adamw(case, seed):
    t = _adamw_inputs(case, seed)
    sizes, starts, total = _arena(case)
    if case["bits"] == 8:
        rng = torch.Generator(device="cuda").manual_seed(int(seed) + 5)
        for name, top in (("m", 15), ("v", 31)):
            value, dither = t[name], torch.randint(65536, (total,), generator=rng, device="cuda")
            t[name], t[name + "_exp"] = _encode(value, dither, top)
            t[name + "_values"] = torch.zeros(total, device="cuda")
    if case["copy"] != "none":
        t["p16"] = torch.zeros(total, dtype=DTYPES[case["copy"]], device="cuda")
    table = np.zeros(len(sizes), TENSOR)
    at = np.array(starts, np.uint64)

    def pointers(name, scale=None):
        return np.uint64(t[name].data_ptr()) + at * np.uint64(t[name].element_size()) if scale is None else np.uint64(t[name].data_ptr()) + at // np.uint64(scale)

    table["param"], table["grad"], table["m"], table["v"] = pointers("p"), pointers("grad"), pointers("m"), pointers("v")
    table["count"], table["state_bits"], table["grad_dtype"] = sizes, case["bits"], CODES[case["grad"]]
    table["weight_decay"] = [DECAY if s >= DECAYED else 0.0 for s in sizes]
    out = {"case": case, "t": t, "table": table, "step": 100, "tensors": len(sizes)}
    if case["bits"] == 8:
        table["m_exp"], table["v_exp"] = pointers("m_exp", BLOCK), pointers("v_exp", BLOCK)
        out["m_values"], out["v_values"] = pointers("m_values"), pointers("v_values")
    if case["copy"] != "none":
        table["param16"], table["param16_dtype"] = pointers("p16"), CODES[case["copy"]]
    return out


def prepare(case, seed):
    if case["kind"] == "adamw":
        st = _prepare_adamw(case, seed)
    elif case["kind"] == "scan":
        t = _scan_inputs(case, seed)
        rows = t["x"].shape[:2]
        if case["backward"]:
            h, _ = _scan_fwd(case, t)
            t["h"] = h  # what the forward kept
            if case["packed"]:
                t["dxf"] = torch.empty_like(t["xf"])
                t["dx"], t["df"] = t["dxf"][..., :case["channels"]], t["dxf"][..., case["channels"]:]
            else:
                t["dx"], t["df"] = torch.empty_like(t["x"]), torch.empty_like(t["f"])
            t["dh0"] = torch.empty_like(t["h0"])
        else:
            t["h"] = torch.empty(*rows, case["channels"], dtype=t["x"].dtype, device="cuda")
            t["hT"] = torch.empty_like(t["h0"])
        st = {"case": case, "t": t}
    else:
        t = _norm_inputs(case, seed)
        f32 = {"dtype": torch.float32, "device": "cuda"}
        if case["backward"]:
            fwd = _norm_fwd(case, t)
            for name in ("r_out", "rstd1", "rstd2"):  # what the forward kept
                if name in fwd:
                    t[name] = fwd[name]
            t["dy"] = torch.empty_like(t["y"])
            for of in ("g", "r", "w1", "s", "w2"):
                if of in t:
                    t["d" + of] = torch.empty_like(t[of])
        else:
            t["r_out"] = torch.empty_like(t["y"])
            if "w1" in t:
                t["rstd1"] = torch.empty(case["rows"], **f32)
            if "w2" in t:
                t["n_out"], t["rstd2"] = torch.empty_like(t["y"]), torch.empty(case["rows"], **f32)
        st = {"case": case, "t": t}
    # the pointers and the stream, as a program that drives a C ABI holds them
    st["p"] = {name: v.data_ptr() for name, v in st["t"].items()}
    st["stream"] = torch.cuda.current_stream().cuda_stream
    return st


# ---- the framework's calls ----


def _own_scan(case, t, p, stream):
    from ml_framework_amd import capi
    b, n, c = case["batch"], case["time"], case["channels"]
    ld = 2 * c if case["packed"] else c
    flags = (GATES[case["gate"]], int(case["time_major"]), CODES[case["dtype"]])
    if not case["backward"]:
        capi.call("seera_hip_gated_scan_fwd_async", p["x"], p["f"], p["h0"], p.get("lengths"), p["h"], p["hT"], b, n, c, ld, ld, *flags, stream)
        return {"h": t["h"], "hT": t["hT"]}
    capi.call("seera_hip_gated_scan_bwd_async", p["x"], p["f"], p["h0"], p.get("lengths"), p["h"], p["dh"], p["dhT"], p["dx"], p["df"], p["dh0"],
              b, n, c, ld, ld, ld, ld, *flags, stream)
    return {"dx": t["dx"], "df": t["df"], "dh0": t["dh0"]}


def _own_norm(case, t, p, stream):
    from ml_framework_amd import capi
    n, c = case["rows"], case["cols"]
    flags = (ACTS[case["act"]], CODES[case["dtype"]])
    if not case["backward"]:
        capi.call("seera_hip_block_norm_fwd_async", p["y"], p.get("g"), p.get("r"), p.get("w1"), p.get("s"), p.get("w2"), p["r_out"], p.get("n_out"),
                  p.get("rstd1"), p.get("rstd2"), n, c, c, c, EPS, *flags, stream)
        return {k: t[k] for k in ("r_out", "n_out", "rstd1", "rstd2") if k in t}
    capi.call("seera_hip_block_norm_bwd_async", p["y"], p.get("g"), p["r_out"], p.get("w1"), p.get("s"), p.get("w2"), p.get("rstd1"), p.get("rstd2"),
              p["dr_out"], p.get("dn"), p["dy"], p.get("dg"), p.get("dr"), p.get("dw1"), p.get("ds"), p.get("dw2"), n, c, c, c, c, c, *flags, stream)
    return {k: t[k] for k in ("dy", "dg", "dr", "dw1", "ds", "dw2") if k in t}


def _own_adamw(st):
    from ml_framework_amd import capi
    case, t = st["case"], st["t"]
    capi.call("seera_hip_adamw_step_async", st["table"].ctypes.data, st["tensors"], LR, BETA1, BETA2, ADAM_EPS, st["step"], st["step"], st["p"]["scale"], st["stream"])
    out = {"p": t["p"]}
    if case["bits"] == 8:
        capi.call("seera_hip_adamw_state_values_async", st["table"].ctypes.data, st["tensors"], st["m_values"].ctypes.data, st["v_values"].ctypes.data, st["stream"])
        out["m"], out["v"] = t["m_values"], t["v_values"]
    else:
        out["m"], out["v"] = t["m"], t["v"]
    if "p16" in t:
        out["p16"] = t["p16"]
    return out


# ---- the plain form ----


def _batch_major(case, v):
    return v.transpose(0, 1) if case["time_major"] else v


def _valid(case, t):
    """Which rows [batch, time] take part, or None for all."""
    if "lengths" not in t:
        return None
    return torch.arange(case["time"], device="cuda")[None, :] < t["lengths"][:, None]


def _affine_scan(a, b):
    """For c_t = a_t c_{t-1} + b_t over dimension 1 with c_{-1} = 0: all c_t and
    the products of a up to t, by doubling the span that each step covers."""
    span, time = 1, a.shape[1]
    while span < time:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b, a


def _gates(case, f):
    """a and 1 - a."""
    f = f.float()
    return (f, None) if case["gate"] == "linear" else (torch.sigmoid(f), torch.sigmoid(-f))


def _scan_fwd(case, t):
    x, f, valid = _batch_major(case, t["x"]).float(), _batch_major(case, t["f"]), _valid(case, t)
    a, rest = _gates(case, f)
    b = x if rest is None else rest * x
    if valid is not None:
        a, b = torch.where(valid[..., None], a, 1.0), torch.where(valid[..., None], b, 0.0)
    c, reach = _affine_scan(a, b)
    h = c + reach * t["h0"][:, None]
    last = h[:, -1].clone()
    if valid is not None:
        h = torch.where(valid[..., None], h, 0.0)
    return _batch_major(case, h).to(t["x"].dtype).contiguous(), last


def _scan_bwd(case, t):
    x, f, h, dh = (_batch_major(case, t[k]).float() for k in ("x", "f", "h", "dh"))
    valid = _valid(case, t)
    a, rest = _gates(case, f)
    if valid is not None:
        a, dh = torch.where(valid[..., None], a, 1.0), torch.where(valid[..., None], dh, 0.0)
    c, reach = _affine_scan(a.flip(1), (a * dh).flip(1))
    c = (c + reach * t["dhT"][:, None]).flip(1)
    g = dh + torch.cat([c[:, 1:], t["dhT"][:, None]], 1)
    before = torch.cat([t["h0"][:, None], h[:, :-1]], 1)
    dx, df = (g, g * before) if rest is None else (g * rest, g * (before - x) * a * rest)
    if valid is not None:
        dx, df = torch.where(valid[..., None], dx, 0.0), torch.where(valid[..., None], df, 0.0)
    return {"dx": _batch_major(case, dx).to(t["x"].dtype), "df": _batch_major(case, df).to(t["x"].dtype), "dh0": c[:, 0].clone()}


def _act(case, g):
    sig = torch.sigmoid(g)
    return (g * sig, sig * (1 + g * (1 - sig))) if case["act"] == "silu" else (sig, sig * (1 - sig))


def _norm_fwd(case, t):
    dtype, y, out = t["y"].dtype, t["y"].float(), {}
    u = y
    if "w1" in t:
        rstd = torch.rsqrt(y.square().mean(1) + EPS)
        out["rstd1"], u = rstd, y * rstd[:, None] * t["w1"]
    if "g" in t:
        u = u * _act(case, t["g"].float())[0]
    if "s" in t:
        u = u * t["s"]
    r = u + t["r"].float() if "r" in t else u
    out["r_out"] = r.to(dtype)
    if "w2" in t:
        r = out["r_out"].float()  # the next norm is of the residual stream as it is kept
        rstd = torch.rsqrt(r.square().mean(1) + EPS)
        out["rstd2"], out["n_out"] = rstd, (r * rstd[:, None] * t["w2"]).to(dtype)
    return out


def _norm_bwd(case, t):
    dtype, y, d, out = t["y"].dtype, t["y"].float(), t["dr_out"].float(), {}
    if "w2" in t:
        dn, hat = t["dn"].float(), t["r_out"].float() * t["rstd2"][:, None]
        q = dn * t["w2"]
        out["dw2"] = (dn * hat).sum(0)
        d = d + t["rstd2"][:, None] * (q - hat * (q * hat).mean(1, keepdim=True))
    if "r" in t:
        out["dr"] = d.to(dtype)
    hat = y * t["rstd1"][:, None] if "w1" in t else y
    z = hat * t["w1"] if "w1" in t else y
    if "s" in t:
        gated = _act(case, t["g"].float())[0] * z if "g" in t else z
        out["ds"] = (d * gated).sum(0)
        d = d * t["s"]
    if "g" in t:
        act, slope = _act(case, t["g"].float())
        out["dg"] = (d * z * slope).to(dtype)
        d = d * act
    if "w1" in t:
        out["dw1"] = (d * hat).sum(0)
        q = d * t["w1"]
        d = t["rstd1"][:, None] * (q - hat * (q * hat).mean(1, keepdim=True))
    out["dy"] = d.to(dtype)
    return out


def _shared_exponents(a):
    """For each block of non-negative values, the (biased) exponent of the
    smallest power of two whose 1.875-fold reaches the largest of them."""
    largest = a.view(-1, BLOCK).amax(1)
    return ((largest.view(torch.int32) + 0x0FFFFF) >> 23).to(torch.uint8)


def _pow2(k):
    """2**k of a whole number -126 <= k <= 127, by its bits."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _encode(value, dither, top):
    """8-bit codes and exponents of `value`: 3 bits of mantissa below an exponent
    field that is `top` at the block's exponent (top 15: a sign bit too), rounded
    up or down by `dither` of 65536."""
    a = value.abs()
    exponents = _shared_exponents(a)
    z = (a.view(-1, BLOCK) * _pow2(127 - exponents.int())[:, None]).view(-1)
    low = 1 - top
    k = torch.where(z > 0, torch.frexp(z)[1] - 1, low).clamp_min_(low)
    ticks = torch.round(z * _pow2(23 - k)).int()  # of 2^(k - 23)
    code = (k + (top - 1)) * 8 + ((ticks + 16 * dither.int()) >> 20)
    if top == 31:
        code = torch.where(a > 0, code.clamp_min(1), code)
    else:
        code = code + torch.where(value < 0, 128, 0)
    return code.to(torch.uint8), exponents


def _decode(codes, exponents, top):
    c = codes.int()
    size = c & 127 if top == 15 else c
    field = size >> 3
    k = field.clamp_min(1) - top
    mantissa = (size & 7) + torch.where(field > 0, 8, 0)
    value = mantissa.float() * _pow2(k - 3)
    value = (value.view(-1, BLOCK) * _pow2(exponents.int() - 127)[:, None]).view(-1)
    return torch.where(c >= 128, -value, value) if top == 15 else value


WORD = 0xFFFFFFFF


def _mix(x):
    """A 32-bit hash (in 64-bit integers)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & WORD
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & WORD
    return x ^ (x >> 16)


def _hashes(case, seed):
    """The rounding's random bits: of (seed, tensor, index in the tensor)."""
    sizes, starts, total = _arena(case)
    keys = _mix((torch.arange(len(sizes), device="cuda") * 0x9E3779B9 + seed) & WORD)
    spans = torch.tensor([b - a for a, b in zip(starts, starts[1:] + [total])], device="cuda")
    first = torch.tensor(starts, device="cuda")
    which = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), spans, output_size=total)
    index = torch.arange(total, device="cuda") - first[which]
    return _mix((index * 0x9E3779B9 + keys[which]) & WORD)


def _plain_adamw(st):
    case, t, step = st["case"], st["t"], st["step"]
    sizes, starts, total = _arena(case)
    decayed = next((at for n, at in zip(sizes, starts) if n < DECAYED), total)  # sizes fall: weights that decay come first
    grad = t["grad"].float() * t["scale"]
    bits8 = case["bits"] == 8
    m = _decode(t["m"], t["m_exp"], 15) if bits8 else t["m"]
    v = _decode(t["v"], t["v_exp"], 31) if bits8 else t["v"]
    m = m * BETA1 + grad * (1 - BETA1)
    v = v * BETA2 + (grad * grad) * (1 - BETA2)
    update = m * (LR / (1 - BETA1**step)) / (torch.sqrt(v) / math.sqrt(1 - BETA2**step) + ADAM_EPS)
    t["p"][:decayed] *= 1 - LR * DECAY
    t["p"] -= update
    out = {"p": t["p"]}
    if "p16" in t:
        out["p16"] = t["p16"].copy_(t["p"])
    if not bits8:
        out["m"], out["v"] = t["m"].copy_(m), t["v"].copy_(v)
        return out
    bits = _hashes(case, step)
    t["m"], t["m_exp"] = _encode(m, bits & 0xFFFF, 15)
    t["v"], t["v_exp"] = _encode(v, bits >> 16, 31)
    out["m"], out["v"] = _decode(t["m"], t["m_exp"], 15), _decode(t["v"], t["v_exp"], 31)
    return out


def run(state):
    case, t = state["case"], state["t"]
    if case["kind"] == "adamw":
        out = _own_adamw(state) if own else _plain_adamw(state)
        state["step"] += 1
        return out
    if own:
        return (_own_scan if case["kind"] == "scan" else _own_norm)(case, t, state["p"], state["stream"])
    if case["kind"] == "scan":
        if case["backward"]:
            return _scan_bwd(case, t)
        h, last = _scan_fwd(case, t)
        return {"h": h, "hT": last}
    return _norm_bwd(case, t) if case["backward"] else _norm_fwd(case, t)


# ---- the same in 64 bits ----


def _exact_scan(case, t):
    """Step by step along time."""
    d = {k: v.double() for k, v in t.items() if k != "lengths"}
    time_dim = 0 if case["time_major"] else 1
    n = t.get("lengths")
    linear = case["gate"] == "linear"
    x, f = (d[k].movedim(time_dim, 0).contiguous() for k in ("x", "f"))
    a = f if linear else 1 / (1 + torch.exp(-f))
    b = x if linear else x / (1 + torch.exp(f))
    steps = range(case["time"])
    if not case["backward"]:
        h, state = torch.zeros_like(x), d["h0"]
        for i in steps:
            new = a[i] * state + b[i]
            if n is None:
                h[i] = state = new
            else:
                live = (n > i)[:, None]
                h[i], state = torch.where(live, new, 0.0), torch.where(live, new, state)
        return {"h": h.movedim(0, time_dim).contiguous(), "hT": state}
    h, dh = (d[k].movedim(time_dim, 0).contiguous() for k in ("h", "dh"))
    dx, df, carry = torch.zeros_like(x), torch.zeros_like(x), d["dhT"]
    for i in reversed(steps):
        g = dh[i] + carry
        before = h[i - 1] if i else d["h0"]
        one = g if linear else g / (1 + torch.exp(f[i]))
        two = g * before if linear else one * (before - x[i]) * a[i]
        new = a[i] * g
        if n is not None:
            live = (n > i)[:, None]
            one, two, new = torch.where(live, one, 0.0), torch.where(live, two, 0.0), torch.where(live, new, carry)
        dx[i], df[i], carry = one, two, new
    return {"dx": dx.movedim(0, time_dim).contiguous(), "df": df.movedim(0, time_dim).contiguous(), "dh0": carry}


def _exact_norm(case, t):
    """The forward's formulas, and its gradient by automatic differentiation."""
    names = [k for k in ("y", "g", "r", "w1", "s", "w2") if k in t]
    d = {k: t[k].double().requires_grad_(case["backward"]) for k in names}

    def rms(v):
        rstd = (v.pow(2).sum(1, keepdim=True) / case["cols"] + EPS).pow(-0.5)
        return v * rstd, rstd[:, 0]

    def block():
        out, u = {}, d["y"]
        if "w1" in d:
            u, out["rstd1"] = rms(u)
            u = u * d["w1"]
        if "g" in d:
            sig = 1 / (1 + torch.exp(-d["g"]))
            u = u * (d["g"] * sig if case["act"] == "silu" else sig)
        u = u * d["s"] if "s" in d else u
        out["r_out"] = u + d["r"] if "r" in d else u
        return out

    out = block()
    if "w2" in d:
        # the next norm is of the residual stream as it is kept, rounded
        r = out["r_out"].detach()
        kept = out["r_out"] + (r.to(t["y"].dtype).double() - r)
        n, out["rstd2"] = rms(kept)
        out["n_out"] = n * d["w2"]
    if not case["backward"]:
        return {k: out[k] for k in ("r_out", "n_out", "rstd1", "rstd2") if k in out}
    loss = (out["r_out"] * t["dr_out"].double()).sum()
    if "w2" in d:
        loss = loss + (out["n_out"] * t["dn"].double()).sum()
    grads = dict(zip(names, torch.autograd.grad(loss, [d[k] for k in names])))
    return {"d" + k: grads[k] for k in ("y", "g", "r", "w1", "s", "w2") if k in grads}


def _exact_codes(value, dither, top):
    """What the 8-bit state holds of `value`, in 64 bits."""
    a = value.abs().view(-1, BLOCK)
    largest = a.amax(1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0)))
    e = e + (largest > 1.875 * 2.0**e)
    lowest = 2.0 ** (e + 1 - top)
    own_power = 2.0 ** torch.floor(torch.log2(torch.where(a > 0, a, 1.0)))
    unit = torch.maximum(torch.where(a > 0, own_power, 0.0), lowest) / 8
    held = torch.floor(a / unit + dither.view(-1, BLOCK).double() / 65536) * unit
    if top == 31:
        held = torch.where(a > 0, torch.maximum(held, lowest / 8), held)
    return torch.copysign(held.view(-1), value)


def _exact_adamw(case, seed):
    state = _prepare_adamw(case, seed)
    t, step = state["t"], state["step"]
    sizes, starts, total = _arena(case)
    m, v = t["m"], t["v"]
    if case["bits"] == 8:
        m, v = _decode(m, t["m_exp"], 15), _decode(v, t["v_exp"], 31)
    g = t["grad"].double() * t["scale"].double()
    m = BETA1 * m.double() + (1 - BETA1) * g
    v = BETA2 * v.double() + (1 - BETA2) * g * g
    decay = torch.zeros(total, dtype=torch.float64, device="cuda")
    for n, at in zip(sizes, starts):
        if n >= DECAYED:
            decay[at:at + n] = DECAY
    p = t["p"].double()
    p = p - LR * (decay * p + m / (1 - BETA1**step) / (torch.sqrt(v / (1 - BETA2**step)) + ADAM_EPS))
    out = {"p": p}
    if "p16" in t:
        out["p16"] = p
    if case["bits"] == 8:
        bits = _hashes(case, step)
        m, v = _exact_codes(m, bits & 0xFFFF, 15), _exact_codes(v, bits >> 16, 31)
    out["m"], out["v"] = m, v
    return out


def exact(case, seed):
    if case["kind"] == "adamw":
        return _exact_adamw(case, seed)
    if case["kind"] == "scan":
        t = _scan_inputs(case, seed)
        if case["backward"]:
            t["h"], _ = _scan_fwd(case, t)
        return _exact_scan(case, t)
    return _exact_norm(case, _norm_inputs(case, seed))
