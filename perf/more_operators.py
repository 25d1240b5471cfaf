"""The operators with which a language model answers in 8 bits, as a program that
holds tensors on the GPU calls them, and the same in elementary operations.

Kinds of case (``case["kind"]``):
  norm      the norms after and before a block with the gate, the residual scale and
            the residual between them, the next product's operand in 8 bits with a
            scale for each 128 columns of a row
  quantize  a weight matrix in 8 bits with a scale for each block of 128 x 128
  matmul    the product of two such operands
  sample    a token for each row of logits: temperature, top-k, top-p and min-p from
            given random numbers

8-bit values are e4m3 codes (4 bits of exponent, 3 of mantissa, largest 448); rows
of codes are padded with zeros to a multiple of 128. Activations, products' results
and logits are in the case's ``dtype``; weights of norms and scales are fp32.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain form

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # the library's numbers for the types
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTS = {"silu": 0, "sigmoid": 1}
F8 = torch.float8_e4m3fn
BLOCK, LARGEST = 128, 448.0
EPS = 1e-6


def listed():
    return [
        # The rows of one decoding step of 16 sequences.
        {"name": "norm_16x4096", "kind": "norm", "rows": 16, "cols": 4096, "dtype": "bf16", "act": "silu", "parts": "full"},
        # A prompt of 16384 tokens (or as many prompts' rows), with every part.
        {"name": "norm_16384x4096", "kind": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "act": "silu", "parts": "full"},
        # Rows that no vector load fits, in the type of the framework's tensors.
        {"name": "norm_odd", "kind": "norm", "rows": 3001, "cols": 1501, "dtype": "f32", "act": "sigmoid", "parts": "pre"},
        # A square weight of a small model as the framework trains it: fp32, [in, out].
        {"name": "quantize_1024x1024", "kind": "quantize", "n": 1024, "k": 1024, "dtype": "f32", "transposed": False},
        # The projection [x | f | g] of a block of width 4096.
        {"name": "quantize_12288x4096", "kind": "quantize", "n": 12288, "k": 4096, "dtype": "bf16", "transposed": False},
        # One token of one sequence: the smallest call of generation.
        {"name": "matmul_1x4096x4096", "kind": "matmul", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": False},
        # A step of 64 sequences through [x | f | g].
        {"name": "matmul_64x12288x4096", "kind": "matmul", "m": 64, "n": 12288, "k": 4096, "dtype": "bf16", "bias": False},
        # Odd in every size, with a bias, in the type of the framework's tensors.
        {"name": "matmul_odd", "kind": "matmul", "m": 777, "n": 1501, "k": 1000, "dtype": "f32", "bias": True},
        # A prompt of 8192 tokens through [x | f | g].
        {"name": "matmul_8192x12288x4096", "kind": "matmul", "m": 8192, "n": 12288, "k": 4096, "dtype": "bf16", "bias": False},
        # The next token of one sequence, with every cut.
        {"name": "sample_1x32768", "kind": "sample", "rows": 1, "vocab": 32768, "dtype": "f32", "cuts": "kpm", "masked": False},
        # A batch that samples from the nucleus of a large vocabulary.
        {"name": "sample_64x131072", "kind": "sample", "rows": 64, "vocab": 131072, "dtype": "bf16", "cuts": "p", "masked": False},
        # A grammar forbids most tokens; rows that no vector load fits.
        {"name": "sample_256x50001", "kind": "sample", "rows": 256, "vocab": 50001, "dtype": "f16", "cuts": "kp", "masked": True},
    ]


# A drawn case is no larger than the largest listed one of its kind.
MOST_NORM, MOST_QUANTIZE, MOST_MATMUL, MOST_SAMPLE = 16384 * 4096, 12288 * 4096, 8192 * 12288 * 4096, 256 * 50001


def _log(rng, low, high):
    """A size spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _round(rng, v, low):
    """Most sizes of real models are multiples of a power of two; half of the drawn ones are."""
    step = rng.choice([1, 1, 1, 8, 64, 128])
    return max(low, v // step * step if v >= step else v)


def draw(rng):
    """One more case of the same kinds and ranges."""
    kind = rng.choice(["norm", "quantize", "matmul", "matmul", "matmul", "sample", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    while True:
        if kind == "norm":
            case = {"kind": kind, "rows": _log(rng, 1, 32768), "cols": _round(rng, _log(rng, 64, 16384), 64), "dtype": dtype,
                    "act": rng.choice(["silu", "sigmoid"]), "parts": rng.choice(["full", "full", "pre", "gated", "none"])}
            if case["rows"] * case["cols"] <= MOST_NORM:
                return case
        elif kind == "quantize":
            case = {"kind": kind, "n": _round(rng, _log(rng, 64, 32768), 64), "k": _round(rng, _log(rng, 64, 16384), 64), "dtype": dtype,
                    "transposed": rng.random() < 0.5}
            if case["n"] * case["k"] <= MOST_QUANTIZE:
                return case
        elif kind == "matmul":
            case = {"kind": kind, "m": rng.choice([1, _log(rng, 1, 128), _log(rng, 64, 16384)]), "n": _round(rng, _log(rng, 64, 32768), 64),
                    "k": _round(rng, _log(rng, 64, 16384), 64), "dtype": dtype, "bias": rng.random() < 0.5}
            if case["m"] * case["n"] * case["k"] <= MOST_MATMUL:
                return case
        else:
            case = {"kind": kind, "rows": _log(rng, 1, 512), "vocab": _round(rng, _log(rng, 256, 262144), 256), "dtype": dtype,
                    "cuts": rng.choice(["", "k", "p", "m", "kp", "kpm"]), "masked": rng.random() < 0.25}
            if case["rows"] * case["vocab"] <= MOST_SAMPLE:
                return case


def _padded(k):
    return -(-k // BLOCK) * BLOCK


def _parts(case):
    """Which of y, g, r, w1, s, w2 a norm case has."""
    return {"full": (1, 1, 1, 1, 1, 1),  # after the block and before the next
            "pre": (1, 0, 1, 0, 0, 1),  # the residual, then the next block's norm
            "gated": (1, 1, 0, 1, 0, 0),  # the gated norm inside a block
            "none": (1, 0, 0, 0, 0, 0)}[case["parts"]]  # an operand that needs no norm


def work(case):
    """Each input read once, each output written once."""
    e = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        r, c = case["rows"], case["cols"]
        _, g, res, w1, s, w2 = _parts(case)
        return {"bytes": r * c * e * (1 + g + 2 * res) + r * (_padded(c) + _padded(c) // BLOCK * 4) + 4 * c * (w1 + s + w2), "flops": r * c * 20}
    if case["kind"] == "quantize":
        n, k = case["n"], case["k"]
        return {"bytes": n * k * e + n * _padded(k) + _padded(n) // BLOCK * (_padded(k) // BLOCK) * 4, "flops": n * k * 4}
    if case["kind"] == "matmul":
        m, n, k = case["m"], case["n"], _padded(case["k"])
        scales = 4 * (k // BLOCK) * (m + _padded(n) // BLOCK)
        return {"bytes": (m + n) * k + scales + m * n * e + 4 * n * case["bias"], "flops": 2 * m * n * case["k"]}
    return {"bytes": case["rows"] * (case["vocab"] * e + 28), "flops": case["rows"] * case["vocab"] * 20}


# ---- inputs ----


class _Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, seed, dtype=torch.float32):
        self.device, self.dtype = torch.device("cuda"), dtype
        self.gen = torch.Generator(device=self.device).manual_seed(int(seed) * 7919 + 31)

    def normal(self, *shape, scale=1.0, shift=0.0, dtype=None):
        return torch.randn(*shape, generator=self.gen, device=self.device).mul_(scale).add_(shift).to(dtype or self.dtype)

    def chance(self, *shape):
        return torch.rand(*shape, generator=self.gen, device=self.device)


def _norm_inputs(case, seed):
    n, c = case["rows"], case["cols"]
    r = _Inputs(seed, DTYPES[case["dtype"]])
    _, g, res, w1, s, w2 = _parts(case)
    st = {"y": r.normal(n, c, scale=0.7)}
    if g:
        st["g"] = r.normal(n, c)
    if res:
        # a residual stream has channels far larger than the rest
        st["r"] = (r.normal(n, c, scale=2.0, dtype=torch.float32) * torch.where(r.chance(c) < 0.01, 10.0, 1.0)).to(r.dtype)
    f32 = {"dtype": torch.float32}
    if w1:
        st["w1"] = r.normal(c, scale=0.1, shift=1.0, **f32)
    if s:
        st["s"] = r.normal(c, scale=0.05, shift=0.3, **f32)
    if w2:
        st["w2"] = r.normal(c, scale=0.1, shift=1.0, **f32)
    return st


def _quantize_inputs(case, seed):
    n, k = case["n"], case["k"]
    r = _Inputs(seed, DTYPES[case["dtype"]])
    shape = (n, k) if case["transposed"] else (k, n)
    return {"w": r.normal(*shape, scale=1 / math.sqrt(k))}


def _matmul_inputs(case, seed):
    m, n, k = case["m"], case["n"], case["k"]
    r = _Inputs(seed)
    a = r.normal(m, k) * torch.where(r.chance(k) < 0.01, 8.0, 1.0)
    st = {}
    st["a"], st["a_scales"] = _quantize_rows(a)
    st["w"], st["w_scales"] = _quantize_blocks(r.normal(n, k, scale=1 / math.sqrt(k)))
    if case["bias"]:
        st["bias"] = r.normal(n, scale=0.1)
    return st


def _sample_inputs(case, seed):
    n, v = case["rows"], case["vocab"]
    r = _Inputs(seed, DTYPES[case["dtype"]])
    # a broad body, and a few tokens that the text asks for
    z = r.normal(n, v, scale=2.0, dtype=torch.float32)
    z += torch.where(r.chance(n, v) < 20.0 / v, 7.0, 0.0)
    if case["masked"]:
        z = torch.where(r.chance(n, v) < 0.9, -math.inf, z)
        z[:, v // 2] = 0.0
    st = {"logits": z.to(r.dtype), "uniform": r.chance(n)}
    greedy = r.chance(n) < 1 / 16
    st["temperature"] = torch.where(greedy, 0.0, 0.6 + 0.6 * r.chance(n))
    if "k" in case["cuts"]:
        st["top_k"] = (1 + r.chance(n) ** 2 * min(v, 1000)).int()
    if "p" in case["cuts"]:
        st["top_p"] = 1 - 0.3 * r.chance(n) ** 2
    if "m" in case["cuts"]:
        st["min_p"] = 0.1 * r.chance(n) ** 2
    return st


def prepare(case, seed):
    new = {"device": "cuda"}
    f32 = {"dtype": torch.float32, **new}
    if case["kind"] == "norm":
        t = _norm_inputs(case, seed)
        if "r" in t:
            t["r_out"] = torch.empty_like(t["y"])
        kp = _padded(case["cols"])
        t["codes"], t["scales"] = torch.empty(case["rows"], kp, dtype=F8, **new), torch.empty(case["rows"], kp // BLOCK, **f32)
    elif case["kind"] == "quantize":
        t = _quantize_inputs(case, seed)
        kp = _padded(case["k"])
        t["codes"] = torch.empty(case["n"], kp, dtype=F8, **new)
        t["scales"] = torch.empty(_padded(case["n"]) // BLOCK, kp // BLOCK, **f32)
    elif case["kind"] == "matmul":
        t = _matmul_inputs(case, seed)
        t["c"] = torch.empty(case["m"], case["n"], dtype=DTYPES[case["dtype"]], **new)
    else:
        t = _sample_inputs(case, seed)
        t["tokens"], t["logp"] = torch.empty(case["rows"], dtype=torch.int32, **new), torch.empty(case["rows"], **f32)
    # the pointers and the stream, as a program that drives a C ABI holds them
    return {"case": case, "t": t, "p": {name: v.data_ptr() for name, v in t.items()}, "stream": torch.cuda.current_stream().cuda_stream}


# ---- the framework's calls ----


def _own(case, t, p, stream):
    from ml_framework_amd import capi
    dtype = CODES[case["dtype"]]
    if case["kind"] == "norm":
        n, c = case["rows"], case["cols"]
        capi.call("seera_hip_block_norm_fwd_f8_async", p["y"], p.get("g"), p.get("r"), p.get("w1"), p.get("s"), p.get("w2"), p.get("r_out"), p["codes"],
                  p["scales"], n, c, c, c, EPS, ACTS[case["act"]], dtype, stream)
        return {k: t[k] for k in ("r_out", "codes", "scales") if k in t}
    if case["kind"] == "quantize":
        n, k = case["n"], case["k"]
        capi.call("seera_hip_quantize_weights_f8_async", p["w"], p["codes"], p["scales"], n, k, k if case["transposed"] else n, int(case["transposed"]), dtype, stream)
        return {"codes": t["codes"], "scales": t["scales"]}
    if case["kind"] == "matmul":
        capi.call("seera_hip_matmul_f8_async", p["a"], p["a_scales"], p["w"], p["w_scales"], p.get("bias"), p["c"], case["m"], case["n"], case["k"],
                  case["n"], dtype, stream)
        return t["c"]
    capi.call("seera_hip_sample_async", p["logits"], p["uniform"], p["temperature"], p.get("top_k"), p.get("top_p"), p.get("min_p"), p["tokens"], p["logp"],
              case["rows"], case["vocab"], case["vocab"], dtype, stream)
    return {"tokens": t["tokens"], "logp": t["logp"]}


# ---- the plain form ----


def _codes(v, scale):
    """e4m3 codes of v / scale; 0 where the block has only zeros."""
    return torch.where(scale > 0, v / scale, 0.0).to(F8)


def _quantize_rows(v):
    """Codes and scales, one for each 128 values of a row."""
    rows, k = v.shape
    blocks = torch.nn.functional.pad(v, (0, _padded(k) - k)).view(rows, -1, BLOCK)
    scales = blocks.abs().amax(2) / LARGEST
    return _codes(blocks, scales[..., None]).view(rows, -1), scales


def _quantize_blocks(v):
    """Codes and scales, one for each 128 x 128 values."""
    n, k = v.shape
    blocks = torch.nn.functional.pad(v, (0, _padded(k) - k, 0, _padded(n) - n)).reshape(_padded(n) // BLOCK, BLOCK, -1, BLOCK)
    scales = blocks.abs().amax((1, 3)) / LARGEST
    return _codes(blocks, scales[:, None, :, None]).reshape(_padded(n), -1)[:n].contiguous(), scales


def _norm(case, t):
    dtype, u, out = t["y"].dtype, t["y"].float(), {}
    if "w1" in t:
        u = u * torch.rsqrt(u.square().mean(1, keepdim=True) + EPS) * t["w1"]
    if "g" in t:
        g = t["g"].float()
        u = u * (g * torch.sigmoid(g) if case["act"] == "silu" else torch.sigmoid(g))
    if "s" in t:
        u = u * t["s"]
    if "r" in t:
        u = u + t["r"].float()
    kept = u.to(dtype)
    if "r" in t:
        out["r_out"] = kept
    n = kept.float()  # the next norm is of the residual stream as it is kept
    if "w2" in t:
        n = n * torch.rsqrt(n.square().mean(1, keepdim=True) + EPS) * t["w2"]
    out["codes"], out["scales"] = _quantize_rows(n)
    return out


def _quantize(case, t):
    w = t["w"].float() if case["transposed"] else t["w"].float().t()
    codes, scales = _quantize_blocks(w)
    return {"codes": codes, "scales": scales}


def _matmul(case, t):
    m, n = case["m"], case["n"]
    a = (t["a"].float().view(m, -1, BLOCK) * t["a_scales"][..., None]).view(m, -1)
    w = t["w"].float().view(n, -1, BLOCK) * t["w_scales"].repeat_interleave(BLOCK, 0)[:n, :, None]
    c = a @ w.view(n, -1).t()
    if "bias" in t:
        c = c + t["bias"]
    return c.to(DTYPES[case["dtype"]])


def _sample(case, t):
    """In 64 bits: a cut and a draw both compare a sum of many terms with a border."""
    z, index = torch.sort(t["logits"].float(), dim=1, descending=True, stable=True)
    greedy = t["temperature"] <= 0
    z = (z.double() - z[:, :1].double()) / torch.where(greedy, 1.0, t["temperature"]).double()[:, None]
    w = torch.exp(z)
    keep = torch.ones_like(w, dtype=torch.bool)
    if "top_k" in t:
        keep = torch.arange(case["vocab"], device="cuda")[None, :] < t["top_k"][:, None]
    if "top_p" in t:
        kept = torch.where(keep, w, 0.0)
        before = kept.cumsum(1) - kept
        keep = keep & (before < t["top_p"].double()[:, None] * kept.sum(1, keepdim=True))
    if "min_p" in t:
        keep = keep & (w >= t["min_p"].double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    mass = kept.cumsum(1)
    drawn = (mass <= t["uniform"].double()[:, None] * mass[:, -1:]).sum(1, keepdim=True).clamp_(max=case["vocab"] - 1)
    logp = torch.log(kept.gather(1, drawn) / mass[:, -1:])[:, 0]
    tokens = torch.where(greedy, index[:, 0], drawn[:, 0]).int()
    return {"tokens": tokens, "logp": torch.where(greedy, 0.0, logp).float()}


def run(state):
    case, t = state["case"], state["t"]
    if own:
        return _own(case, t, state["p"], state["stream"])
    return {"norm": _norm, "quantize": _quantize, "matmul": _matmul, "sample": _sample}[case["kind"]](case, t)


# ---- the same in 64 bits ----


def _exact_codes(v, scale):
    """The e4m3 value nearest to v / scale: 4 significant bits, none below 2^-9."""
    x = torch.where(scale > 0, v / torch.where(scale > 0, scale, 1.0), 0.0)
    power = torch.floor(torch.log2(torch.where(x == 0, 1.0, x.abs()))).clamp_(min=-6.0)
    unit = torch.pow(2.0, power - 3)
    return torch.round(x / unit) * unit


def _exact_norm(case, t):
    d = {k: t[k].double() for k in ("y", "g", "r", "w1", "s", "w2") if k in t}

    def rms(v):
        return v / torch.sqrt(v.pow(2).sum(1, keepdim=True) / case["cols"] + EPS)

    u, out = d["y"], {}
    if "w1" in d:
        u = rms(u) * d["w1"]
    if "g" in d:
        u = u / (1 + torch.exp(-d["g"])) * (d["g"] if case["act"] == "silu" else 1.0)
    if "s" in d:
        u = u * d["s"]
    if "r" in d:
        u = out["r_out"] = u + d["r"]
    n = u.to(t["y"].dtype).double()
    if "w2" in d:
        n = rms(n) * d["w2"]
    whole = n.new_zeros(case["rows"], _padded(case["cols"]))
    whole[:, :case["cols"]] = n
    out["scales"] = torch.stack([b.abs().max(1).values for b in whole.split(BLOCK, 1)], 1) / 448
    kept = out["scales"].float().double()  # codes are of the values over the scale as it is kept
    out["codes"] = _exact_codes(whole, kept.repeat_interleave(BLOCK, 1))
    return out


def _exact_quantize(case, t):
    w = t["w"].double()
    w = w if case["transposed"] else w.T
    n, k = w.shape
    whole = w.new_zeros(_padded(n), _padded(k))
    whole[:n, :k] = w
    scales = torch.stack([torch.stack([b.abs().max() for b in row.split(BLOCK, 1)]) for row in whole.split(BLOCK, 0)]) / 448
    kept = scales.float().double()
    return {"codes": _exact_codes(whole, kept.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1))[:n], "scales": scales}


def _exact_matmul(case, t):
    sums = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for b in range(_padded(case["k"]) // BLOCK):
        part = t["a"][:, b * BLOCK:(b + 1) * BLOCK].double() @ t["w"][:, b * BLOCK:(b + 1) * BLOCK].double().T.contiguous()
        part *= t["a_scales"][:, b].double()[:, None]
        part *= t["w_scales"][:, b].double().repeat_interleave(BLOCK)[:case["n"]]
        sums += part
    return sums + t["bias"].double() if "bias" in t else sums


def _exact_sample(case, t):
    """Row by row on the host, by the definition."""
    host = {k: v.float().cpu().numpy().astype(np.float64) for k, v in t.items() if k not in ("tokens", "logp")}
    logp = np.zeros(case["rows"])
    for i, z in enumerate(host["logits"]):
        if host["temperature"][i] <= 0:
            continue
        order = np.argsort(-z, kind="stable")
        w = np.exp((z[order] - z.max()) / host["temperature"][i])
        if "top_k" in host:
            w = w[:int(host["top_k"][i])]
        if "top_p" in host:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), host["top_p"][i] * math.fsum(w))) + 1)]
        if "min_p" in host:
            w = w[w >= host["min_p"][i]]
        chosen = np.sort(order[:len(w)])
        weights = np.exp((z[chosen] - z.max()) / host["temperature"][i])
        mass = np.cumsum(weights)
        at = min(int(np.searchsorted(mass, host["uniform"][i] * mass[-1], side="right")), len(mass) - 1)
        logp[i] = math.log(weights[at] / math.fsum(weights))
    return {"tokens": None, "logp": torch.from_numpy(logp)}


def exact(case, seed):
    t = prepare(case, seed)["t"]
    return {"norm": _exact_norm, "quantize": _exact_quantize, "matmul": _exact_matmul, "sample": _exact_sample}[case["kind"]](case, t)
