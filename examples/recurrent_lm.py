"""A small recurrent language model trained on text and then run character by
character, on the ``seera_cuda`` module alone.

    python examples/recurrent_lm.py            # trains for a few seconds, then prints what the model writes

Each block is

    [x | f | g] = n W_in             one projection (cuda_matmul)
    h = gated scan of x by f         cuda_gated_scan_fwd, reading two slices of the projection
    y = h W_out                      cuda_matmul
    r, n = block norm of y, g, r     cuda_block_norm_fwd: norm after the block, gate, residual scale,
                                     residual, and the next block's norm

and the step is cuda_adamw_step over all tensors: the products' weights with
8-bit states, the norms' with 32-bit ones.
"""
from __future__ import annotations

import os
import sys

import numpy as np

if __package__ in (None, ""):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import ml_framework_amd

TEXT = ("the scan carries a state from each step to the next. the gate says how much of it stays. "
        "the norm keeps the stream of the residual in bounds. the step moves every weight a little. ")
EPS = 1e-6


class Buffers:
    """Device memory by name."""

    def __init__(self, sc):
        self.sc, self.ptr, self.shape = sc, {}, {}

    def new(self, name, shape, value=None):
        shape = tuple(int(n) for n in shape)
        if name in self.ptr:
            self.sc.cuda_free(self.ptr[name])
        if value is None:
            self.ptr[name] = self.sc.cuda_zeros_f(int(np.prod(shape)))
        else:
            self.ptr[name] = self.sc.to_device_f32(np.ascontiguousarray(value, np.float32))
        self.shape[name] = shape
        return self.ptr[name]

    def __getitem__(self, name):
        return self.ptr[name]

    def host(self, name):
        return self.sc.to_host_f32(self.ptr[name], self.shape[name])

    def close(self):
        for p in self.ptr.values():
            self.sc.cuda_free(p)
        self.ptr.clear()


class RecurrentLM:
    def __init__(self, vocab, width=64, blocks=2, seed=0):
        self.sc = ml_framework_amd.seera_cuda()
        self.vocab, self.width, self.blocks = vocab, width, blocks
        self.weights, self.work = Buffers(self.sc), Buffers(self.sc)
        r = np.random.default_rng(seed)
        c = width

        def matrix(rows, cols):
            return r.standard_normal((rows, cols)) / np.sqrt(rows)

        shapes = {"embed": r.standard_normal((vocab, c)) * 0.5, "first": np.ones(c), "head": matrix(c, vocab)}
        for i in range(blocks):
            shapes[f"in{i}"], shapes[f"out{i}"] = matrix(c, 3 * c), matrix(c, c)
            shapes[f"after{i}"], shapes[f"scale{i}"], shapes[f"before{i}"] = np.ones(c), np.full(c, 0.5), np.ones(c)
        self.tensors = []
        for name, value in shapes.items():
            self.weights.new(name, value.shape, value)
            self.weights.new("d_" + name, value.shape)
            t = self.sc.AdamwTensor()
            t.param, t.grad, t.count = self.weights[name], self.weights["d_" + name], value.size
            t.state_bits = 8 if value.ndim == 2 else 32
            t.weight_decay = 0.01 if value.ndim == 2 else 0.0
            # zero bytes are zeros in both forms; one value's four bytes hold four codes or exponents
            t.m, t.v = self.weights.new("m_" + name, value.shape), self.weights.new("v_" + name, value.shape)
            blocks128 = (value.size + 127) // 128
            t.m_exp, t.v_exp = self.weights.new("me_" + name, (blocks128,)), self.weights.new("ve_" + name, (blocks128,))
            self.tensors.append(t)
        self.steps = 0

    def _room(self, batch, time):
        """Buffers for batch x time rows."""
        if getattr(self, "_rows", None) == (batch, time):
            return
        self._rows = (batch, time)
        n, c, v = batch * time, self.width, self.vocab
        for name in ("onehot", "logits", "prob", "d_logits", "d_onehot"):
            self.work.new(name, (n, v))
        for name in ("r0", "n0", "d_emb", "d_y", "d_h", "d_n", "d_r", "d_r2"):
            self.work.new(name, (n, c))
        self.work.new("s2_first", (n,))
        for i in range(self.blocks):
            self.work.new(f"proj{i}", (n, 3 * c))
            self.work.new(f"d_proj{i}", (n, 3 * c))
            for name in (f"h{i}", f"y{i}", f"r{i + 1}", f"n{i + 1}"):
                self.work.new(name, (n, c))
            for name in (f"s1_{i}", f"s2_{i}"):
                self.work.new(name, (n,))

    def forward(self, tokens, states=None):
        """Logits (on the device) of tokens [batch, time]. `states`: a device pointer
        to [batch, width] for each block, read and moved on."""
        sc, w, b = self.sc, self.weights, self.work
        batch, time = tokens.shape
        self._room(batch, time)
        n, c, v = batch * time, self.width, self.vocab
        b.new("onehot", (n, v), np.eye(v, dtype=np.float32)[tokens.reshape(-1)])
        sc.cuda_matmul(b["onehot"], w["embed"], b["r0"], n, c, v, 1)
        sc.cuda_block_norm_fwd(b["r0"], 0, 0, 0, 0, w["first"], 0, b["n0"], 0, b["s2_first"], n, c, c, c, EPS, sc.GATE_ACT_SILU, sc.DTYPE_F32)
        for i in range(self.blocks):
            proj = b[f"proj{i}"]
            x, f, g = proj, proj + 4 * c, proj + 8 * c  # slices of rows that lie 3 c apart
            state = states[i] if states else 0
            sc.cuda_matmul(b[f"n{i}"], w[f"in{i}"], proj, n, 3 * c, c, 1)
            sc.cuda_gated_scan_fwd(x, f, state, 0, b[f"h{i}"], state, batch, time, c, 3 * c, 3 * c, sc.GATE_SIGMOID, 0, sc.DTYPE_F32)
            sc.cuda_matmul(b[f"h{i}"], w[f"out{i}"], b[f"y{i}"], n, c, c, 1)
            sc.cuda_block_norm_fwd(b[f"y{i}"], g, b[f"r{i}"], w[f"after{i}"], w[f"scale{i}"], w[f"before{i}"], b[f"r{i + 1}"], b[f"n{i + 1}"],
                                   b[f"s1_{i}"], b[f"s2_{i}"], n, c, c, 3 * c, EPS, sc.GATE_ACT_SILU, sc.DTYPE_F32)
        sc.cuda_matmul(b[f"n{self.blocks}"], w["head"], b["logits"], n, v, c, 1)
        return b["logits"]

    def train_step(self, tokens, targets, lr):
        """One step; the mean cross entropy before it."""
        sc, w, b = self.sc, self.weights, self.work
        batch, time = tokens.shape
        n, c, v = batch * time, self.width, self.vocab
        self.forward(tokens)
        sc.cuda_softmax_fwd(b["logits"], b["prob"], n, v)
        prob = b.host("prob")
        loss = -np.log(np.maximum(prob[np.arange(n), targets.reshape(-1)], 1e-30)).mean()
        b.new("target", (n, v), np.eye(v, dtype=np.float32)[targets.reshape(-1)])
        sc.cuda_elemsub(b["prob"], b["target"], b["d_logits"], n * v)
        sc.cuda_scaler_multiply_f(b["d_logits"], 1.0 / n, n * v)
        sc.cuda_matmul_bwd(b[f"n{self.blocks}"], w["head"], b["d_logits"], b["d_n"], w["d_head"], n, v, c, 1)
        above, below = 0, b["d_r"]  # gradients of the residual stream; none comes from above the last block
        for i in reversed(range(self.blocks)):
            proj, d_proj = b[f"proj{i}"], b[f"d_proj{i}"]
            sc.cuda_block_norm_bwd(b[f"y{i}"], proj + 8 * c, b[f"r{i + 1}"], w[f"after{i}"], w[f"scale{i}"], w[f"before{i}"], b[f"s1_{i}"], b[f"s2_{i}"],
                                   above, b["d_n"], b["d_y"], d_proj + 8 * c, below, w[f"d_after{i}"], w[f"d_scale{i}"], w[f"d_before{i}"],
                                   n, c, c, 3 * c, c, 3 * c, sc.GATE_ACT_SILU, sc.DTYPE_F32)
            sc.cuda_matmul_bwd(b[f"h{i}"], w[f"out{i}"], b["d_y"], b["d_h"], w[f"d_out{i}"], n, c, c, 1)
            sc.cuda_gated_scan_bwd(proj, proj + 4 * c, 0, 0, b[f"h{i}"], b["d_h"], 0, d_proj, d_proj + 4 * c, 0, batch, time, c,
                                   3 * c, 3 * c, 3 * c, 3 * c, sc.GATE_SIGMOID, 0, sc.DTYPE_F32)
            sc.cuda_matmul_bwd(b[f"n{i}"], w[f"in{i}"], d_proj, b["d_n"], w[f"d_in{i}"], n, 3 * c, c, 1)
            above, below = below, b["d_r2"] if below == b["d_r"] else b["d_r"]
        sc.cuda_block_norm_bwd(0, 0, b["r0"], 0, 0, w["first"], 0, b["s2_first"], above, b["d_n"], b["d_emb"], 0, 0, 0, 0, w["d_first"],
                               n, c, c, c, c, c, sc.GATE_ACT_SILU, sc.DTYPE_F32)
        sc.cuda_matmul_bwd(b["onehot"], w["embed"], b["d_emb"], b["d_onehot"], w["d_embed"], n, c, v, 1)
        self.steps += 1
        sc.cuda_adamw_step(self.tensors, lr, 0.9, 0.99, 1e-8, self.steps, self.steps, 0)
        return float(loss)

    def generate(self, prompt, count):
        """Greedy continuation of a prompt, one token a call with carried states."""
        c, v = self.width, self.vocab
        states = [self.sc.cuda_zeros_f(c) for _ in range(self.blocks)]
        out = list(prompt)
        for i in range(len(prompt) + count - 1):
            self.forward(np.array([[out[i]]]), states)
            if i + 1 >= len(prompt):
                out.append(int(self.work.host("logits").reshape(v).argmax()))
        for p in states:
            self.sc.cuda_free(p)
        return out

    def close(self):
        self.weights.close()
        self.work.close()


def batches(text, batch, time, seed=0):
    """Random windows of the (circular) text and their next characters."""
    letters = sorted(set(text))
    codes = np.array([letters.index(ch) for ch in text])
    r = np.random.default_rng(seed)
    while True:
        at = (r.integers(0, len(codes), (batch, 1)) + np.arange(time + 1)) % len(codes)
        yield codes[at[:, :-1]], codes[at[:, 1:]]


def main(steps=250):
    letters = sorted(set(TEXT))
    model = RecurrentLM(len(letters))
    try:
        for i, (tokens, targets) in zip(range(steps), batches(TEXT, 16, 64)):
            loss = model.train_step(tokens, targets, 3e-3 * min(1.0, 4 * (1 - i / steps)))
            if i % 50 == 0 or i == steps - 1:
                print(f"step {i:4d}  loss {loss:.4f}", flush=True)
        start = [letters.index(ch) for ch in TEXT[:12]]
        print("".join(letters[k] for k in model.generate(start, 160)))
    finally:
        model.close()


if __name__ == "__main__":
    main()
