"""examples/recurrent_lm.py: the scan, the block norm and the AdamW step together,
through the seera_cuda module. The whole model's gradient against differences of
its loss, the loss over training, and generation token by token against the whole
sequence."""
import numpy as np
import pytest

from examples import recurrent_lm as lm
from ml_framework_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture
def model():
    assert capi.gpu_available(), "no HIP device visible"
    m = lm.RecurrentLM(11, width=32, blocks=2, seed=1)
    yield m
    m.close()


def _loss(model, tokens, targets):
    model.forward(tokens)
    z = model.work.host("logits").astype(np.float64)
    z -= z.max(1, keepdims=True)
    return (np.log(np.exp(z).sum(1)) - z[np.arange(len(z)), targets.reshape(-1)]).mean()


def test_gradients_against_differences(model):
    """Along a random direction of each kind of weight. The products round their
    operands to fp16 (2^-11): the slope of the loss is right to about that share of
    its magnitude, and a difference over a step of 0.05 adds the third derivative's."""
    r = np.random.default_rng(2)
    tokens, targets = r.integers(0, 11, (3, 21)), r.integers(0, 11, (3, 21))
    names = ["embed", "first", "in0", "out0", "after0", "scale0", "before0", "in1", "after1", "scale1", "before1", "head"]
    start = {k: model.weights.host(k) for k in names}
    model.train_step(tokens, targets, 0.0)
    for name in names:
        grad = model.weights.host("d_" + name).astype(np.float64)
        d = grad / np.linalg.norm(grad)  # along the gradient the slope is its norm
        step, ends = 0.05, []
        for sign in (1, -1):
            model.weights.new(name, start[name].shape, start[name] + sign * step * d)
            ends.append(_loss(model, tokens, targets))
        model.weights.new(name, start[name].shape, start[name])
        slope = (ends[0] - ends[1]) / (2 * step)
        assert abs(slope - np.linalg.norm(grad)) <= 0.03 * np.linalg.norm(grad) + 1e-4, (name, slope, np.linalg.norm(grad))


def test_it_learns_and_writes_the_text():
    letters = sorted(set(lm.TEXT))
    codes = [letters.index(ch) for ch in lm.TEXT]
    model = lm.RecurrentLM(len(letters))
    try:
        losses = [model.train_step(*b, 3e-3) for _, b in zip(range(250), lm.batches(lm.TEXT, 16, 64))]
        assert losses[0] > 2.5 and losses[-1] < 0.5, (losses[0], losses[-1])
        # one call for the whole sequence, and one call a token
        whole = np.array([codes[:40]])
        model.forward(whole)
        want = model.work.host("logits")
        c = model.width
        states = [model.sc.cuda_zeros_f(c) for _ in range(model.blocks)]
        steps = []
        for t in range(40):
            model.forward(whole[:, t:t + 1], states)
            steps.append(model.work.host("logits")[0])
        for p in states:
            model.sc.cuda_free(p)
        # the same products on the same operands but for fp32 roundings before fp16 ones
        assert np.abs(np.array(steps) - want).max() <= 2e-2 * np.abs(want).max()
        assert np.array_equal(np.array(steps).argmax(1), want.argmax(1))
    finally:
        model.close()


def test_module_refusals():
    import ml_framework_amd

    sc = ml_framework_amd.seera_cuda()
    t = sc.AdamwTensor()
    t.count, t.state_bits = 4, 32
    with pytest.raises(RuntimeError, match="null"):
        sc.cuda_adamw_step([t], 1e-3, 0.9, 0.999, 1e-8, 1, 0, 0)
    with pytest.raises(ValueError, match="one pointer"):
        sc.cuda_adamw_state_values([t], [], [0])
    with pytest.raises(RuntimeError, match="dims"):
        sc.cuda_gated_scan_fwd(0, 0, 0, 0, 0, 0, -1, 1, 1, 1, 1, 0, 0, 0)
    with pytest.raises(RuntimeError, match="above"):
        sc.cuda_block_norm_fwd(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 20000, 20000, 20000, 1e-6, 0, 0)
