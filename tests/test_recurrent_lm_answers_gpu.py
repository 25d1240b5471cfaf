"""examples/recurrent_lm.py answering in 8 bits, through the seera_cuda module."""
import numpy as np
import pytest

from examples import recurrent_lm as lm
from ml_framework_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [32, 200])
def test_answers(width):
    assert capi.gpu_available(), "no HIP device visible"
    model = lm.RecurrentLM(11, width=width, blocks=2, seed=1)
    try:
        r = np.random.default_rng(2)
        tokens = r.integers(0, 11, (3, 21))
        model.train_step(tokens, tokens, 1e-3)
        model.to_8_bits()
        prompt = [1, 2, 3]
        first = model.answer(prompt, 20, seed=4)
        assert len(first) == 23 and first[:3] == prompt and all(0 <= t < 11 for t in first)
        assert model.answer(prompt, 20, seed=4) == first
        # a temperature of 0, top_k 1 and top_p 0 all take the largest logit
        greedy = model.answer(prompt, 20, temperature=0.0)
        assert model.answer(prompt, 20, top_k=1, seed=5) == greedy and model.answer(prompt, 20, top_p=0.0, seed=6) == greedy
        assert len(set(map(tuple, (model.answer(prompt, 20, temperature=3.0, top_p=1.0, seed=s) for s in range(5))))) > 1
        model.train_step(tokens, tokens, 1e-3)  # training goes on from the fp32 weights
        model.to_8_bits()
        assert len(model.answer(prompt, 3)) == 6
    finally:
        model.close()


def test_module_refusals():
    import ml_framework_amd

    sc = ml_framework_amd.seera_cuda()
    with pytest.raises(RuntimeError, match="null"):
        sc.cuda_matmul_f8(0, 0, 0, 0, 0, 0, 1, 1, 1, 1, 0)
    with pytest.raises(RuntimeError, match="above"):
        sc.cuda_block_norm_fwd_f8(0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 20000, 20000, 20000, 1e-6, 0, 0)
    with pytest.raises(RuntimeError, match="ldw"):
        sc.cuda_quantize_weights_f8(0, 0, 0, 8, 8, 7, 0, 0)
    with pytest.raises(RuntimeError, match="dims"):
        sc.cuda_sample(0, 0, 0, 0, 0, 0, 0, 0, -1, 1, 1, 0)
