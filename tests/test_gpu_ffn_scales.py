"""CausalLm.set_ffn_scales with a call right behind it."""
import numpy as np
import pytest

from oracle import oracle as O
from trit_b200 import CausalLm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("decode", ["persistent", "layered"])
def test_call_right_behind(mini_models, decode):
    """Every call sees the scales set just before it, whole."""
    path = mini_models["mini_qwen3_q8_0"]
    oracle = O.Oracle(path)
    rng = np.random.default_rng(41)
    prompt = rng.integers(0, oracle.vocab, size=8).tolist()
    sets = [rng.uniform(0.2, 2.0, (2, oracle.width)).astype(np.float32) for _ in range(3)] + [None]
    want = []
    for scales in sets:
        oracle.set_ffn_scales(scales)
        want.append(oracle.generate(prompt, 4)["tokens"])
    with CausalLm.load(path, kv="f32", decode=decode, max_context=64) as lm:
        for turn in range(20):
            for scales, tokens in zip(sets, want):
                lm.set_ffn_scales(scales)
                assert lm.generate(prompt, max_new=4) == tokens
