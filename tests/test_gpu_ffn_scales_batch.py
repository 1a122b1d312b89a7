"""CausalLm.set_ffn_scales between batches, whose steps are a recorded graph that later batches of the same size replay."""
import numpy as np
import pytest

from oracle import oracle as O
from trit_b200 import CausalLm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["mini_qwen3_q8_0", "mini_qwen3_ternary"])
def test_batches_between_scales(mini_models, name):
    path = mini_models[name]
    oracle = O.Oracle(path)
    rng = np.random.default_rng(43)
    prompts = [rng.integers(0, oracle.vocab, size=9 + i).tolist() for i in range(3)]
    sets = [rng.uniform(0.2, 2.0, (2, oracle.width)).astype(np.float32) for _ in range(2)]
    with CausalLm.load(path, kv="f32", max_context=64, max_streams=3) as lm:
        for scales in (None, sets[0], sets[1], None, None, sets[0]):
            oracle.set_ffn_scales(scales)
            lm.set_ffn_scales(scales)
            got = lm.generate_batch(prompts, max_new=12)
            assert got == [oracle.generate(p, 12)["tokens"] for p in prompts]
