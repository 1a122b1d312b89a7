"""The decoder's batches over its 8-bit cache ("kv": "q8"): an answer does not
depend on the batches before it."""
import numpy as np
import pytest

from trit_b200 import CausalLm

pytestmark = pytest.mark.gpu


def test_a_batch_after_a_longer_one(mini_models):
    """The steps of a batch are recorded once and replayed. A longer batch cuts its positions into more shares; the same
    batch before and after it has the same tokens, over steps enough for another order of sums to show."""
    rng = np.random.default_rng(7)
    S = 24
    short = [[int(t) for t in rng.integers(0, 4000, 5 + i)] for i in range(S)]
    long = [[int(t) for t in rng.integers(0, 4000, 1500)]] + short[1:]
    opts = dict(kv="q8", max_context=2048, page_tokens=16, max_streams=S)
    with CausalLm.load(mini_models["mini_qwen3_q8_0"], **opts) as lm:
        first = lm.generate_batch(short, max_new=400)
        lm.generate_batch(long, max_new=402)
        second = lm.generate_batch(short, max_new=400)
    assert first == second
