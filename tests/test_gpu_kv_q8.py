"""The decoder with its cache in 8 bits ("kv": "q8")."""
import numpy as np
import pytest

from oracle import oracle as O
from trit_b200 import CausalLm, TritError

pytestmark = pytest.mark.gpu


def cosine(a, b):
    a, b = a.astype(np.float64), b.astype(np.float64)
    return (a * b).sum(-1) / np.sqrt((a * a).sum(-1) * (b * b).sum(-1))


@pytest.mark.parametrize("name", ["mini_qwen3_q8_0", "mini_mistral_q8_0", "mini_gqa8_q8_0", "mini_mha_q8_0",
                                  "mini_granite_q8_0", "mini_qwen3_ternary"])
def test_logits_near_the_reference(mini_models, name):
    """The first token's logits behind a prompt of several pages. A code is off by half a step of max|x| / 127: about 1 %
    of a value's size (the largest of a page's 2048 to 8192 normal values is about four times their deviation, a
    uniform error of a step deviates by 0.29 steps). Scores and outputs of two layers each carry it, so logits turn by a
    few parts in a hundred at most: cosine over 0.99 leaves room for the int8 activations that move with them."""
    rng = np.random.default_rng(3)
    path = mini_models[name]
    oracle = O.Oracle(path)
    for n in (5, 150, 300):
        prompt = [int(t) for t in rng.integers(0, 2000, n)]
        want = oracle.generate(prompt, 1, trace=True)
        with CausalLm.load(path, kv="q8", max_context=512, page_tokens=32) as lm:
            assert lm.status()["kv"] == "q8" and lm.status()["decode"] == "layered"
            _, logits = lm.generate_traced(prompt, max_new=1)
        assert cosine(logits[0], want["logits"][0]) > 0.99


def test_prefixes_streams_and_chunks(mini_models):
    """A prefix (whole and partial pages), prompts cut into passes, and streams side by side. A row reads the page it is in
    as f16 or as codes by whether the page had filled when its pass ran, so these agree with a plain call as the
    cache agrees with the reference (see above), and with themselves to the bit."""
    rng = np.random.default_rng(4)
    prompt = [int(t) for t in rng.integers(0, 4000, 200)]
    path = mini_models["mini_qwen3_q8_0"]
    opts = dict(kv="q8", max_context=400, page_tokens=16)
    with CausalLm.load(path, max_streams=3, **opts) as lm:
        toks, plain = lm.generate_traced(prompt, max_new=12)
        again, same = lm.generate_traced(prompt, max_new=12)
        assert again == toks and np.array_equal(same, plain)
        for cut in (7, 16, 100, 160):
            used = lm.prefix_pages()[0]
            p = lm.prefix(prompt[:cut])
            assert lm.prefix_pages()[0] == used + cut // 16
            _, logits = lm.generate_traced(prompt, prefix=p, max_new=1)
            assert cosine(logits[0], plain[0]) > 0.99
            a = lm.generate_batch([prompt, prompt[:cut] + [5, 6], [9] * 40], max_new=8, prefix=p)
            b = lm.generate_batch([prompt, prompt[:cut] + [5, 6], [9] * 40], max_new=8, prefix=p)
            assert a == b and all(len(x) == 8 for x in a)
            p.close()
            assert lm.prefix_pages()[0] == used
        rows = lm.embed(prompt)
        assert lm.generate_rows(rows, max_new=12) == toks
    with CausalLm.load(path, prefill_rows=48, **opts) as lm:
        _, logits = lm.generate_traced(prompt, max_new=1)
        assert cosine(logits[0], plain[0]) > 0.99
        assert len(lm.generate_additive(prompt[:20], rows[:60])) == 41
    with CausalLm.load(path, kv="q8", max_context=400) as lm:
        assert len(lm.bidirectional_tokens(rows[:90], 3)) == 87


def test_a_page_of_positions_is_f16(mini_models):
    """While no page is full the cache is f16 to the bit, so the first logits are those of the f16 cache up to the order
    of sums."""
    path = mini_models["mini_qwen3_q8_0"]
    prompt = list(range(30, 90))
    with CausalLm.load(path, kv="f16", max_context=128) as lm:
        _, want = lm.generate_traced(prompt, max_new=1)
    with CausalLm.load(path, kv="q8", max_context=128, page_tokens=128) as lm:
        _, got = lm.generate_traced(prompt, max_new=1)
    assert cosine(got[0], want[0]) > 0.9999


def test_many_prefixes_are_refused(mini_models):
    with CausalLm.load(mini_models["mini_qwen3_q8_0"], kv="q8", max_context=64) as lm:
        kept = [lm.prefix([1, 2, 3]) for _ in range(16)]
        with pytest.raises(TritError, match="are free"):
            lm.prefix([1, 2, 3])
        kept.pop().close()
        kept.append(lm.prefix([4, 5]))
        assert len(lm.generate([4, 5, 6], prefix=kept[-1], max_new=4)) == 4
