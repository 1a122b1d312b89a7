"""Single steps of the decoder over its 8-bit cache ("kv": "q8"), whose rows
find their sequence and position on the device, against the same tokens as a
prompt."""
import numpy as np
import pytest

from trit_b200 import CausalLm

pytestmark = pytest.mark.gpu

NAMES = ["mini_qwen3_q8_0", "mini_mistral_q8_0", "mini_gqa8_q8_0", "mini_mha_q8_0", "mini_granite_q8_0",
         "mini_qwen3_ternary"]


def cosine(a, b):
    a, b = a.astype(np.float64), b.astype(np.float64)
    return float((a * b).sum() / np.sqrt((a * a).sum() * (b * b).sum()))


def near_best(logits, token):
    """Whether a token is the best up to the sums' order."""
    return logits.max() - logits[token] <= 1e-3 * logits.std()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("page", [16, 32])
def test_steps_over_page_borders(mini_models, name, page):
    """A prompt taken a row a pass sees its pages as steps do: f16 until a page is full, codes from then on. It runs as
    rows of known sequence and position, the form that the attention's own tests compare with 64 bits. So the logits
    agree but for the order of sums, and what that moves among the int8 activations; a token or a position less
    moves them more."""
    rng = np.random.default_rng(11)
    prompt = [int(t) for t in rng.integers(0, 2000, 11)]
    with CausalLm.load(mini_models[name], kv="q8", max_context=256, page_tokens=page, prefill_rows=1) as lm:
        toks, logits = lm.generate_traced(prompt, max_new=90)
        for i in (1, page - 12, page - 11, page - 10, 2 * page - 11, 2 * page - 10, 60, 89):
            _, want = lm.generate_traced(prompt + toks[:i], max_new=1)
            assert cosine(logits[i], want[0]) > 0.9999, i
        _, other = lm.generate_traced((prompt + toks[:89])[1:], max_new=1)
        assert cosine(logits[89], other[0]) < 0.9999


@pytest.mark.parametrize("name", NAMES)
def test_steps_of_a_page_that_is_f16(mini_models, name):
    """While no page is full the cache is f16 to the bit: the steps' logits are those of the f16 cache's prompts, a kernel
    of its own that keeps the reference's order. The sums' order moves some int8 activations by a code (1 part in 127
    of a group's largest) in two layers: a cosine over 0.999."""
    rng = np.random.default_rng(12)
    prompt = [int(t) for t in rng.integers(0, 2000, 11)]
    with CausalLm.load(mini_models[name], kv="q8", max_context=128, page_tokens=128) as lm:
        toks, logits = lm.generate_traced(prompt, max_new=100)
    with CausalLm.load(mini_models[name], kv="f16", max_context=128) as lm:
        for i in range(1, 100, 7):
            _, want = lm.generate_traced(prompt + toks[:i], max_new=1)
            assert cosine(logits[i], want[0]) > 0.999, i


@pytest.mark.parametrize("name", NAMES)
def test_steps_of_a_batch(mini_models, name):
    """Streams of several lengths side by side, eagerly once and then as a graph: each token is the best behind the
    stream's own tokens, taken as a prompt a row a pass."""
    rng = np.random.default_rng(13)
    prompts = [[int(t) for t in rng.integers(0, 2000, n)] for n in (3, 15, 7, 1, 12)]
    opts = dict(kv="q8", max_context=128, page_tokens=16)
    with CausalLm.load(mini_models[name], max_streams=5, **opts) as lm:
        made = lm.generate_batch(prompts, max_new=60)
    with CausalLm.load(mini_models[name], prefill_rows=1, **opts) as lm:
        for prompt, toks in zip(prompts, made):
            for i in (0, 1, 2, 16 - len(prompt), 33 - len(prompt), 50, 59):
                _, want = lm.generate_traced(prompt + toks[:i], max_new=1)
                assert near_best(want[0], toks[i]), (len(prompt), i)


@pytest.mark.parametrize("name", NAMES)
def test_steps_with_added_rows(mini_models, name):
    """generate_additive: each token is the best behind the same sums of embeddings and rows as a prompt."""
    rng = np.random.default_rng(14)
    prompt = [int(t) for t in rng.integers(0, 2000, 15)]
    with CausalLm.load(mini_models[name], kv="q8", max_context=128, page_tokens=16, prefill_rows=1) as lm:
        rows = 0.5 * lm.embed([int(t) for t in rng.integers(0, 2000, 70)])
        made = lm.generate_additive(prompt, rows)
        assert len(made) == 56
        for i in (0, 1, 2, 17, 18, 33, 55):
            _, want = lm.answer([], lm.embed(prompt + made[:i]) + rows[:15 + i], [], max_new=1, trace=True)
            assert near_best(want[0], made[i]), i


@pytest.mark.parametrize("name", NAMES)
def test_rows_without_order(mini_models, name):
    """bidirectional_tokens in one page (f16 to the bit) and over many: the f16 cache's tokens but for near ties, of which
    codes (1 % of a value) make more."""
    rng = np.random.default_rng(15)
    for n, page, least in ((90, 128, 0.9), (200, 16, 0.75)):
        with CausalLm.load(mini_models[name], kv="f16", max_context=256) as lm:
            rows = lm.embed([int(t) for t in rng.integers(0, 2000, n)])
            want = lm.bidirectional_tokens(rows, 3)
        with CausalLm.load(mini_models[name], kv="q8", max_context=256, page_tokens=page) as lm:
            got = lm.bidirectional_tokens(rows, 3)
        assert np.mean(np.array(got) == np.array(want)) >= least
