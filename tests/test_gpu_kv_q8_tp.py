"""The decoder's 8-bit cache ("kv": "q8") with two-way tensor parallelism, one
process a GPU: each rank caches its own key/value heads, so the tokens are
those of one GPU but for near ties. Skipped with fewer than two GPUs."""
import numpy as np
import pytest
import torch.multiprocessing as mp

from tests.test_gpu_tp import MODEL, collect, finish

pytestmark = pytest.mark.gpu


def rank_main(rank, path, tp_id, prompts, queue):
    from trit_b200 import CausalLm

    try:
        with CausalLm.load(path, device=rank, kv="q8", max_context=128, page_tokens=16, max_streams=len(prompts), tp_size=2,
                           tp_rank=rank, tp_id=tp_id, tp_timeout_s=60) as lm:
            queue.put((rank, lm.generate_batch(prompts, max_new=40), lm.generate(prompts[0], max_new=40), None))
    except Exception as e:  # reported to the test, which fails on it
        queue.put((rank, None, None, repr(e)))


def test_two_ranks(mini_models):
    """Each rank's tokens are the other's, and the best, up to the order of sums, behind the same tokens on one GPU."""
    torch = pytest.importorskip("torch")
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from trit_b200 import CausalLm, lm

    path = mini_models[MODEL]
    rng = np.random.default_rng(51)
    prompts = [[int(t) for t in rng.integers(0, 2000, n)] for n in (3, 15, 7)]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    tp_id = lm.tp_id()
    procs = [ctx.Process(target=rank_main, args=(r, path, tp_id, prompts, queue)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = collect(queue, procs, 2, 240)
    finally:
        finish(procs)
    errors = {r: g[3] for r, g in got.items() if g[3]}
    assert not errors and sorted(got) == [0, 1], f"rank errors: {errors}; reported: {sorted(got)}"
    assert got[0][1:] == got[1][1:]
    with CausalLm.load(path, kv="q8", max_context=128, page_tokens=16, prefill_rows=1) as one:
        for prompt, toks in zip(prompts + prompts[:1], got[0][1] + [got[0][2]]):
            for i in (0, 1, 20, 39):
                _, want = one.generate_traced(prompt + toks[:i], max_new=1)
                # Partial products are summed in another order: int8 activations move by a code here and there.
                assert want[0].max() - want[0][toks[i]] <= 0.1 * want[0].std(), i
