"""PagedRunner.verify with a draft whose accepted branch is known."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200.model import CudaQwen  # noqa: E402
from harsh4b_b200.paged import PagedCache, PagedRunner  # noqa: E402
from harsh4b_b200.synthetic import synthetic_checkpoint, synthetic_prompt, tiny_config  # noqa: E402


def test_sure_tokens_are_accepted():
    """Prompts whose greedy tokens lead by more than the two ways' logits may differ (4 % of a row's norm per sqrt(vocab)
    each, twice): the tree's branch of these tokens is accepted whole."""
    model = CudaQwen.from_checkpoint(synthetic_checkpoint(tiny_config(), seed=7), kv_dtype="float16")
    cache = PagedCache.for_model(model, pages=64)
    runner = PagedRunner(model, cache, max_tokens=128)
    sure = 0
    for seed in range(40):
        prompt = [int(t) for t in synthetic_prompt(model.config, 50, seed=seed)]
        s = cache.new_sequence()
        runner.step({s: prompt[:-1]})
        fork, feed, chain, clear = cache.fork(s), prompt[-1], [], True
        for _ in range(3):
            logits = runner.step({fork: [feed]})[fork].double()
            best = logits.topk(2)
            clear &= bool(best.values[0] - best.values[1] > 2 * 0.04 * logits.norm() / math.sqrt(logits.numel()))
            feed = int(best.indices[0])
            chain.append(feed)
        cache.free(fork)
        if clear:
            wrong = [(t + 1) % model.vocab for t in chain]
            tokens = [prompt[-1], wrong[0], chain[0], chain[1], wrong[1], chain[1], wrong[2]] + [chain[0]] * 60
            parents = [-1, 0, 0, 1, 2, 2, 5] + [0] * 60
            got = runner.verify({s: (tokens, parents)})[s]
            assert got == chain and cache.length(s) == 49 + 3
            assert cache.pages - cache.free_pages == len(cache.table(s)) == 4
            sure += 1
        cache.free(s)
        if sure == 3:
            break
    runner.status()
    assert sure == 3
