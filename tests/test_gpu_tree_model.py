"""PagedRunner.verify: a step of the model over drafted trees.

Logits tolerance: as derived in test_gpu_paged_model.py, 2 % of a row's norm
against the exact single-session path (fp16 cache)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200.model import CudaQwen  # noqa: E402
from harsh4b_b200.paged import PagedCache, PagedRunner  # noqa: E402
from harsh4b_b200.synthetic import synthetic_checkpoint, synthetic_prompt, tiny_config  # noqa: E402
from test_gpu_paged_model import exact, off  # noqa: E402


@pytest.fixture(scope="module")
def model():
    return CudaQwen.from_checkpoint(synthetic_checkpoint(tiny_config(), seed=7), kv_dtype="float16")


def branch(parents, node):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


def test_every_node_has_the_logits_of_its_branch(model):
    prompts = [[int(t) for t in synthetic_prompt(model.config, n, seed=n)] for n in (70, 33)]
    cache = PagedCache.for_model(model, pages=64)
    runner = PagedRunner(model, cache, max_tokens=128)
    a, b = cache.new_sequence(), cache.new_sequence()
    runner.step({a: prompts[0], b: prompts[1]})
    trees = {a: ([5, 9, 11, 9, 7, 2, 3, 8], [-1, 0, 0, 1, 1, 2, 5, 5]), b: ([17, 4, 6], [-1, 0, 1])}
    got = runner.verify(trees)
    runner.status()
    first = 0
    for s, prompt in ((a, prompts[0]), (b, prompts[1])):
        tokens, parents = trees[s]
        for node in range(len(tokens)):
            ids = prompt + [tokens[i] for i in branch(parents, node)]
            assert off(runner.node_logits[first + node], exact(model, ids)) < 0.02
        greedy = runner.node_logits[first:first + len(tokens)].argmax(-1).tolist()
        path = [0]
        while True:  # the branch that agrees with these logits
            more = [i for i, p in enumerate(parents) if p == path[-1] and tokens[i] == greedy[path[-1]]]
            if not more:
                break
            path.append(more[0])
        assert got[s] == [greedy[i] for i in path]
        assert cache.length(s) == len(prompt) + len(path)
        first += len(tokens)


def test_a_tree_that_holds_the_greedy_tokens_is_accepted(model):
    """Two rounds with trees of which one branch is what the model says, at changing places, beside an ordinary step; what
    stays in the cache is what a session of the accepted tokens has."""
    prompt = [int(t) for t in synthetic_prompt(model.config, 60, seed=3)]
    cache = PagedCache.for_model(model, pages=64)
    runner = PagedRunner(model, cache, max_tokens=128)
    s, other = cache.new_sequence(), cache.new_sequence()
    runner.step({s: prompt[:-1], other: prompt[:20]})
    ids, next_token = prompt[:-1], prompt[-1]
    for turn in range(2):
        # the greedy continuation, found by single steps on a fork
        fork, feed, chain = cache.fork(s), next_token, []
        for _ in range(4):
            feed = int(runner.step({fork: [feed]})[fork].argmax())
            chain.append(feed)
        cache.free(fork)
        wrong = [(t + 1) % model.vocab for t in chain]
        if turn == 0:  # right tokens at nodes 2, 5, 6
            tokens, parents = [next_token, wrong[0], chain[0], 3, wrong[1], chain[1], chain[2], 4], [-1, 0, 0, 1, 2, 2, 5, 5]
            nodes = [0, 2, 5, 6]
        else:  # at 1, 3
            tokens, parents = [next_token, chain[0], wrong[0], chain[1], wrong[1]], [-1, 0, 0, 1, 1]
            nodes = [0, 1, 3]
        got = runner.verify({s: (tokens, parents)})[s]
        # (the logits' roundings differ between the two ways: a token may be another one only within the tolerance)
        logits = runner.node_logits[nodes]
        same = [int(row.argmax()) == t for row, t in zip(logits, chain)]
        for row, t in zip(logits, chain):
            assert row[t] >= row.max() - 0.04 * row.norm() / np.sqrt(row.numel())
        upto = same.index(False) if False in same else len(same)
        assert got[:upto] == chain[:upto] and len(got) >= min(upto + 1, len(nodes))
        ids, next_token = ids + [next_token] + got[:-1], got[-1]
        assert cache.length(s) == len(ids)
    logits = runner.step({s: [next_token], other: prompt[20:25]})
    runner.status()
    assert off(logits[s], exact(model, ids + [next_token])) < 0.02
    assert off(logits[other], exact(model, prompt[:25])) < 0.02


def test_verify_of_one_node_is_a_step(model):
    prompt = [int(t) for t in synthetic_prompt(model.config, 40, seed=5)]
    cache = PagedCache.for_model(model, pages=32)
    runner = PagedRunner(model, cache, max_tokens=64)
    s = cache.new_sequence()
    runner.step({s: prompt})
    t = cache.fork(s)
    logits = runner.step({s: [9]})[s].clone()
    got = runner.verify({t: ([9], [-1])})[t]
    assert torch.equal(runner.node_logits[0], logits) and got == [int(logits.argmax())]
    assert cache.length(t) == cache.length(s)


def test_window_and_shared_pages(model):
    """Trees of forks that share the prompt's last page, under a window that passes pages."""
    prompt = [int(t) for t in synthetic_prompt(model.config, 200, seed=6)]
    cache = PagedCache.for_model(model, pages=40)
    runner = PagedRunner(model, cache, max_tokens=64, window=50, sinks=2)
    s = cache.new_sequence()
    for start in range(0, 200, 50):
        runner.step({s: prompt[start:start + 50]})
    forks = [cache.fork(s) for _ in range(3)]
    chain = runner.step({forks[0]: [1]})
    single = {f: runner.step({f: [k + 2]})[f].clone() for k, f in enumerate(forks[1:])}
    again = [cache.fork(s) for _ in range(2)]
    runner.verify({f: ([k + 2, 7, 8], [-1, 0, 0]) for k, f in enumerate(again)})
    runner.status()
    assert torch.isfinite(chain[forks[0]]).all()
    for k, f in enumerate(forks[1:]):
        assert off(runner.node_logits[3 * k], single[f]) < 0.02
    assert all(cache.length(f) >= 201 for f in again)


def test_refusals(model):
    cache = PagedCache.for_model(model, pages=40)
    runner = PagedRunner(model, cache, max_tokens=300, max_sequences=2)
    s = cache.new_sequence()
    for draft in (([], []), ([1, 2], [-1]), ([1, 2], [-1, 1]), ([1, 2], [-1, -1]), ([1, 2], [0, 0]), ([1], [-2]),
                  ([-1], [-1]), ([model.vocab], [-1]), ([1] * 257, [-1] + list(range(256)))):
        with pytest.raises(ValueError):
            runner.verify({s: draft})
    with pytest.raises(ValueError):
        runner.verify({})
    assert cache.length(s) == 0 and cache.free_pages == 40
    small = PagedCache.for_model(model, pages=1)
    t = small.new_sequence()
    with pytest.raises(RuntimeError, match="out of pages"):
        PagedRunner(model, small, max_tokens=64).verify({t: ([1] * 17, [-1] + [0] * 16)})
