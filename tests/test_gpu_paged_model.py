"""The model over a paged cache against its exact single-session path.

Tolerance, derived before the first run: q, k, v and the attended rows carry
16-bit rounding (k and v do on both sides). A fp16 rounding of an attended
value, 2^-11 |v|, moves its int8 code (127 to the row's maximum) with a
probability of about 0.06 |v| / max, so the o projection's input gains an error
of about sqrt(0.02) steps of max / 127, some 0.4 % of its norm, in each layer,
and the logits of two layers at most 1 %; asked for is 2 % (bf16, whose
rounding is 8 times coarser: sqrt(8) times that, 6 %).
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200.model import CudaQwen  # noqa: E402
from harsh4b_b200.paged import PagedCache, PagedRunner  # noqa: E402
from harsh4b_b200.synthetic import synthetic_checkpoint, synthetic_prompt, tiny_config  # noqa: E402


@pytest.fixture(scope="module")
def model():
    return CudaQwen.from_checkpoint(synthetic_checkpoint(tiny_config(), seed=7), kv_dtype="float16")


def exact(model, ids):
    state = model.new_state(len(ids) + 1)
    return model.prefill(ids, state, attention="exact").clone()


def off(got, want):
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype,bound", [("float16", 0.02), ("bfloat16", 0.06)])
@pytest.mark.parametrize("chunk", [300, 64, 7, 1])
def test_chunks_of_a_prompt(model, dtype, bound, chunk):
    ids = synthetic_prompt(model.config, 100 if chunk == 1 else 300, seed=1)
    cache = PagedCache.for_model(model, pages=32, dtype=dtype)
    runner = PagedRunner(model, cache, max_tokens=300)
    sequence = cache.new_sequence()
    for start in range(0, len(ids), chunk):
        logits = runner.step({sequence: ids[start:start + chunk]})[sequence]
    runner.status()
    assert cache.length(sequence) == len(ids)
    assert off(logits, exact(model, ids)) < bound


def test_mixed_steps_and_forks(model):
    """Prompt chunks and decoded tokens in the same steps, forks over a shared prompt."""
    prompt = [int(t) for t in synthetic_prompt(model.config, 150, seed=2)]
    other = [int(t) for t in synthetic_prompt(model.config, 90, seed=3)]
    cache = PagedCache.for_model(model, pages=64)
    runner = PagedRunner(model, cache, max_tokens=256)
    a, b = cache.new_sequence(), cache.new_sequence()
    runner.step({a: prompt[:100], b: other[:1]})
    runner.step({b: other[1:60], a: prompt[100:]})
    used = cache.pages - cache.free_pages
    forks = [cache.fork(a) for _ in range(3)]
    assert cache.pages - cache.free_pages == used  # shared
    logits = runner.step({forks[0]: [11], forks[1]: [22, 33], b: other[60:], forks[2]: [44]})
    runner.status()
    for fork, tail in zip(forks, ([11], [22, 33], [44])):
        assert off(logits[fork], exact(model, prompt + tail)) < 0.02
    assert off(logits[b], exact(model, other)) < 0.02
    cache.free(a)
    cache.free(forks[1])
    assert cache.compact() > 0
    logits = runner.step({forks[2]: [55, 66], forks[0]: [77]})
    assert off(logits[forks[2]], exact(model, prompt + [44, 55, 66])) < 0.02
    assert off(logits[forks[0]], exact(model, prompt + [11, 77])) < 0.02
    runner.status()


def test_window_gives_pages_back(model):
    """A windowed session holds a bounded number of pages, and tokens within the
    window give the unwindowed result."""
    ids = [int(t) for t in synthetic_prompt(model.config, 400, seed=4)]
    cache = PagedCache.for_model(model, pages=16)
    runner = PagedRunner(model, cache, max_tokens=64, window=100, sinks=4)
    sequence = cache.new_sequence()
    for start in range(0, 96, 48):
        logits = runner.step({sequence: ids[start:start + 48]})[sequence]
    assert off(logits, exact(model, ids[:96])) < 0.02
    for start in range(96, 400, 16):
        logits = runner.step({sequence: ids[start:start + 16]})[sequence]
        assert cache.pages - cache.free_pages <= 1 + 100 // 16 + 2
    runner.status()
    assert torch.isfinite(logits).all()


def test_generate_equals_the_steps(model):
    prompts = {0: synthetic_prompt(model.config, 70, seed=5), 1: synthetic_prompt(model.config, 20, seed=6)}
    cache = PagedCache.for_model(model, pages=64)
    assert [cache.new_sequence() for _ in prompts] == [0, 1]
    out = PagedRunner(model, cache, max_tokens=64).generate({s: [int(t) for t in p] for s, p in prompts.items()}, 6, chunk=32)
    for s, prompt in prompts.items():
        ids = [int(t) for t in prompt]
        assert len(out[s]) == 6
        for token in out[s]:  # each greedy token is a maximum within the tolerance
            logits = exact(model, ids)
            assert logits[token] >= logits.max() - 0.04 * logits.norm() / np.sqrt(logits.numel())
            ids.append(token)


def test_refusals(model):
    cache = PagedCache.for_model(model, pages=4)
    runner = PagedRunner(model, cache, max_tokens=32, max_sequences=2)
    s = cache.new_sequence()
    for feed in ({}, {s: []}, {s: list(range(33))}, {s: [-1]}, {s: [model.vocab]}):
        with pytest.raises(ValueError):
            runner.step(feed)
    with pytest.raises(RuntimeError, match="out of pages"):
        for _ in range(3):
            runner.step({s: list(range(32))})
    with pytest.raises(ValueError, match="layers and heads"):
        PagedRunner(model, PagedCache(1, 1, 64, pages=4))
    with pytest.raises(ValueError, match="window"):
        PagedRunner(model, cache, sinks=4)
