"""Two streams over one paged cache: a step follows the steps before it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200.model import CudaQwen  # noqa: E402
from harsh4b_b200.paged import PagedCache, PagedRunner  # noqa: E402
from harsh4b_b200.synthetic import synthetic_checkpoint, synthetic_prompt, tiny_config  # noqa: E402


def run(model, switch):
    """Two windowed sessions whose pages go from one to the other as they are
    given back, each step on its own stream if `switch`."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()] if switch else [torch.cuda.current_stream()] * 2
    prompts = [[int(t) for t in synthetic_prompt(model.config, 160, seed=s)] for s in (31, 32)]
    torch.cuda.synchronize()
    results = []
    with torch.cuda.stream(streams[1]):
        cache = PagedCache.for_model(model, pages=12)
        runners = [PagedRunner(model, cache, max_tokens=64, window=40) for _ in range(2)]
    sessions = [cache.new_sequence() for _ in range(2)]
    for start in range(0, 160, 20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                if switch:
                    torch.cuda._sleep(2_000_000)
                logits = runners[i].step({sessions[i]: prompts[i][start:start + 20]})
                results.append(logits[sessions[i]].clone())
    torch.cuda.synchronize()
    runners[0].status()
    return results


def test_pages_pass_between_streams():
    model = CudaQwen.from_checkpoint(synthetic_checkpoint(tiny_config(), seed=7), kv_dtype="float16")
    for a, b in zip(run(model, False), run(model, True)):
        assert torch.equal(a, b)
