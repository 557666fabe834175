"""The host side of PagedRunner.verify: the pages that a sequence holds after a
tree of which a part was accepted (the kernels are stand-ins)."""
import pytest

torch = pytest.importorskip("torch")

from harsh4b_b200 import paged  # noqa: E402
from test_paged_cache import cache, consistent, grow  # noqa: E402, F401
from test_paged_cache_limits import cpu_runner  # noqa: E402


def verifying(monkeypatch, cache, accepted, **kwargs):  # noqa: F811
    """A runner whose steps accept the first accepted[b] nodes of sequence b's tree."""
    runner = cpu_runner(monkeypatch, cache, **kwargs)
    step = paged.lib()
    step.h4b_forward_paged_tree = lambda *a: 0
    monkeypatch.setattr(paged, "lib", lambda: step)
    monkeypatch.setattr(paged.ops, "accept_workspace", lambda *a: torch.zeros(16, dtype=torch.uint8))

    def accept(tokens, parents, offsets, logits, *, max_path, workspace):
        path = torch.full((offsets.numel() - 1, max_path), -1, dtype=torch.int32)
        for b, n in enumerate(accepted):
            path[b, :n] = torch.arange(n, dtype=torch.int32)
        return path, torch.tensor(accepted, dtype=torch.int32), None, torch.zeros_like(tokens)

    monkeypatch.setattr(paged.ops, "accept_tree", accept)
    monkeypatch.setattr(paged.ops, "keep_tokens", lambda *a: None)
    return runner


def wide(nodes):
    return [1] * nodes, [-1] + [0] * (nodes - 1)


@pytest.mark.parametrize("before", [0, 5, 15, 16, 31])
@pytest.mark.parametrize("accepted", [1, 2, 33, 50])
def test_rejected_nodes_hold_no_pages(cache, monkeypatch, before, accepted):  # noqa: F811
    runner = verifying(monkeypatch, cache, [accepted])
    a, same = cache.new_sequence(), cache.new_sequence()
    grow(cache, a, before)
    grow(cache, same, before + accepted)
    runner.verify({a: wide(50)})
    assert cache.length(a) == before + accepted
    assert len(cache.table(a)) == len(cache.table(same))  # as if only the accepted tokens had been appended
    consistent(cache)
    # what the others needed is another sequence's to take
    other = cache.new_sequence()
    cache.reserve({other: cache.free_pages * 16})
    assert cache.free_pages == 0


def test_room_of_the_callers_own_stays(cache, monkeypatch):  # noqa: F811
    runner = verifying(monkeypatch, cache, [1, 2])
    a, b = cache.new_sequence(), cache.new_sequence()
    grow(cache, a, 20)
    grow(cache, b, 16)
    cache.reserve({a: 70})  # pages for 90 tokens
    table = cache.table(a)
    runner.verify({a: wide(20), b: wide(40)})
    assert cache.table(a) == table and cache.length(a) == 21
    assert len(cache.table(b)) == 2 and cache.length(b) == 18
    consistent(cache)


def test_under_a_window_and_from_a_shared_page(cache, monkeypatch):  # noqa: F811
    runner = verifying(monkeypatch, cache, [1, 3], window=20, sinks=2)
    a = cache.new_sequence()
    grow(cache, a, 40)
    b = cache.fork(a)
    runner.verify({a: wide(30), b: wide(20)})
    assert cache.length(a) == 41 and cache.length(b) == 43
    assert len(cache.table(a)) == 3 and len(cache.table(b)) == 3
    consistent(cache)


def test_a_step_that_fails_keeps_no_pages(cache, monkeypatch):  # noqa: F811
    runner = verifying(monkeypatch, cache, [1, 1])
    a, b = cache.new_sequence(), cache.new_sequence()
    grow(cache, a, 20)
    grow(cache, b, 3)
    tables, free = [cache.table(a), cache.table(b)], cache.free_pages

    def fails(*args, **kwargs):
        raise RuntimeError("no memory")

    monkeypatch.setattr(paged.ops, "accept_tree", fails)
    with pytest.raises(RuntimeError, match="no memory"):
        runner.verify({a: wide(40), b: wide(20)})
    assert [cache.table(a), cache.table(b)] == tables and cache.free_pages == free
    assert (cache.length(a), cache.length(b)) == (20, 3)
    consistent(cache)
