"""The host side of the paged cache where its promises could break: forks over
reserved room (the copies are recorded, not run)."""
import pytest

from test_paged_cache import cache, consistent, grow, read  # noqa: F401 (cache is a fixture)

torch = pytest.importorskip("torch")


def write(cache, sequence, value):
    """One token into the reserved room."""
    p = cache.length(sequence)
    cache.k_pages[:, cache.table(sequence)[p // 16], :, p % 16] = value
    cache.advance(sequence, 1)


@pytest.mark.parametrize("length", [0, 5, 16, 20, 32])
def test_fork_leaves_reserved_room_to_its_owner(cache, length):  # noqa: F811
    a = cache.new_sequence()
    cache.reserve({a: length + 40})
    for p in range(length):
        write(cache, a, p)
    own = cache.table(a)
    b = cache.fork(a)
    cache.reserve({a: 1, b: 1})
    consistent(cache)
    assert not set(cache.table(a)[length // 16:]) & set(cache.table(b)[length // 16:])
    write(cache, a, 70)
    write(cache, b, 71)
    assert read(cache, a) == list(range(length)) + [70] and read(cache, b) == list(range(length)) + [71]
    assert len(cache.table(a)) == len(own)  # a's room is still there


@pytest.mark.parametrize("length", [5, 16, 20])
def test_reserved_room_outlives_a_fork(cache, length):  # noqa: F811
    """The owner goes on in its room without reserving anew."""
    a = cache.new_sequence()
    cache.reserve({a: length + 30})
    for p in range(length):
        write(cache, a, p)
    b = cache.fork(a)
    for p in range(length, length + 10):
        write(cache, a, p)
    grow(cache, b, 20)
    for p in range(length + 10, length + 30):
        write(cache, a, p)
    assert read(cache, a) == list(range(length + 30))
    assert read(cache, b) == list(range(length)) + [p + 100 * b for p in range(length, length + 20)]
    consistent(cache)


# ---- what a window has passed ---------------------------------------------------
def seen_pages(length, window, sinks):
    """Pages of the tokens that the next one (at `length`) sees, by the definition."""
    return {j // 16 for j in range(length) if not window or j > length - window or j < sinks}


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 4), (40, 0), (40, 17), (100, 0)])
@pytest.mark.parametrize("trimmed,kept", [(40, 0), (20, 4), (100, 33)])
@pytest.mark.parametrize("forked", [False, True])
def test_tokens_given_back_are_not_seen_again(cache, window, sinks, trimmed, kept, forked):  # noqa: F811
    a = cache.new_sequence()
    grow(cache, a, 160)
    cache.trim(a, trimmed, kept)
    for length in (160, 159, 144, 143, 130, 96, 48, 16, 1, 0):
        cache.truncate(a, length)
        s = cache.fork(a) if forked else a
        missing = [p for p in seen_pages(length, window, sinks) if cache.table(s)[p] < 0]
        if missing:
            with pytest.raises(RuntimeError, match="given back"):
                cache.check_visible(s, window, sinks)
        else:
            cache.check_visible(s, window, sinks)
        if forked:
            cache.free(s)


def cpu_runner(monkeypatch, cache, **kwargs):  # noqa: F811
    """A runner whose model step and workspace are stand-ins."""
    from types import SimpleNamespace

    from harsh4b_b200 import paged

    monkeypatch.setattr(paged.ops, "paged_workspace", lambda *a: torch.zeros(16, dtype=torch.uint8))
    monkeypatch.setattr(paged, "lib", lambda: SimpleNamespace(h4b_forward_paged=lambda *a: 0))
    monkeypatch.setattr(paged.torch.cuda, "current_stream", lambda *a: SimpleNamespace(cuda_stream=0))
    return cpu_runner_over(cache, **kwargs)


def cpu_runner_over(cache, **kwargs):  # noqa: F811
    from types import SimpleNamespace

    from harsh4b_b200 import paged

    model = SimpleNamespace(n_layers=2, kv_heads=2, head_dim=64, hidden=8, intermediate=8, q_size=128, kv_size=128,
                            vocab=50, max_pos=4096, desc=paged.PagedStepDesc(), embedding=cache.k_pages)
    return paged.PagedRunner(model, cache, max_tokens=64, **kwargs)


def test_a_step_behind_its_window_is_refused(cache, monkeypatch):  # noqa: F811
    runner = cpu_runner(monkeypatch, cache, window=40)
    a = cache.new_sequence()
    for _ in range(10):
        runner.step({a: [1] * 16})  # gives back what the window passes
    runner.step({a: [1]})
    cache.truncate(a, 152)  # the next token sees 113 and later, which are there
    before = cache.table(a), cache.free_pages
    cache.truncate(a, 144)  # and here 105 and later: page 6 is gone
    before = cache.table(a), cache.free_pages
    with pytest.raises(RuntimeError, match="given back"):
        runner.step({a: [1]})
    assert (cache.table(a), cache.free_pages) == before and cache.length(a) == 144
    cache.truncate(a, 0)
    runner.step({a: [1] * 20})
    assert cache.length(a) == 20


def test_an_unwindowed_step_over_a_trimmed_sequence_is_refused(cache, monkeypatch):  # noqa: F811
    a = cache.new_sequence()
    grow(cache, a, 60)
    cache.trim(a, 20)
    with pytest.raises(RuntimeError, match="given back"):
        cpu_runner(monkeypatch, cache).step({a: [1]})


# ---- generate -------------------------------------------------------------------
def generating(monkeypatch, cache, **kwargs):  # noqa: F811
    """A runner whose greedy token is the number of rows fed so far, and its record of steps."""
    runner = cpu_runner(monkeypatch, cache, **kwargs)
    plain, runner.feeds = runner.step, []

    def step(feed):
        logits = plain(feed)
        runner.feeds.append({s: list(t) for s, t in feed.items()})
        runner.next_tokens[:len(feed)] = torch.tensor([cache.length(s) % 50 for s in feed], dtype=torch.int32)
        return logits

    runner.step = step
    return runner


def test_generate_refuses_before_its_first_step(cache, monkeypatch):  # noqa: F811
    runner = generating(monkeypatch, cache)
    a, b = cache.new_sequence(), cache.new_sequence()
    for prompts, chunk in (({a: [1, 2], b: []}, 512), ({a: [1]}, 0), ({a: [1]}, -3)):
        with pytest.raises(ValueError):
            runner.generate(prompts, 3, chunk=chunk)
    with pytest.raises(KeyError):
        runner.generate({a: [1], 77: [2]}, 3)
    assert runner.feeds == [] and cache.length(a) == cache.length(b) == 0
    assert runner.generate({a: [1], b: [2]}, 0) == {a: [], b: []} and runner.generate({}, 4) == {}


@pytest.mark.parametrize("most", [1, 2, 3, 5])
@pytest.mark.parametrize("chunk", [1, 3, 512])
def test_generate_more_prompts_than_a_step_holds(cache, monkeypatch, most, chunk):  # noqa: F811
    runner = generating(monkeypatch, cache, max_sequences=most)
    prompts = {cache.new_sequence(): [7] * n for n in (5, 1, 20, 3, 9)}
    out = runner.generate(prompts, 4, chunk=chunk)
    for s, prompt in prompts.items():
        assert out[s] == [len(prompt) + i for i in range(4)]
        fed = [t for feed in runner.feeds for t in feed.get(s, [])]
        assert fed == prompt + out[s][:3] and cache.length(s) == len(fed)
    assert max(len(feed) for feed in runner.feeds) == most


def test_generate_checks_ids_and_positions_first(cache, monkeypatch):  # noqa: F811
    runner = generating(monkeypatch, cache)
    runner.model.max_pos = 30
    a, b = cache.new_sequence(), cache.new_sequence()
    for prompt, steps in (([-1], 2), ([50], 2), ([1] * 31, 1), ([1] * 28, 4)):
        with pytest.raises(ValueError):
            runner.generate({a: [1], b: prompt}, steps, chunk=8)
    assert runner.feeds == []
    assert len(runner.generate({b: [1] * 28}, 3, chunk=8)[b]) == 3


# ---- devices --------------------------------------------------------------------
def test_every_tensor_must_be_on_the_current_device(monkeypatch):
    from harsh4b_b200 import ops

    class On(torch.Tensor):  # a CPU tensor that says it lies on CUDA device 1
        is_cuda, device = True, "cuda:1"

        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 100 + index)
    assert ops._here(1) == 101
    with pytest.raises(ValueError, match="current device, cuda:1, not cuda:0"):
        ops._here(0)
    tensor = torch.zeros(4, 4).as_subclass(On)
    for pointer in (ops._on, ops._rows):
        assert pointer(tensor, torch.float32, "x", 1) == tensor.data_ptr()
        for device in (0, 2):
            with pytest.raises(ValueError, match="x must be on the device of the other tensors"):
                pointer(tensor, torch.float32, "x", device)
        with pytest.raises(ValueError, match="x must be a CUDA tensor"):
            pointer(torch.zeros(4, 4), torch.float32, "x", -1)


def test_steps_and_copies_make_the_caches_device_current(cache, monkeypatch):  # noqa: F811
    from contextlib import contextmanager
    from types import SimpleNamespace

    from harsh4b_b200 import paged

    current, seen = [], []

    @contextmanager
    def device(index):
        current.append(index)
        yield
        current.pop()

    runner = cpu_runner(monkeypatch, cache)
    monkeypatch.setattr(paged, "on_device", device)
    monkeypatch.setattr(paged, "lib", lambda: SimpleNamespace(h4b_forward_paged=lambda *a: seen.append(list(current)) or 0))
    copy = paged.ops.copy_pages
    monkeypatch.setattr(paged.ops, "copy_pages", lambda *a: (seen.append(list(current)), copy(*a)))
    a = cache.new_sequence()
    runner.step({a: [1] * 20})
    runner.step({cache.fork(a): [2]})  # a copy and a step
    assert [devices[-1:] for devices in seen] == [[cache.device]] * 3


def test_a_cache_on_another_device_is_refused(cache, monkeypatch):  # noqa: F811
    from types import SimpleNamespace

    runner = cpu_runner(monkeypatch, cache)
    runner.model.embedding = SimpleNamespace(device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="model's device"):
        type(runner)(runner.model, cache)


# ---- streams --------------------------------------------------------------------
class Streams:
    """Stand-ins for CUDA streams and the cache's event: what waits for what."""

    def __init__(self, monkeypatch, cache):  # noqa: F811
        from types import SimpleNamespace

        from harsh4b_b200 import paged

        self.log, self.now = [], None
        self.made = {name: SimpleNamespace(name=name, cuda_stream=0, wait_event=lambda e, name=name: self.log.append(f"{name} waits"))
                     for name in "AB"}
        cache._event = SimpleNamespace(record=lambda stream: self.log.append(f"{stream.name} records"))
        monkeypatch.setattr(paged.torch.cuda, "current_stream", lambda *a: self.made[self.now])

    def on(self, name):
        self.now = name
        self.log.clear()


def test_work_on_another_stream_waits(cache, monkeypatch):  # noqa: F811
    runner, other = cpu_runner(monkeypatch, cache, window=20), cpu_runner(monkeypatch, cache)
    streams = Streams(monkeypatch, cache)
    a, b = cache.new_sequence(), cache.new_sequence()
    streams.on("A")
    runner.step({a: [1] * 60})  # gives pages back while its kernels may still read them
    assert streams.log[-1] == "A records"
    streams.on("A")
    runner.step({a: [1]})
    assert "A waits" not in streams.log and streams.log[-1] == "A records"
    streams.on("B")
    other.step({b: [1] * 40})
    assert streams.log[0] == "B waits" and streams.log[-1] == "B records"
    cache.free(a)
    streams.on("A")
    assert cache.compact() > 0
    assert streams.log == ["A waits", "A records"]
    streams.on("B")
    cache.reserve({cache.fork(b): 1})  # the copy of a shared page
    assert streams.log == ["B waits", "B records"]


def test_a_runner_follows_its_caches_streams(cache, monkeypatch):  # noqa: F811
    """Its scratch is zeroed on the stream that makes it."""
    cpu_runner(monkeypatch, cache)
    streams = Streams(monkeypatch, cache)
    streams.on("A")
    runner = cpu_runner_over(cache)
    assert streams.log[-1] == "A records"
    streams.on("B")
    runner.step({cache.new_sequence(): [1]})
    assert streams.log[0] == "B waits"


@pytest.mark.parametrize("options", [{"window": (1 << 32) + 8}, {"window": 8, "sinks": 1 << 31}])
def test_windows_past_32_bits_are_refused(cache, monkeypatch, options):  # noqa: F811
    with pytest.raises(ValueError, match="32 bits"):
        cpu_runner(monkeypatch, cache, **options)


def test_advance_goes_forward_only(cache):  # noqa: F811
    a = cache.new_sequence()
    grow(cache, a, 20)
    with pytest.raises(ValueError):
        cache.advance(a, -1)
    assert cache.length(a) == 20
    cache.advance(a, 0)
