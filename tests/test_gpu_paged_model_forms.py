"""The model over a paged cache in its other forms: past a window against the
CPU oracle, as a captured graph, and in another shape than the tiny one.

Where the two sides round differently (q, the attended rows: 16 bits here), an
int8 activation that lies near a rounding boundary gets the neighbouring code.
An error of e steps (e < 1, a step is max / 127) before a quantisation flips a
share 0.8 e of its codes, so it leaves with sqrt(0.8 e) steps: small errors grow
from site to site until 0.8 steps, where they stay. With max = 3.5 rms a step is
2.8 % of a row's norm, so a row's error is at most 2.2 % after any one site,
and the logits, with the residual stream's error and the last quantisation's,
at most sqrt(2) times that and usually half; asked for is 5 % of every row
whatever the number of layers."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import oracle  # noqa: E402
from harsh4b_b200 import _lib, ops  # noqa: E402
from harsh4b_b200.model import CudaQwen  # noqa: E402
from harsh4b_b200.paged import PagedCache, PagedRunner  # noqa: E402
from harsh4b_b200.synthetic import synthetic_checkpoint, synthetic_prompt, tiny_config  # noqa: E402


class WindowedOracle(oracle.OracleQwen):
    """The oracle with a sliding window and first tokens that stay visible."""

    window, sinks = 0, 0

    def attention(self, state, layer_index, q):
        p = state.position
        j = np.arange(p + 1)
        seen = np.flatnonzero((j > p - self.window) | (j < self.sinks))
        k = state.keys[layer_index, seen].astype(np.float64)
        v = state.values[layer_index, seen].astype(np.float64)
        for h in range(self.heads):
            s = k[:, h // self.groups] @ q[h].astype(np.float64) / np.sqrt(self.head_dim)
            w = np.exp(s - s.max())
            state.attended[h * self.head_dim:(h + 1) * self.head_dim] = (w / w.sum()) @ v[:, h // self.groups]


BOUND = 0.05


def off(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


@pytest.fixture(scope="module")
def tiny():
    checkpoint = synthetic_checkpoint(tiny_config(), seed=7)
    layers = [oracle.OracleLayer(*[oracle.OracleProjection(*p) for p in checkpoint.layer(i)[:4]], *checkpoint.layer(i)[4:])
              for i in range(2)]
    windowed = WindowedOracle(checkpoint.config, layers, checkpoint.embedding, checkpoint.embedding_scales,
                              checkpoint.norms["model.norm.weight"], kv_dtype=np.float16)
    return CudaQwen.from_checkpoint(checkpoint, kv_dtype="float16"), windowed


@pytest.mark.parametrize("window,sinks", [(60, 4), (29, 0), (1, 0), (18, 33)])
@pytest.mark.parametrize("chunk", [1, 5, 48])
def test_past_the_window(tiny, window, sinks, chunk):
    """Every row within the bound, and nearest of all to the oracle of this very
    window: one token more or fewer is further off."""
    model, windowed = tiny
    ids = [int(t) for t in synthetic_prompt(model.config, 160, seed=41)]

    def oracle_rows(w, s):
        windowed.window, windowed.sinks = w, s
        state = windowed.new_state(len(ids))
        return np.stack([windowed.forward_token(t, state).copy() for t in ids])

    cache = PagedCache.for_model(model, pages=16)
    runner = PagedRunner(model, cache, max_tokens=64, window=window, sinks=sinks)
    sequence = cache.new_sequence()
    got = {}
    for start in range(0, len(ids), chunk):
        logits = runner.step({sequence: ids[start:start + chunk]})[sequence]
        got[min(start + chunk, len(ids)) - 1] = logits.cpu().numpy().copy()
    runner.status()
    assert -1 in cache.table(sequence)

    want = oracle_rows(window, sinks)
    assert max(off(row, want[p]) for p, row in got.items()) < BOUND
    later = [p for p in got if p >= window + sinks + 1]

    def mean(rows):
        return np.mean([off(got[p], rows[p]) for p in later])

    neighbours = [(w, s) for w, s in ((window + 1, sinks), (window - 1, sinks), (window, sinks + 1), (window, sinks - 1))
                  if w >= 1 and s >= 0]
    assert mean(want) < min(mean(oracle_rows(*other)) for other in neighbours)


def test_another_shape():
    """Four layers, 16 q heads over 4 kv heads, bf16 and fp16 pages of 64 tokens."""
    config = tiny_config(num_hidden_layers=4, hidden_size=1024, intermediate_size=2048, num_attention_heads=16,
                         num_key_value_heads=4, vocab_size=4096, max_position_embeddings=1024)
    model = CudaQwen.from_checkpoint(synthetic_checkpoint(config, seed=9), kv_dtype="float16")
    prompts = [[int(t) for t in synthetic_prompt(config, n, seed=n)] for n in (700, 129, 1)]
    want = []
    for ids in prompts:
        state = model.new_state(len(ids) + 1)
        want.append(model.prefill(ids, state, attention="exact").cpu().numpy().copy())
    for dtype in ("float16", "bfloat16"):
        cache = PagedCache.for_model(model, pages=32, page_size=64, dtype=dtype)
        runner = PagedRunner(model, cache, max_tokens=830)
        sessions = [cache.new_sequence() for _ in prompts]
        logits = runner.step(dict(zip(sessions, prompts)))
        for s, w in zip(sessions, want):
            assert off(logits[s].cpu().numpy(), w) < BOUND
        runner.status()


@pytest.mark.parametrize("rows", [1, 40])
def test_a_captured_step_follows_its_tables(tiny, rows):
    """h4b_forward_paged in a graph: replayed over another batch of that shape
    it gives what the call gives."""
    model, _ = tiny
    cache = PagedCache.for_model(model, pages=80)
    runner = PagedRunner(model, cache, max_tokens=3 * rows)
    prompts = [[int(t) for t in synthetic_prompt(model.config, n, seed=n)] for n in (70, 20, 33)]
    sessions = [cache.new_sequence() for _ in prompts]
    for s, ids in zip(sessions, prompts):
        for start in range(0, len(ids), 3 * rows):
            runner.step({s: ids[start:start + 3 * rows]})
    feeds = [[[int(t) for t in synthetic_prompt(model.config, rows, seed=100 + 10 * turn + i)] for i in range(3)]
             for turn in range(3)]
    forks = [cache.fork(s) for s in sessions]
    want = []
    for feed in feeds:
        logits = runner.step(dict(zip(forks, feed)))
        want.append(torch.stack([logits[s] for s in forks]).clone())

    # the same from fixed tables, the first turn as a plain call, the others replayed
    width = 12
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    offsets = torch.arange(0, 3 * rows + 1, rows, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    layers, pages, kv_heads, page_size, head_dim = cache.k_pages.shape
    kv = _lib.PagedKvDesc(cache.k_pages.data_ptr(), cache.v_pages.data_ptr(), table.data_ptr(), offsets.data_ptr(),
                          lengths.data_ptr(), 1, pages, page_size, kv_heads, head_dim, 3, width, 3 * rows)
    step = _lib.PagedStepDesc(kv, cache.k_pages[0].numel() * 2, 0, 0, rows, *[t.data_ptr() for t in (
        runner.tokens, runner.x, runner.x8, runner.act_scale, runner.act_sum, runner.qkv, runner.q, runner.attended16,
        runner.attended, runner.gate_up, runner.act, runner.last, runner.logits, runner.next_tokens, runner.workspace)],
        runner.workspace.numel())

    def launch():
        _lib.check(_lib.lib().h4b_forward_paged(ctypes.byref(model.desc), ctypes.byref(step), _lib.stream_handle()), "step")

    graph = None
    for feed, expected in zip(feeds, want):
        cache.reserve({s: rows for s in sessions})
        host, _, now = cache.batch_tables(sessions, [rows] * 3)
        table[:, :host.shape[1]] = torch.from_numpy(host).cuda()
        lengths.copy_(torch.from_numpy(now))
        runner.tokens[:3 * rows] = torch.tensor(sum(feed, []), dtype=torch.int32)
        if graph is None:
            launch()
            graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                launch()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(runner.logits[:3], expected)
        assert torch.equal(runner.next_tokens[:3].long(), expected.argmax(-1))
        for s in sessions:
            cache.advance(s, rows)
    assert _lib.device_status() == 0
