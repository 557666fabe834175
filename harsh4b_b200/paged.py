"""A paged K/V cache and the model's steps over it.

``PagedCache`` owns the pages of every layer and the host's side of them: which
pages a sequence holds, how many sequences share a page, which are free.
Sequences may share pages (``fork``: a common prompt is computed and stored
once); a page that is written while shared is copied first (the partly filled
last page of a fork). ``trim`` gives back pages that a sliding window has
passed, ``compact`` moves the live pages to the front. The reference keeps one
contiguous cache per session (cpu_lightspark.py:275-309).

``PagedRunner`` runs ``h4b_forward_paged``: prompt chunks and decoded tokens of
any number of sequences in one step.

    cache = PagedCache.for_model(model, pages=4096)
    runner = PagedRunner(model, cache, max_tokens=2048)
    first = cache.new_sequence()
    logits = runner.step({first: prompt_ids})[first]
    second = cache.fork(first)                      # shares the prompt's pages
    logits = runner.step({first: [a], second: [b]})

``verify`` runs a drafted tree of tokens for each sequence in one step and keeps
the branch that agrees with the model's greedy tokens.
"""
from __future__ import annotations

import ctypes
from contextlib import contextmanager, nullcontext

import numpy as np
import torch

from . import ops
from ._lib import STATUS_BAD_PAGE, TREE_NODES, PagedKvDesc, PagedStepDesc, check, device_status, lib

CACHE_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def on_device(device: torch.device):
    """Makes a CUDA device current (the library launches there)."""
    return torch.cuda.device(device) if device.type == "cuda" else nullcontext()


class PagedCache:
    """Pages [layers][pages][kv_heads][page_size][head_dim] of K and V, and the
    sequences that hold them. Lengths count tokens; `reserve` makes room (and
    private) what the next append writes.

    Pages that are given back may be taken again while kernels that read them
    are still queued, so all work on the pages is in one order: the cache's
    copies and its runners' steps follow those before them, whichever streams
    they are on. Launches of one's own belong into ``with cache.ordered():``
    where several streams use the cache."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 16,
                 dtype: str = "float16", device=None):
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"dtype must be one of {sorted(CACHE_DTYPES)}")
        if min(layers, kv_heads, pages) < 1:
            raise ValueError("layers, kv_heads and pages must be positive")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError("page_size must be a power of two in 16..1024")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=CACHE_DTYPES[dtype], device=device)
        self.v_pages = torch.zeros(shape, dtype=CACHE_DTYPES[dtype], device=device)
        self.page_size, self.pages, self.device = page_size, pages, self.k_pages.device
        self._free = list(range(pages - 1, -1, -1))  # the lowest page is taken next
        self._shared = np.zeros(pages, dtype=np.int32)  # sequences that hold a page
        self._tables: dict[int, list[int]] = {}         # page ids; -1 where trimmed
        self._lengths: dict[int, int] = {}
        self._trimmed: set[int] = set()                 # sequences with a -1 in their table
        self._next = 0
        # the end of the latest work on the pages (none on a CPU) and its stream
        self._event = torch.cuda.Event() if self.device.type == "cuda" else None
        self._stream = None
        with self.ordered():
            pass  # the pages are zeroed here

    @contextmanager
    def ordered(self):
        """Work on the pages that is launched in here, on the current stream,
        runs after all such work before it and before all that follows."""
        with on_device(self.device):
            if self._event is None:
                yield
                return
            stream = torch.cuda.current_stream(self.device)
            if self._stream is not None and stream != self._stream:
                stream.wait_event(self._event)
            try:
                yield
            finally:
                self._event.record(stream)
                self._stream = stream

    @classmethod
    def for_model(cls, model, pages: int, page_size: int = 16, dtype: str = "float16") -> "PagedCache":
        return cls(model.n_layers, model.kv_heads, model.head_dim, pages, page_size, dtype, model.device)

    # -- sequences ---------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._lengths[sequence]

    def table(self, sequence: int) -> list[int]:
        return list(self._tables[sequence])

    def new_sequence(self) -> int:
        sequence, self._next = self._next, self._next + 1
        self._tables[sequence], self._lengths[sequence] = [], 0
        return sequence

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens, sharing every page that holds
        some (room that `sequence` has reserved beyond them stays its own)."""
        length = self._lengths[sequence]
        table = self._tables[sequence][:-(-length // self.page_size)]
        new = self.new_sequence()
        self._tables[new], self._lengths[new] = table, length
        if sequence in self._trimmed:
            self._trimmed.add(new)
        for page in table:
            if page >= 0:
                self._shared[page] += 1
        return new

    def free(self, sequence: int) -> None:
        for page in self._tables.pop(sequence):
            self._drop(page)
        del self._lengths[sequence]
        self._trimmed.discard(sequence)

    def truncate(self, sequence: int, length: int) -> None:
        """Forget the tokens from `length` on. What `trim` gave back does not
        return with an earlier end: see check_visible."""
        if not 0 <= length <= self._lengths[sequence]:
            raise ValueError("length must be within the sequence")
        self._lengths[sequence] = length
        self.release(sequence)

    def release(self, sequence: int, pages: int = 0) -> None:
        """Give back the pages reserved behind the sequence's last token, but
        for the first `pages` that it holds."""
        table = self._tables[sequence]
        held = max(pages, -(-self._lengths[sequence] // self.page_size))
        for page in table[held:]:
            self._drop(page)
        del table[held:]

    def trim(self, sequence: int, window: int, sinks: int = 0) -> int:
        """Give back the pages that no later token sees under (window, sinks);
        returns how many."""
        if window < 1 or sinks < 0:
            raise ValueError("window must be positive and sinks not negative")
        table = self._tables[sequence]
        first = max(0, self._lengths[sequence] + 1 - window)  # that the next token sees
        dropped = 0
        for index in range(-(-sinks // self.page_size), first // self.page_size):
            if table[index] >= 0:
                self._drop(table[index])
                table[index] = -1
                dropped += 1
        if dropped:
            self._trimmed.add(sequence)
        return dropped

    def check_visible(self, sequence: int, window: int = 0, sinks: int = 0) -> None:
        """RuntimeError if the next token would see, under (window, sinks),
        tokens whose pages `trim` gave back (after a truncation, or when the
        window is wider than the one trimmed for): they would read as zeros."""
        length, size = self._lengths[sequence], self.page_size
        if sequence not in self._trimmed or length == 0:
            return
        table, first = self._tables[sequence], max(0, length + 1 - window) if window else 0
        seen = table[first // size:-(-length // size)] if first < length else []
        if -1 in seen or -1 in table[:-(-min(sinks, length) // size)]:
            raise RuntimeError(f"sequence {sequence} sees tokens whose pages were given back")

    def reserve(self, wanted: dict[int, int]) -> None:
        """Room for `wanted[sequence]` more tokens of each sequence; what they
        are written to is the sequence's own afterwards (a shared last page is
        copied on the current stream). All or nothing: RuntimeError when the
        pages do not suffice."""
        size = self.page_size
        plans, need = [], 0
        sharing: dict[int, int] = {}  # last pages that this call itself unshares
        for sequence, count in wanted.items():
            if count < 0:
                raise ValueError("cannot reserve a negative number of tokens")
            if count == 0:
                continue
            table, length = self._tables[sequence], self._lengths[sequence]
            last = table[length // size] if length % size else -1
            copy = last >= 0 and self._shared[last] - sharing.get(last, 0) > 1
            if copy:
                sharing[last] = sharing.get(last, 0) + 1
            elif length % size and last < 0:
                raise RuntimeError("the page to append to was trimmed")
            more = -(-(length + count) // size) - len(table)
            plans.append((sequence, copy, max(0, more)))
            need += copy + max(0, more)
        if need > len(self._free):
            raise RuntimeError(f"out of pages: {need} needed, {len(self._free)} free")
        moves = []
        for sequence, copy, more in plans:
            table = self._tables[sequence]
            if copy:
                index = self._lengths[sequence] // size
                page = self._take()
                moves.append((table[index], page))
                self._drop(table[index])
                table[index] = page
            table.extend(self._take() for _ in range(more))
        self._copy(moves)

    def advance(self, sequence: int, count: int) -> None:
        """`count` tokens were appended to the reserved room."""
        if count < 0:
            raise ValueError("tokens are taken back with truncate")
        length = self._lengths[sequence] + count
        if length > len(self._tables[sequence]) * self.page_size:
            raise ValueError("more tokens than were reserved")
        self._lengths[sequence] = length

    def compact(self) -> int:
        """Move the live pages to the front (a page's sequences follow it);
        returns how many moved."""
        live = np.flatnonzero(self._shared > 0)
        gaps = np.flatnonzero(self._shared[:live.size] == 0)
        movers = live[live >= live.size]
        moves = list(zip(movers.tolist(), gaps.tolist()))  # no page is in both lists
        self._copy(moves)
        to = dict(moves)
        for table in self._tables.values():
            table[:] = [to.get(page, page) for page in table]
        for source, target in moves:
            self._shared[target], self._shared[source] = self._shared[source], 0
        self._free = list(range(self.pages - 1, live.size - 1, -1))
        return len(moves)

    # -- what a step needs --------------------------------------------------
    def batch_tables(self, sequences, new) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """(page table, row offsets, lengths with the new tokens), int32."""
        width = max(1, max((len(self._tables[s]) for s in sequences), default=1))
        table = np.full((len(sequences), width), -1, dtype=np.int32)
        for row, s in enumerate(sequences):
            table[row, :len(self._tables[s])] = self._tables[s]
        lengths = np.array([self._lengths[s] + n for s, n in zip(sequences, new)], dtype=np.int32)
        return table, np.concatenate(([0], np.cumsum(new))).astype(np.int32), lengths

    # -- pages ---------------------------------------------------------------
    def _take(self) -> int:
        page = self._free.pop()
        self._shared[page] = 1
        return page

    def _drop(self, page: int) -> None:
        if page < 0:
            return
        self._shared[page] -= 1
        if self._shared[page] == 0:
            self._free.append(page)

    def _copy(self, moves) -> None:
        if not moves:
            return
        ids = torch.tensor(moves, dtype=torch.int32).T.contiguous().to(self.device)
        with self.ordered():
            ops.copy_pages(self.k_pages, self.v_pages, ids[0], ids[1])


class PagedRunner:
    """The model over a paged cache, with scratch for `max_tokens` rows and
    `max_sequences` sequences a step. window > 0: every layer's attention sees
    the last `window` tokens and the first `sinks`."""

    def __init__(self, model, cache: PagedCache, max_tokens: int = 2048, max_sequences: int = 64, window: int = 0,
                 sinks: int = 0):
        if max_tokens < 1 or max_sequences < 1:
            raise ValueError("max_tokens and max_sequences must be positive")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError("sinks need a window, and neither is negative")
        if max(window, sinks) > 0x7fffffff:
            raise ValueError("window and sinks must fit 32 bits")
        layers, _, kv_heads, _, head_dim = cache.k_pages.shape
        if (layers, kv_heads, head_dim) != (model.n_layers, model.kv_heads, model.head_dim):
            raise ValueError("the cache does not have the model's layers and heads")
        if cache.device != model.embedding.device:
            raise ValueError("the cache is not on the model's device")
        self.model, self.cache, self.max_tokens, self.max_sequences = model, cache, max_tokens, max_sequences
        self.window, self.sinks = window, sinks
        with cache.ordered():  # its first step may be on another stream
            self._allocate()

    def _allocate(self) -> None:
        model, cache = self.model, self.cache
        dev, max_tokens, max_sequences = cache.device, self.max_tokens, self.max_sequences
        H, I, Q, KV = model.hidden, model.intermediate, model.q_size, model.kv_size
        M, B, either = max_tokens, max_sequences, max(max_tokens, max_sequences)
        f32, i32 = dict(dtype=torch.float32, device=dev), dict(dtype=torch.int32, device=dev)
        self.tokens, self.next_tokens = torch.zeros(M, **i32), torch.zeros(B, **i32)
        self.x, self.x8 = torch.zeros(M, H, **f32), torch.zeros(either, max(H, Q, I), dtype=torch.int8, device=dev)
        self.act_scale, self.act_sum = torch.zeros(either, **f32), torch.zeros(either, **i32)
        self.qkv = torch.zeros(M, Q + 2 * KV, **f32)
        self.q = torch.zeros(M, Q, dtype=cache.k_pages.dtype, device=dev)
        self.attended16, self.attended = torch.zeros_like(self.q), torch.zeros(M, Q, **f32)
        self.gate_up, self.act = torch.zeros(M, 2 * I, **f32), torch.zeros(M, I, **f32)
        self.last, self.logits = torch.zeros(B, H, **f32), torch.zeros(B, model.vocab, **f32)
        self.workspace = ops.paged_workspace(model.head_dim, dev)
        self.node_logits = self.accept_workspace = None  # verify's

    def step(self, feed: dict[int, list[int]]) -> dict[int, torch.Tensor]:
        """Append feed[sequence] (token ids, at least one each) to each sequence
        and return the logits after its last one (views, overwritten by the
        next step)."""
        sequences = list(feed)
        ids, new = self._checked([[int(t) for t in feed[s]] for s in sequences])
        cache = self.cache
        if max(cache.length(s) + n for s, n in zip(sequences, new)) > self.model.max_pos:
            raise ValueError(f"a sequence would pass the model's {self.model.max_pos} positions")
        for s in sequences:
            cache.check_visible(s, self.window, self.sinks)
        with cache.ordered():
            cache.reserve(dict(zip(sequences, new)))
            self._launch(sequences, new, ids)
        for s, n in zip(sequences, new):
            cache.advance(s, n)
            if self.window:
                cache.trim(s, self.window, self.sinks)
        return {s: self.logits[b] for b, s in enumerate(sequences)}

    def verify(self, drafts: dict[int, tuple[list[int], list[int]]]) -> dict[int, list[int]]:
        """One step over a drafted tree of tokens for each sequence:
        drafts[sequence] = (token ids, parents), node 0 the token that follows
        the sequence's cached ones (decided before, parent -1), every other
        node a child of an earlier one; at most 256 nodes. Node 0 and the
        branch that agrees with the model's greedy tokens stay in the cache.
        Returns the greedy tokens that follow node 0: the accepted branch's
        and the one after it, of which the last is not in the cache (node 0 of
        the next tree). The nodes' logits are `node_logits` until the next
        call. Pages that only the other nodes needed are given back."""
        sequences = list(drafts)
        ids, new = self._checked([[int(t) for t in drafts[s][0]] for s in sequences])
        trees = [[int(p) for p in drafts[s][1]] for s in sequences]
        cache, model = self.cache, self.model
        for s, tree, n in zip(sequences, trees, new):
            if len(tree) != n or n > TREE_NODES:
                raise ValueError(f"a tree has a parent for each of its nodes, at most {TREE_NODES}")
            if tree[0] != -1 or not all(0 <= p < i for i, p in enumerate(tree) if i):
                raise ValueError("a tree's node 0 is its root, the others have earlier parents")
            if cache.length(s) + n > model.max_pos:
                raise ValueError(f"a sequence would pass the model's {model.max_pos} positions")
            cache.check_visible(s, self.window, self.sinks)
        total = len(ids)
        held = [len(cache.table(s)) for s in sequences]  # room of the caller's own stays
        try:
            with cache.ordered():
                cache.reserve(dict(zip(sequences, new)))
                if self.node_logits is None or self.node_logits.shape[0] < total:
                    self.node_logits = None  # (given back first)
                    self.node_logits = torch.empty(total, model.vocab, dtype=torch.float32, device=cache.device)
                if self.accept_workspace is None:
                    self.accept_workspace = ops.accept_workspace(self.max_tokens, self.max_sequences, cache.device)
                parents = torch.tensor([p for tree in trees for p in tree], dtype=torch.int32).to(cache.device)
                table, offsets, lengths = self._launch(sequences, new, ids, parents)
                path, counts, _, targets = ops.accept_tree(self.tokens[:total], parents, offsets, self.node_logits[:total],
                                                           max_path=max(new), workspace=self.accept_workspace)
                ops.keep_tokens(cache.k_pages, cache.v_pages, table, offsets, lengths, path, counts)
                path, counts, targets = path.tolist(), counts.tolist(), targets.tolist()
            for s, count in zip(sequences, counts):
                cache.advance(s, count)
        finally:  # (a step that fails keeps none of its room)
            for s, pages in zip(sequences, held):
                cache.release(s, pages)
        result, first = {}, 0
        for s, n, nodes, count in zip(sequences, new, path, counts):
            result[s] = [targets[first + node] for node in nodes[:count]]
            first += n
            if self.window:
                cache.trim(s, self.window, self.sinks)
        return result

    def _checked(self, rows: list[list[int]]) -> tuple[np.ndarray, list[int]]:
        """A step's token ids, one sequence after the other, and how many each has."""
        new = [len(r) for r in rows]
        total = sum(new)
        if not rows or min(new) < 1:
            raise ValueError("every sequence of a step needs a token")
        if total > self.max_tokens or len(rows) > self.max_sequences:
            raise ValueError(f"a step holds {self.max_tokens} tokens of {self.max_sequences} sequences")
        ids = np.fromiter((t for r in rows for t in r), dtype=np.int32, count=total)
        if ids.min() < 0 or ids.max() >= self.model.vocab:
            raise ValueError("token ID outside the vocabulary")
        return ids, new

    def _launch(self, sequences, new, ids: np.ndarray, parents: torch.Tensor | None = None):
        cache, model, total = self.cache, self.model, len(ids)
        tables = table, offsets, lengths = tuple(torch.from_numpy(a).to(cache.device)
                                                 for a in cache.batch_tables(sequences, new))
        self.tokens[:total].copy_(torch.from_numpy(ids))
        layers, pages, kv_heads, page_size, head_dim = cache.k_pages.shape
        code = 1 if cache.k_pages.dtype == torch.float16 else 2
        kv = PagedKvDesc(cache.k_pages.data_ptr(), cache.v_pages.data_ptr(), table.data_ptr(), offsets.data_ptr(),
                         lengths.data_ptr(), code, pages, page_size, kv_heads, head_dim, len(sequences), table.shape[1],
                         total)
        step = PagedStepDesc(kv, cache.k_pages[0].numel() * 2, self.window, self.sinks, max(new), *[t.data_ptr() for t in (
            self.tokens, self.x, self.x8, self.act_scale, self.act_sum, self.qkv, self.q, self.attended16, self.attended,
            self.gate_up, self.act, self.last, self.logits if parents is None else self.node_logits, self.next_tokens,
            self.workspace)], self.workspace.numel())
        stream = torch.cuda.current_stream(cache.device).cuda_stream
        if parents is None:
            check(lib().h4b_forward_paged(ctypes.byref(model.desc), ctypes.byref(step), stream), "h4b_forward_paged")
        else:
            check(lib().h4b_forward_paged_tree(ctypes.byref(model.desc), ctypes.byref(step), parents.data_ptr(), stream),
                  "h4b_forward_paged_tree")
        return tables

    def status(self) -> None:
        """Raise if a kernel met a page, offset or length out of range."""
        with on_device(self.cache.device):
            code = device_status()
        if code & STATUS_BAD_PAGE:
            raise RuntimeError("a page id, row offset or length was out of range")
        if code:
            raise RuntimeError(f"device status {code}")

    def generate(self, prompts: dict[int, list[int]], steps: int, chunk: int = 512) -> dict[int, list[int]]:
        """Greedy tokens of every sequence: prompts go in `chunk` tokens at a
        time while the others already decode (each step holds the chunks and
        the decoding sequences' single tokens; sequences that a step has no
        room for wait). Prompts are checked before the first step."""
        pending = {s: [int(t) for t in p] for s, p in prompts.items()}
        if chunk < 1:
            raise ValueError("chunk must be positive")
        for s, rest in pending.items():
            if not rest or min(rest) < 0 or max(rest) >= self.model.vocab:
                raise ValueError("every prompt needs a token, and its IDs must be in the vocabulary")
            if self.cache.length(s) + len(rest) + max(steps, 1) - 1 > self.model.max_pos:
                raise ValueError(f"a sequence would pass the model's {self.model.max_pos} positions")
        out: dict[int, list[int]] = {s: [] for s in prompts}
        while any(len(o) < steps for o in out.values()):
            feed, left = {}, self.max_tokens
            for s, rest in pending.items():
                if len(feed) == self.max_sequences:
                    break
                if len(out[s]) >= steps:
                    continue
                take = 1 if out[s] else min(chunk, len(rest), left)
                if take < 1 or take > left:
                    continue
                feed[s] = [out[s][-1]] if out[s] else rest[:take]
                left -= take
            self.step(feed)
            greedy = self.next_tokens[:len(feed)].tolist()
            for b, s in enumerate(feed):
                if not out[s]:
                    del pending[s][:len(feed[s])]
                    if pending[s]:
                        continue
                out[s].append(greedy[b])
        return out
