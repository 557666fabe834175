"""Drafted token trees over the paged cache: attention and append, against
their definitions in 64 bits.

Attention tolerance: as derived in test_gpu_paged.py (the same roundings: p and
the result once each to the cache's type, fp32 for the rest):
1.1 (u (A + |o|) + 2^-13 A) + n 2^-26 max|v| with A = softmax(S) |V|, and 2e-4
for the log-sum-exp.
"""
import math
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib, ops  # noqa: E402
from test_gpu_paged import SHAPES, UNIT, Batch  # noqa: E402


def draft(n, spread, roots=1, seed=0):
    """Parents of a tree of n nodes: each among the `spread` nodes before it."""
    rng = random.Random(seed)
    roots = min(roots, n)
    return [-1] * roots + [rng.randrange(max(0, i - spread), i) for i in range(roots, n)]


def depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


class Trees(Batch):
    """A Batch whose new tokens are trees' nodes."""

    def __init__(self, parents, total, **kwargs):
        super().__init__([len(p) for p in parents], total, **kwargs)
        self.trees = parents
        self.parents = torch.tensor([p for tree in parents for p in tree], dtype=torch.int32, device="cuda").reshape(-1)

    def call(self, q=None, **kwargs):
        kwargs.setdefault("lse", torch.full((self.rows, self.heads), 7.0, device="cuda"))
        kwargs.setdefault("max_query", max(max(self.new, default=1), 1))
        out = ops.paged_tree_attention(self.q if q is None else q, self.k_pages, self.v_pages, self.table, self.offsets,
                                       self.lens, self.parents, window=self.window, sinks=self.sinks, **kwargs)
        return out, kwargs["lse"]

    def seen(self, b):
        """[nodes][length]: what a node of sequence b sees."""
        tree, n, total = self.trees[b], self.new[b], self.total[b]
        context, depth = total - n, depths(self.trees[b])
        stands = list(range(context)) + [context + d for d in depth]
        rows = []
        for i in range(n):
            mine, j = set(), i
            while j >= 0:
                mine.add(context + j)
                j = tree[j]
            at = context + depth[i]
            rows.append([(j < context or j in mine) and
                         (not self.window or at - stands[j] < self.window or stands[j] < self.sinks) for j in range(total)])
        return torch.tensor(rows, device="cuda").reshape(n, total)

    def expected(self):
        group = self.heads // self.kv_heads
        out = torch.zeros(self.rows, self.heads, self.dim, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        lse = torch.full((self.rows, self.heads), -math.inf, dtype=torch.float64, device="cuda")
        u, at = UNIT[self.dtype], 0
        for b, (n, total) in enumerate(zip(self.new, self.total)):
            if n == 0:
                continue
            seen = self.seen(b)
            for h in range(self.heads):
                k, v = self.k[b][:, h // group].double(), self.v[b][:, h // group].double()
                s = (self.q[at:at + n, h].double() @ k.T / math.sqrt(self.dim)).masked_fill(~seen, -math.inf)
                lse[at:at + n, h] = torch.logsumexp(s, -1)
                w = torch.softmax(s, -1)
                o, a = w @ v, w @ v.abs()
                out[at:at + n, h] = o
                bound[at:at + n, h] = 1.1 * (u * (a + o.abs()) + 2.0 ** -13 * a) + total * 2.0 ** -26 * v.abs().max()
            at += n
        return out, lse, bound

    def set_key(self, b, j, k=None, v=None):
        """Other values at place j of sequence b (every kv head)."""
        held = int(self.table[b, j // self.page])
        for value, mine, pages in ((k, self.k, self.k_pages), (v, self.v, self.v_pages)):
            if value is not None:
                mine[b][j] = value
                pages[held, :, j % self.page] = value


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
@pytest.mark.parametrize("spread", [1, 4, 300])
def test_sizes_and_shapes(heads, kv_heads, dim, page, dtype, spread):
    sizes = [1, 2, 3, 0, 5, 16, 17, 33, 64, 1]
    context = [0, 1, 127, 40, 300, 112, 250, 95, 700, 2049]
    parents = [draft(n, spread, seed=i) for i, n in enumerate(sizes)]
    Trees(parents, [c + n for c, n in zip(context, sizes)], heads=heads, kv_heads=kv_heads, dim=dim, page=page,
          dtype=dtype).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
def test_large_trees(heads, kv_heads, dim, page, dtype):
    parents = [draft(256, 8, roots=3), draft(200, 256, seed=1), draft(129, 1, seed=2)]
    Trees(parents, [256, 517, 700], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seed=1).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 0), (16, 4), (100, 17), (128, 130), (5000, 3)])
def test_window_and_sinks(heads, kv_heads, dim, page, dtype, window, sinks):
    parents = [draft(7, 3, roots=2), draft(1, 1), draft(40, 1), draft(60, 20, seed=1), draft(3, 3)]
    Trees(parents, [700, 1, 400, 517, 129], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, window=window,
          sinks=sinks, seed=2).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES[:4])
@pytest.mark.parametrize("longest,sequences", [(384, 1), (384, 9), (900, 9), (900, 160)])
def test_short_tables_and_long_ones_give_the_same(heads, kv_heads, dim, page, dtype, longest, sequences):
    """Tables that bound the lengths keep items whole, wider ones do not: the keys' sums differ in their order only."""
    rng = random.Random(sequences)
    parents = [draft(rng.randint(0, 40 if sequences < 100 else 6), 3, seed=i) for i in range(sequences)]
    total = [max(len(p), rng.randint(0, longest - 64)) for p in parents]
    trees = Trees(parents, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seed=9)
    width = -(-max(max(total), 1) // page)  # pages that the longest needs
    wide = torch.full((sequences, trees.table.shape[1] + 4096 // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :trees.table.shape[1]] = trees.table
    trees.table = wide[:, :width].contiguous()
    trees.check()
    trees.table = wide
    trees.check()


@pytest.mark.parametrize("page", [16, 512, 1024])
@pytest.mark.parametrize("n", [3, 20, 33])
def test_page_sizes(n, page):
    """Pages that end inside a tile, and tiles inside a page (one and two tiles of rows)."""
    for dim in (64, 128):
        Trees([draft(n, 4), draft(n, 2, seed=1)], [1500 + n, 1020 + n], heads=16, kv_heads=2, dim=dim, page=page,
              dtype=torch.bfloat16, seed=7).check()


@pytest.mark.parametrize("hint", [1, 2, 4, 20, 256, 100000])
def test_the_expected_size_changes_no_answer(hint):
    parents = [draft(n, 4, seed=n) for n in (1, 9, 70, 0, 256)]
    for heads, kv_heads, dim in ((8, 2, 128), (6, 2, 64)):
        Trees(parents, [260, 9, 513, 12, 300], heads=heads, kv_heads=kv_heads, dim=dim, page=32, dtype=torch.float16,
              seed=3).check(max_query=hint)


def test_a_chain_is_a_chunk():
    """A tree without branches is paged_attention's chunk of new tokens."""
    trees = Trees([draft(40, 1), draft(9, 1)], [400, 90], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    out, lse = trees.call()
    chunk, chunk_lse = Batch.call(trees)
    _, _, bound = trees.expected()
    assert ((out.double() - chunk.double()).abs() <= 2 * bound).all()
    assert (lse - chunk_lse).abs().max() <= 4e-4


def test_many_sequences():
    """More sequences than threads, and one long one among them."""
    parents = [draft(1 + i % 5, 2, seed=i) for i in range(500)]
    total = [len(p) + (37 * i) % 90 for i, p in enumerate(parents)]
    total[311] = 9000
    Trees(parents, total, heads=4, kv_heads=1, dim=128, page=16, dtype=torch.float16, seed=4).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_small_trees_among_large_ones(dim):
    """Most trees fill a part of one tile of rows, some two tiles, and their keys a block or two: what the warps of a
    tile without rows pass by at once, the others still read."""
    sizes = [1 + (7 * i) % 12 if i % 9 else 30 for i in range(260)]
    parents = [draft(n, 1 + i % 5, seed=i) for i, n in enumerate(sizes)]
    total = [n + (11 * i) % 70 for i, n in enumerate(sizes)]
    trees = Trees(parents, total, heads=8, kv_heads=1, dim=dim, page=16, dtype=torch.float16, seed=8)
    first = [t.clone() for t in trees.call()]
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(trees.call(), first))
    trees.check()
    Trees(parents, total, heads=8, kv_heads=1, dim=dim, page=16, dtype=torch.float16, seed=8, window=9, sinks=1).check()


@pytest.mark.parametrize("n,total", [(1, 33000), (5, 20011), (64, 12345), (32, 16384 + 128)])
def test_long_contexts_are_split(n, total):
    Trees([draft(n, 4)], [total], heads=8, kv_heads=2, dim=128, page=64, dtype=torch.bfloat16, seed=5).check()


@pytest.mark.parametrize("n", [4, 40])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_who_sees_them(n, what, value):
    """In a drafted node (some nodes see it) and at the window's edge."""
    for dim in (64, 128):
        for window in (0, 100):
            trees = Trees([draft(n, 3, roots=2), draft(n, 3, seed=1)], [300, 211], heads=8, kv_heads=2, dim=dim, page=16,
                          dtype=torch.float16, window=window, sinks=2 if window else 0)
            clean, clean_lse = trees.call()
            hit = []
            for b, j in ((0, 300 - n + 2), (1, 211 - n), (1, 211 - n - 99)):
                hit.append((b, j, trees.seen(b)[:, j]))
                if what == "k":  # the sign of the products is each row's own: inf or -inf
                    trees.set_key(b, j, k=value)
                else:
                    trees.set_key(b, j, v=value)
            out, lse = trees.call()
            assert _lib.device_status() == 0
            touched = torch.zeros(trees.rows, dtype=torch.bool, device="cuda")
            for b, j, rows in hit:
                touched[b * n:(b + 1) * n] |= rows
            assert touched.any()
            assert torch.equal(out[~touched], clean[~touched]) and torch.equal(lse[~touched], clean_lse[~touched])
            if what == "v":
                assert not torch.isfinite(out[touched]).any()
                assert torch.equal(lse[touched], clean_lse[touched])
            elif value != value:
                assert torch.isnan(out[touched]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [20, 40, 150])
@pytest.mark.parametrize("total", [300, 380, 700])
def test_a_value_that_is_not_finite_in_any_block(n, dim, total):
    """Each of a tree's blocks in turn, with tables that keep items whole and others that cut them: a key that
    some rows see, at the windows' first places and among the nodes."""
    for window in (0, 200):
        trees = Trees([draft(n, 4, roots=3)], [total], heads=8, kv_heads=2, dim=dim, page=16, dtype=torch.float16,
                      window=window)
        clean, _ = trees.call()
        context = total - n
        places = list(range(context, total, 13)) + (list(range(max(0, context - window + 1), context - window + 30, 5)) if window else [])
        wide = torch.full((1, trees.table.shape[1] + 256), -1, dtype=torch.int32, device="cuda")
        wide[:, :trees.table.shape[1]] = trees.table
        narrow, values = trees.table, trees.v_pages.clone()
        for j in places:
            rows = trees.seen(0)[:, j]
            trees.set_key(0, j, v=float("inf"))
            for table in (narrow, wide):
                trees.table = table
                out, _ = trees.call()
                assert not torch.isfinite(out[rows]).any(), (window, j)
                if table is narrow:
                    assert torch.equal(out[~rows], clean[~rows])
                else:
                    assert torch.isfinite(out[~rows]).all()
            trees.table = narrow
            trees.v_pages.copy_(values)


def test_scores_of_any_finite_size():
    """Rising and huge scores: the running maximum moves, the weights stay finite."""
    for factor in (8.0, 3000.0):
        trees = Trees([draft(5, 2), draft(40, 3)], [900, 700], heads=4, kv_heads=1, dim=128, page=16, dtype=torch.bfloat16)
        ramp = torch.linspace(0.1, 4.0, 900, device="cuda")
        trees.q = (trees.q.float() * factor).to(torch.bfloat16)
        direction = trees.q[-1, 0].float() / trees.q[-1, 0].float().norm()
        for b in range(2):
            for j in range(trees.total[b]):
                trees.set_key(b, j, k=(trees.k[b][j].float() + factor * ramp[j] * direction).to(torch.bfloat16))
        out, lse = trees.call()
        want, want_lse, bound = trees.expected()
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        if factor < 10:
            trees.check()
        else:
            # The scores carry the rounding of fp32 sums, |error| <= D 2^-24 scale sum|q k|, which is many units here: the
            # weights of keys so near the maximum may be any. The log-sum-exp is off by no more than the scores.
            at = 0
            for b, (n, total) in enumerate(zip(trees.new, trees.total)):
                size = torch.einsum("ihd,jd->ihj", trees.q[at:at + n].double().abs(), trees.k[b][:, 0].double().abs()) / math.sqrt(128)
                bound = 128 * 2.0 ** -24 * size.amax(-1) + 2e-4
                assert ((lse.double() - want_lse)[at:at + n].abs() <= bound).all()
                at += n


def test_equal_keys_give_the_mean():
    """A huge score, the same for all keys: the weights are equal, whatever its size."""
    for n in (3, 40):
        trees = Trees([draft(n, 2)], [300], heads=4, kv_heads=1, dim=64, page=16, dtype=torch.float16)
        trees.q.fill_(60.0)
        for j in range(300):
            trees.set_key(0, j, k=500.0)
        out, lse = trees.call()
        want, want_lse, bound = trees.expected()
        assert ((out.double() - want).abs() <= bound).all()
        # a score is 60 * 500 * 64 / 8 = 240000, whose fp32 neighbours lie 2^-6 apart: the fp32 log-sum-exp cannot
        # be nearer than 2^-7; score, scale, base and sum are rounded once each, 4 x 2^-24 of it in all
        assert ((lse.double() - want_lse).abs() <= 4 * 2.0 ** -24 * want_lse.abs() + 2e-4).all()


def test_rows_of_no_sequence_and_bad_tables():
    good = Trees([draft(6, 3), draft(50, 5)], [200, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    want, want_lse = [t.clone() for t in good.call()]
    # rows behind the last sequence are left as they were
    q = torch.cat((good.q, torch.full_like(good.q[:3], float("nan"))))
    parents = torch.cat((good.parents, good.parents.new_tensor([7, -5, 1 << 30])))
    out, lse = torch.full_like(q, 3.0), torch.full((q.shape[0], 8), 5.0, device="cuda")
    ops.paged_tree_attention(q, good.k_pages, good.v_pages, good.table, good.offsets, good.lens, parents, max_query=50,
                             out=out, lse=lse)
    assert torch.equal(out[:56], want) and torch.equal(lse[:56], want_lse)
    assert (out[56:] == 3).all() and (lse[56:] == 5).all() and _lib.device_status() == 0

    def broken(change, whose, answered=True):
        trees = Trees(good.trees, good.total, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
        change(trees)
        out, lse = trees.call(max_query=50)
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        other = slice(6, None) if whose == 0 else slice(0, 6)
        mine = slice(0, 6) if whose == 0 else slice(6, None)
        assert torch.equal(out[other], want[other]) and torch.equal(lse[other], want_lse[other])
        if answered:
            assert (out[mine] == 0).all() and (lse[mine] == -math.inf).all()

    broken(lambda t: t.lens[0].fill_(5), 0)             # fewer tokens than nodes
    broken(lambda t: t.lens[1].fill_(1 << 28), 1)       # past its table
    broken(lambda t: t.table[0, 3].fill_(1 << 20), 0, answered=False)
    for bad in (3, 40, -2, -(1 << 31), (1 << 31) - 1):   # node 3's parent: a root's
        trees = Trees(good.trees, good.total, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
        trees.parents[3] = bad
        out, lse = trees.call(max_query=50)
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        trees.trees = [trees.trees[0][:3] + [-1] + trees.trees[0][4:], trees.trees[1]]
        trees.parents[3] = -1
        same, same_lse = trees.call(max_query=50)
        assert torch.equal(out, same) and torch.equal(lse, same_lse)
        trees.check()


def test_a_tree_past_256_nodes_counts_as_empty():
    trees = Trees([draft(257, 4), draft(5, 2)], [400, 60], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    out, lse = trees.call(max_query=300)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert (out[:257] == 0).all() and (lse[:257] == -math.inf).all()
    want, _, bound = trees.expected()
    assert ((out.double() - want).abs() <= bound)[257:].all()


def test_strided_queries_and_outputs():
    trees = Trees([draft(3, 2), draft(40, 4)], [77, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16)
    wide = torch.randn(trees.rows, 12 * 128, device="cuda").to(torch.bfloat16)
    wide[:, :1024] = trees.q.reshape(trees.rows, 1024)
    out = torch.zeros(trees.rows, 2, 8, 128, dtype=torch.bfloat16, device="cuda")
    plain, _ = trees.call()
    strided, _ = trees.call(q=wide[:, :1024].unflatten(1, (8, 128)), out=out[:, 1])
    assert torch.equal(strided, plain) and torch.equal(out[:, 1], plain) and (out[:, 0] == 0).all()


@pytest.mark.parametrize("n", [3, 40])
def test_same_bits_every_time_and_workspace_left_ready(n):
    trees = Trees([draft(n, 4), draft(n, 2), draft(1, 1)], [5000, 9001, 4000], heads=8, kv_heads=2, dim=128, page=16,
                  dtype=torch.float16)
    workspace = ops.paged_workspace()
    first = [t.clone() for t in trees.call(workspace=workspace)]
    for _ in range(5):
        again = trees.call(workspace=workspace)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    Batch([1, 60], [700, 900], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16).check(workspace=workspace)


@pytest.mark.parametrize("n", [3, 40])
def test_captured_graph_follows_the_tables(n):
    args = dict(heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    trees, other = Trees([draft(n, 4), draft(n, 1)], [400, 3000], **args), Trees([draft(n, 9, 2), draft(n, 2)], [90, 333], seed=9, **args)
    workspace = ops.paged_workspace()
    out, lse = trees.call(workspace=workspace)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        trees.call(workspace=workspace, out=out, lse=lse)
    trees.lens.copy_(other.lens)
    trees.q.copy_(other.q)
    trees.parents.copy_(other.parents)
    trees.table.fill_(-1)
    for b in range(2):  # the other batch's tokens in the pages that this one owns
        need = -(-other.total[b] // 16)
        held = torch.arange(b * 30, b * 30 + need, device="cuda", dtype=torch.int32)
        trees.table[b, :need] = held
        trees.k_pages[held.long()] = other.k_pages[other.table[b, :need].long()]
        trees.v_pages[held.long()] = other.v_pages[other.table[b, :need].long()]
    graph.replay()
    torch.cuda.synchronize()
    want, _, bound = other.expected()
    assert ((out.double() - want).abs() <= bound).all()


def test_runs_on_the_current_stream():
    trees = Trees([draft(3, 2), draft(30, 4)], [500, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    want, _ = trees.call()
    q = trees.q.clone()
    trees.q.zero_()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        trees.q.copy_(q)
        got, _ = trees.call()
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [2, 30])
def test_offsets_past_32_bits(n):
    """Pages whose values lie past 2^31 elements into the buffers."""
    pages = (1 << 31) // (8 * 64 * 128) + 40
    trees = Trees([draft(n, 3)], [2000], heads=32, kv_heads=8, dim=128, page=64, dtype=torch.float16)
    k_pages = torch.empty(pages, 8, 64, 128, dtype=torch.float16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    held, used = trees.table[0, :32].long(), pages - 32 + torch.arange(32, device="cuda")
    k_pages[used], v_pages[used] = trees.k_pages[held], trees.v_pages[held]
    trees.table[0, :32] = used.to(torch.int32)
    trees.k_pages, trees.v_pages = k_pages, v_pages
    trees.check()


def test_refusals():
    trees = Trees([draft(2, 1)], [40], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    args = (trees.k_pages, trees.v_pages, trees.table, trees.offsets, trees.lens)
    with pytest.raises(ValueError, match="parents must hold one index a token"):
        ops.paged_tree_attention(trees.q, *args, trees.parents[:1])
    with pytest.raises(ValueError, match="parents must be torch.int32"):
        ops.paged_tree_attention(trees.q, *args, trees.parents.long())
    with pytest.raises(ValueError, match="parents must be a CUDA tensor"):
        ops.paged_tree_attention(trees.q, *args, trees.parents.cpu())
    with pytest.raises(ValueError, match="parents must be a CUDA tensor"):
        ops.paged_tree_attention(trees.q, *args, None if False else [0, 1])
    with pytest.raises(ValueError, match="q must be torch.float16"):
        ops.paged_tree_attention(trees.q.float(), *args, trees.parents)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_tree_attention(trees.q, *args, trees.parents, sinks=4)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_tree_attention(trees.q, *args, trees.parents, scale=0.0)
    qkv = torch.zeros(2, 12 * 128, device="cuda")
    with pytest.raises(ValueError, match="parents must hold one index a token"):
        ops.paged_append(qkv, *args, heads=8, parents=trees.parents[:1])
    assert _lib.device_status() == 0


def test_batches_without_nodes():
    for new in ([], [0, 0]):
        trees = Trees([[] for _ in new], [9] * len(new), heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
        out, _ = trees.call()
        assert out.shape == (0, 8, 128)
        q = ops.paged_append(torch.zeros(0, 12 * 128, device="cuda"), trees.k_pages, trees.v_pages, trees.table,
                             trees.offsets, trees.lens, heads=8, parents=trees.parents)
        assert q.shape == (0, 8, 128)
    assert _lib.device_status() == 0


# ---- append -----------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
@pytest.mark.parametrize("source", ["fp32", "16"])
def test_append(heads, kv_heads, dim, page, dtype, source):
    """Every node's row is what the plain append writes for a token at its
    position, bit for bit, and lies at its place; untouched slots keep their bits."""
    parents = [draft(1, 1), [], draft(50, 6, roots=3), draft(256, 2), draft(3, 1)]
    trees = Trees(parents, [9, 4, 130, 260, 64], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, stale=5.0)
    g = torch.Generator("cuda").manual_seed(3)
    width = (heads + 2 * kv_heads) * dim
    wide = torch.empty(trees.rows, width + 64, device="cuda").normal_(generator=g) * 3
    qkv = (wide if source == "fp32" else wide.to(dtype))[:, :width]
    norms = dict(zip(("norm_q", "norm_k"), (1 + 0.1 * torch.empty(dim, device="cuda").normal_(generator=g) for _ in range(2))))
    angles = torch.rand(300, dim // 2, generator=g, device="cuda") * 6
    extra = dict(heads=heads, eps=1e-5, rope_cos=angles.cos(), rope_sin=angles.sin(), **norms)
    before = trees.k_pages.clone(), trees.v_pages.clone()
    q = ops.paged_append(qkv, trees.k_pages, trees.v_pages, trees.table, trees.offsets, trees.lens, parents=trees.parents,
                         **extra)
    # each node alone, as a sequence of its own that ends at its position
    at = torch.tensor([t - len(p) + d for p, t in zip(parents, trees.total) for d in depths(p)], device="cuda")
    alone_k = torch.zeros(trees.rows * (300 // page + 1), kv_heads, page, dim, dtype=dtype, device="cuda")
    alone_v = torch.zeros_like(alone_k)
    table = torch.arange(alone_k.shape[0], dtype=torch.int32, device="cuda").view(trees.rows, -1)
    want_q = ops.paged_append(qkv, alone_k, alone_v, table, torch.arange(trees.rows + 1, dtype=torch.int32, device="cuda"),
                              (at + 1).to(torch.int32), **extra)
    assert torch.equal(q, want_q)
    touched = torch.zeros(before[0].shape[0], page, dtype=torch.bool, device="cuda")
    rows, row = torch.arange(trees.rows, device="cuda"), 0
    own = table[rows, at // page].long(), at % page
    for b, (n, t) in enumerate(zip(trees.new, trees.total)):
        p = torch.arange(t - n, t, device="cuda")
        where = trees.table[b, p // page].long(), p % page
        touched[where] = True
        mine = own[0][row:row + n], own[1][row:row + n]
        assert torch.equal(trees.k_pages[where[0], :, where[1]], alone_k[mine[0], :, mine[1]])
        assert torch.equal(trees.v_pages[where[0], :, where[1]], alone_v[mine[0], :, mine[1]])
        row += n
    keep = ~touched[:, None, :, None]
    assert torch.equal(trees.k_pages * keep, before[0] * keep) and torch.equal(trees.v_pages * keep, before[1] * keep)
    assert _lib.device_status() == 0


def test_append_many_nodes():
    """A large batch (two warps a token) writes what a small one does."""
    parents = [draft(64, 5, seed=i) for i in range(40)]
    trees = Trees(parents, [100 + 3 * i for i in range(40)], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16)
    qkv = torch.randn(trees.rows, 12 * 128, device="cuda")
    angles = torch.rand(300, 64, device="cuda") * 6
    extra = dict(heads=8, rope_cos=angles.cos(), rope_sin=angles.sin())
    q = ops.paged_append(qkv, trees.k_pages, trees.v_pages, trees.table, trees.offsets, trees.lens, parents=trees.parents,
                         **extra)
    k_pages, v_pages = trees.k_pages.clone(), trees.v_pages.clone()
    for b in range(40):
        rows = slice(64 * b, 64 * b + 64)
        one = ops.paged_append(qkv[rows], trees.k_pages, trees.v_pages, trees.table[b:b + 1], trees.offsets[:2],
                               trees.lens[b:b + 1], parents=trees.parents[rows].clone(), **extra)
        assert torch.equal(one, q[rows])
    assert torch.equal(torch.nan_to_num(trees.k_pages), torch.nan_to_num(k_pages))
    assert torch.equal(torch.nan_to_num(trees.v_pages), torch.nan_to_num(v_pages))


def test_append_bad_tables_are_reported_and_harmless():
    trees = Trees([draft(3, 2), draft(2, 1)], [20, 30], heads=4, kv_heads=2, dim=128, page=16, dtype=torch.float16, stale=5.0)
    qkv = torch.randn(5, 8 * 128, device="cuda")
    args = trees.k_pages, trees.v_pages, trees.table, trees.offsets, trees.lens
    before = trees.k_pages.clone()
    trees.lens[0] = 2  # fewer tokens than nodes: nothing is written
    ops.paged_append(qkv, *args, heads=4, parents=trees.parents)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert (trees.k_pages != before).any(-1).any(1).sum().item() == 2
    trees.lens[0] = 20
    trees.parents[1] = 1  # its own parent: counts as a root
    ones = torch.ones(40, 64, device="cuda")
    ops.paged_append(qkv, *args, heads=4, parents=trees.parents, rope_cos=ones, rope_sin=ones)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    trees.parents[1] = 0
    ops.paged_append(qkv, *args, heads=4, parents=trees.parents, rope_cos=ones[:8], rope_sin=ones[:8])
    assert _lib.device_status() == _lib.STATUS_BAD_POSITION
