"""What a verify step of drafted trees does beside attention and append: norm to
int8 rows, acceptance, and the move of the accepted tokens."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib, ops  # noqa: E402
from test_gpu_tree import Trees, draft  # noqa: E402

VALUES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---- residual addition, norm, int8 rows -------------------------------------------
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 32), (1, 2560), (70, 2560), (5, 2056), (9, 9728), (2, 10248), (3, 40000)])
@pytest.mark.parametrize("dtype", list(VALUES))
@pytest.mark.parametrize("delta", [None, *VALUES])
def test_rmsnorm_quantize_rows(rows, width, dtype, delta):
    """The same bits as the addition, rmsnorm and quantize_rows in fp32, and the definition in 64 bits: a code is off by
    half a step and what the fp32 chain adds, less than (width / 256 + 30) 2^-24 of at most 127 steps."""
    g = torch.Generator("cuda").manual_seed(rows + width)
    x = torch.empty(rows, width, device="cuda").normal_(generator=g).to(VALUES[dtype])
    d = None if delta is None else torch.empty(rows, width, device="cuda").normal_(generator=g).to(VALUES[delta])
    weight = 1 + 0.3 * torch.empty(width, device="cuda").normal_(generator=g)
    before = x.clone()
    x8, scales, sums = ops.rmsnorm_quantize_rows(x, weight, 1e-6, delta=d)
    total = before.float() if d is None else before.float() + d.float()
    assert torch.equal(x, total.to(x.dtype))  # in place
    normed = torch.stack([ops.rmsnorm(row.contiguous(), weight, 1e-6) for row in total])
    want8, want_scales, want_sums = ops.quantize_rows(normed)
    assert torch.equal(x8, want8) and torch.equal(scales, want_scales) and torch.equal(sums, want_sums)
    y = total.double()
    y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    scale = y.abs().amax(-1, keepdim=True).clamp(min=1e-5) / 127
    more = 127 * (width / 256 + 30) * 2.0 ** -24
    assert ((x8.double() - y / scale).abs() <= 0.5 + more).all()
    assert ((scales.double() - scale[:, 0]).abs() <= (width / 256 + 30) * 2.0 ** -24 * scale[:, 0]).all()
    assert torch.equal(sums, x8.sum(-1, dtype=torch.int32))


@pytest.mark.parametrize("rows,width,dtype,delta", [
    (2000, 2560, "fp32", "bf16"), (1500, 9728, "bf16", "bf16"), (700, 9728, "fp16", None), (3001, 1032, "bf16", "fp32"),
    (2500, 2048, "fp32", None), (1301, 520, "fp16", "fp16"), (900, 1024, "fp32", "fp32"), (5000, 4104, "bf16", None)])
def test_norm_of_many_rows_is_that_of_each(rows, width, dtype, delta):
    """However the rows are shared out, every one has the bits that it has alone."""
    g = torch.Generator("cuda").manual_seed(width)
    x = torch.empty(rows, width + 8, device="cuda").normal_(generator=g).to(VALUES[dtype])[:, 8:]
    d = None if delta is None else torch.empty(rows, width, device="cuda").normal_(generator=g).to(VALUES[delta])
    weight = torch.rand(width, generator=g, device="cuda")
    out = torch.full((rows + 1, width), 5.0, dtype=VALUES[dtype], device="cuda")
    got = ops.rmsnorm_quantize_rows(x, weight, 1e-6, delta=d, out=out[:rows])
    total = x.float() if d is None else x.float() + d.float()
    if d is not None:
        assert torch.equal(out[:rows], total.to(x.dtype))
    assert (out[rows] == 5).all()
    for part in range(0, rows, 97):
        few = total[part:part + 97].contiguous()  # fp32 rows of the same values, few at a time
        want = ops.rmsnorm_quantize_rows(few, weight, 1e-6)
        assert all(torch.equal(a[part:part + 97], b) for a, b in zip(got, want))
    normed = torch.stack([ops.rmsnorm(total[r].contiguous(), weight, 1e-6) for r in (0, 1, rows // 2, rows - 1)])
    want8, want_scales, want_sums = ops.quantize_rows(normed)
    for k, r in enumerate((0, 1, rows // 2, rows - 1)):
        assert torch.equal(got[0][r], want8[k]) and got[1][r] == want_scales[k] and got[2][r] == want_sums[k]


def test_norm_strided_rows_and_outputs():
    x, d = torch.randn(2, 40, 2560, device="cuda"), torch.randn(40, 2, 2560, device="cuda")
    weight = torch.rand(2560, device="cuda")
    out = torch.zeros(40, 3, 2560, device="cuda")
    x8, scales, sums = ops.rmsnorm_quantize_rows(x[1], weight, 1e-6, delta=d[:, 1], out=out[:, 2])
    want = ops.rmsnorm_quantize_rows(x[1].clone(), weight, 1e-6, delta=d[:, 1].contiguous())
    assert torch.equal(out[:, 2], x[1] + d[:, 1]) and (out[:, :2] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip((x8, scales, sums), want))
    alone = ops.rmsnorm_quantize_rows(x[1][:1], weight, 1e-6)
    assert alone[0].shape == (1, 2560)
    assert ops.rmsnorm_quantize_rows(x[1][:0], weight, 1e-6)[0].shape == (0, 2560)


def test_norm_of_zeros_and_small_rows():
    """An all-zero row has scale 1e-5 / 127 and zero codes; subnormal rows stay finite."""
    x = torch.zeros(3, 256, device="cuda")
    x[1] = 1e-30
    x[2, 7] = 1e-38
    x8, scales, sums = ops.rmsnorm_quantize_rows(x, torch.ones(256, device="cuda"), 1e-6)
    assert (x8[0] == 0).all() and sums[0] == 0 and torch.isfinite(scales).all()
    assert scales[0].item() == pytest.approx(1e-5 / 127, rel=1e-6)


def test_norm_feeds_the_int4_products():
    """Its output is int4_gemm's input."""
    x, delta = torch.randn(37, 512, device="cuda"), torch.randn(37, 512, device="cuda")
    weight = torch.rand(512, device="cuda")
    w = torch.randint(0, 256, (256, 256), dtype=torch.uint8, device="cuda")
    scales = torch.rand(256, device="cuda")
    got = ops.int4_gemm(*ops.rmsnorm_quantize_rows(x, weight, 1e-6, delta=delta), w, scales)
    rows = torch.stack([ops.rmsnorm(row.contiguous(), weight, 1e-6) for row in x])  # (x holds the sum)
    assert torch.equal(got, ops.int4_gemm_rows(rows, w, scales))


def test_norm_refusals():
    x, weight = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="weight"):
        ops.rmsnorm_quantize_rows(x, weight[:32], 1e-6)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ops.rmsnorm_quantize_rows(x.double(), weight, 1e-6)
    with pytest.raises(ValueError, match="x's shape"):
        ops.rmsnorm_quantize_rows(x, weight, 1e-6, delta=x[:2])
    with pytest.raises(ValueError, match="out must be torch.float32"):
        ops.rmsnorm_quantize_rows(x, weight, 1e-6, delta=x, out=x.half())
    with pytest.raises(ValueError, match="weight must be torch.float32"):
        ops.rmsnorm_quantize_rows(x, weight.half(), 1e-6)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.rmsnorm_quantize_rows(torch.zeros(4, 60, device="cuda"), weight[:60].clone(), 1e-6)
    with pytest.raises(ValueError, match="must be contiguous"):
        ops.rmsnorm_quantize_rows(torch.zeros(64, 4, device="cuda").t(), weight, 1e-6)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.rmsnorm_quantize_rows(x.cpu(), weight, 1e-6)


# ---- acceptance ------------------------------------------------------------------
def follow(trees, tokens, targets, max_path):
    """(paths, counts, next tokens), by the definition."""
    paths, counts, following, first = [], [], [], 0
    for tree in trees:
        path = [0] if tree else []
        while path and len(path) < max_path:
            wanted = targets[first + path[-1]]
            more = [i for i, p in enumerate(tree) if p == path[-1] and tokens[first + i] == wanted]
            if not more:
                break
            path.append(more[0])
        paths.append(path + [-1] * (max_path - len(path)))
        counts.append(len(path))
        following.append(targets[first + path[-1]] if path else -1)
        first += len(tree)
    return paths, counts, following


def drafted(trees, vocab, seed, agree=0.7):
    """(targets, tokens) of all nodes: a token is its parent's target with probability `agree`."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(map(len, trees))
    targets = torch.randint(0, vocab, (rows,), generator=g).tolist()
    wrong = torch.randint(0, vocab, (rows,), generator=g).tolist()
    right = (torch.rand(rows, generator=g) < agree).tolist()
    tokens, first = [], 0
    for tree in trees:
        tokens += [targets[first + max(p, 0)] if right[first + i] else wrong[first + i] for i, p in enumerate(tree)]
        first += len(tree)
    return targets, tokens


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda").reshape(-1)


def offsets_of(trees):
    return torch.tensor([0] + [len(t) for t in trees], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def check_accept(trees, tokens, wanted, max_path, **kwargs):
    path, counts, following, chosen = ops.accept_tree(ints(tokens), ints([p for t in trees for p in t]), offsets_of(trees),
                                                      max_path=max_path, **kwargs)
    want = follow(trees, tokens, wanted, max_path)
    assert (path.tolist(), counts.tolist(), following.tolist()) == want
    assert chosen.tolist() == wanted and _lib.device_status() == 0
    return path, counts


FORESTS = {"one": [draft(1, 1)], "chain": [draft(40, 1)], "few": [draft(8, 3), [], draft(5, 2, roots=2), [], []],
           "many": [draft(1 + i % 16, 4, seed=i) for i in range(70)], "large": [draft(256, 2), draft(256, 1), draft(200, 256)],
           "sequences": [draft(2, 1) for _ in range(600)]}


@pytest.mark.parametrize("forest", list(FORESTS))
@pytest.mark.parametrize("vocab", [2, 5, 1000, 50257])
@pytest.mark.parametrize("dtype", list(VALUES))
def test_accept_logits(forest, vocab, dtype):
    trees = FORESTS[forest]
    targets, tokens = drafted(trees, vocab, seed=vocab)
    g = torch.Generator("cuda").manual_seed(1)
    wide = torch.empty(len(targets), vocab + 3, device="cuda").normal_(generator=g).to(VALUES[dtype])
    logits = wide[:, 1:vocab + 1]  # rows that start anywhere
    at = torch.tensor(targets, device="cuda")[:, None]
    logits.scatter_(1, at, logits.amax(-1, keepdim=True) + 1)
    for max_path in (1, 3, 256):
        check_accept(trees, tokens, targets, max_path, logits=logits)
    check_accept(trees, tokens, targets, 7, targets=ints(targets))


@pytest.mark.parametrize("dtype", list(VALUES))
def test_accept_ties_and_values_that_are_not_finite(dtype):
    """The first maximum, as numpy has it: a NaN is the largest, 0 equals -0."""
    vocab, nan, inf = 20000, float("nan"), float("inf")
    logits = torch.zeros(12, vocab, device="cuda", dtype=VALUES[dtype])
    logits[0, 7777:7779] = 1
    logits[1] = -inf
    logits[2, 5], logits[2, 19999] = inf, inf
    logits[3, 9], logits[3, 10001], logits[3, 3] = nan, nan, inf
    logits[4] = nan
    logits[5, 0] = -0.0
    logits[6, 1:] = -0.0
    logits[6, 0] = -1
    logits[7] = -3
    logits[7, 19998] = -2.5
    logits[8, 11] = -nan
    logits[9] = -inf
    logits[9, 123] = -65504.0
    logits[10] = torch.arange(vocab, device="cuda").to(VALUES[dtype])
    want = logits.float().cpu().numpy().argmax(-1).tolist()
    assert want[:10] == [7777, 0, 5, 9, 0, 0, 1, 19998, 11, 123]
    trees = [draft(12, 3)]
    check_accept(trees, [5] * 12, want, 12, logits=logits)


def test_accept_takes_the_first_child_that_agrees():
    trees = [[-1, 0, 0, 0, 1, 2, 2, 5]]
    targets, tokens = [9, 1, 4, 1, 1, 6, 7, 8], [0, 3, 9, 9, 9, 4, 4, 6]
    path, counts = check_accept(trees, tokens, targets, 8, targets=ints(targets))
    assert path[0, :counts[0]].tolist() == [0, 2, 5, 7]


def test_accept_workspace_is_left_ready():
    trees = FORESTS["many"]
    rows = sum(map(len, trees))
    workspace = ops.accept_workspace(rows, len(trees))
    for seed in range(4):
        targets, tokens = drafted(trees, 3000, seed)
        logits = torch.randn(rows, 3000, device="cuda")
        logits.scatter_(1, torch.tensor(targets, device="cuda")[:, None], 9.0)
        check_accept(trees, tokens, targets, 16, logits=logits, workspace=workspace)
        few = FORESTS["few"]
        targets, tokens = drafted(few, 100, seed)
        logits = torch.zeros(13, 100, device="cuda")
        logits.scatter_(1, torch.tensor(targets, device="cuda")[:, None], 9.0)
        check_accept(few, tokens, targets, 4, logits=logits, workspace=workspace)


def test_accept_rows_of_no_sequence_and_bad_offsets():
    trees = FORESTS["few"]
    targets, tokens = drafted(trees, 50, 3)
    logits = torch.zeros(16, 50, device="cuda")
    logits.scatter_(1, torch.tensor(targets + [1, 2, 3], device="cuda")[:, None], 9.0)
    parents = ints([p for t in trees for p in t] + [99, -7, 5])
    offsets, workspace = offsets_of(trees), ops.accept_workspace(16, 5)
    path, counts, following, chosen = ops.accept_tree(ints(tokens + [0, 0, 0]), parents, offsets, logits, max_path=8,
                                                      workspace=workspace)
    want = follow(trees, tokens, targets, 8)
    assert (path.tolist(), counts.tolist(), following.tolist()) == want
    assert chosen[:13].tolist() == targets and _lib.device_status() == 0
    for bad in ([0, 9, 8, 13, 13, 13], [0, 8, 8, 13, 13, 17], [-1, 8, 8, 13, 13, 13]):
        path, counts, following, _ = ops.accept_tree(ints(tokens + [0, 0, 0]), parents, ints(bad), logits, max_path=8,
                                                     workspace=workspace)
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        assert (path == -1).all() and (counts == 0).all() and (following == -1).all()
    # the workspace is as it was
    path, counts, following, _ = ops.accept_tree(ints(tokens + [0, 0, 0]), parents, offsets, logits, max_path=8,
                                                 workspace=workspace)
    assert (path.tolist(), counts.tolist(), following.tolist()) == want and _lib.device_status() == 0
    # given targets: the other sequences are answered
    path, counts, following, _ = ops.accept_tree(ints(tokens), parents[:13], ints([0, 9, 8, 13, 13, 13]), targets=ints(targets),
                                                 max_path=8)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert counts[1] == 0 and following[1] == -1 and counts[2] >= 1


def test_accept_parents_out_of_range_and_large_trees():
    trees = [[-1, 0, 1], draft(257, 1), [-1, 0]]
    rows = 262
    tokens, targets = [4] * rows, [4] * rows
    parents = [p for t in trees for p in t]
    parents[2] = 2
    logits = torch.zeros(rows, 9, device="cuda")
    logits[:, 4] = 1
    for how in (dict(logits=logits), dict(targets=ints(targets))):
        path, counts, following, _ = ops.accept_tree(ints(tokens), ints(parents), offsets_of(trees), max_path=5, **how)
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        assert counts.tolist() == [2, 0, 2] and following.tolist() == [4, -1, 4]
        assert path.tolist() == [[0, 1, -1, -1, -1], [-1] * 5, [0, 1, -1, -1, -1]]


def test_batches_without_nodes():
    none, offsets = ints([]), ints([0, 0, 0])
    for how in (dict(logits=torch.zeros(0, 9, device="cuda")), dict(targets=none)):
        path, counts, following, _ = ops.accept_tree(none, none, offsets, max_path=4, **how)
        assert path.tolist() == [[-1] * 4] * 2 and counts.tolist() == [0, 0] and following.tolist() == [-1, -1]
    path, counts, following, _ = ops.accept_tree(none, none, ints([0]), targets=none)
    assert path.shape[0] == counts.numel() == following.numel() == 0
    k = torch.randn(2, 4, 2, 16, 64, device="cuda").half()
    before, lens = k.clone(), ints([17, 0])
    lengths = ops.keep_tokens(k, k.clone(), ints([0, 1, 2, 3]).view(2, 2), offsets, lens, ints([[0], [-1]]).view(2, 1), ints([0, 0]))
    assert torch.equal(lengths, lens) and torch.equal(k, before) and _lib.device_status() == 0


def test_accept_refusals():
    tokens, parents, offsets = ints([1, 2]), ints([-1, 0]), ints([0, 2])
    logits = torch.zeros(2, 10, device="cuda")
    with pytest.raises(ValueError, match="either logits or targets"):
        ops.accept_tree(tokens, parents, offsets)
    with pytest.raises(ValueError, match="either logits or targets"):
        ops.accept_tree(tokens, parents, offsets, logits, targets=tokens)
    with pytest.raises(ValueError, match=r"logits must be \[rows\]"):
        ops.accept_tree(tokens, parents, offsets, logits[:1])
    with pytest.raises(ValueError, match="logits must be float32"):
        ops.accept_tree(tokens, parents, offsets, logits.double())
    with pytest.raises(ValueError, match="targets must hold"):
        ops.accept_tree(tokens, parents, offsets, targets=ints([1]))
    with pytest.raises(ValueError, match="max_path"):
        ops.accept_tree(tokens, parents, offsets, logits, max_path=0)
    with pytest.raises(ValueError, match="parents must hold"):
        ops.accept_tree(tokens, parents[:1], offsets, logits)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.accept_tree(tokens, parents, offsets, logits, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.accept_tree(tokens.cpu(), parents, offsets, logits)


# ---- the accepted tokens' move -----------------------------------------------------
def kept(pages, table, bases, paths, page):
    """The pages after the move, one (layer, token) after the other."""
    out = pages.clone()
    for b, path in enumerate(paths):
        for i, n in enumerate(path):
            a, z = bases[b] + n, bases[b] + i
            out[:, table[b][z // page], :, z % page] = out[:, table[b][a // page], :, a % page].clone()
    return out


@pytest.mark.parametrize("layers,kv_heads,dim,page,dtype", [
    (3, 8, 128, 16, torch.float16), (1, 1, 64, 16, torch.bfloat16), (2, 3, 64, 128, torch.float16), (36, 2, 128, 32, torch.bfloat16)])
def test_keep_tokens(layers, kv_heads, dim, page, dtype):
    """Every path that ascends: nodes that stay, sources that are targets of later nodes, page borders."""
    paths = [[0], [], [0, 1, 2], [0, 2, 3, 7, 8, 20], [3, 4], list(range(1, 40)), [0, 39], [0, 2, 4, 6, 8, 10, 12, 14, 16, 18, 20, 22]]
    nodes = [1, 5, 3, 21, 9, 40, 40, 23]
    bases = [0, 17, 15, 29, 16, 100, 3, 31]
    need = [-(-(a + n) // page) for a, n in zip(bases, nodes)]
    pages = sum(need) + 2
    ids = torch.randperm(pages).tolist()
    width = max(need) + 1
    table = [[-1] * width for _ in need]
    for row, n in zip(table, need):
        for j in range(n):
            row[j] = ids.pop()
    k = torch.randn(layers, pages, kv_heads, page, dim, device="cuda").to(dtype)
    v = torch.randn(layers, pages, kv_heads, page, dim, device="cuda").to(dtype)
    want_k, want_v = (kept(x, table, bases, paths, page) for x in (k, v))
    longest = max(map(len, paths))
    path = ints([p + [-1] * (longest - len(p)) for p in paths]).view(8, longest)
    args = (torch.tensor(table, dtype=torch.int32, device="cuda"), offsets_of([[0] * n for n in nodes]),
            ints([a + n for a, n in zip(bases, nodes)]), path, ints([len(p) for p in paths]))
    if layers == 1:
        lengths = ops.keep_tokens(k[0], v[0], *args)
    else:
        lengths = ops.keep_tokens(k, v, *args)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert lengths.tolist() == [a + len(p) for a, p in zip(bases, paths)]
    assert _lib.device_status() == 0


def test_keep_bad_paths_leave_their_sequence():
    k = torch.randn(2, 12, 2, 16, 64, device="cuda").half()
    v = torch.randn(2, 12, 2, 16, 64, device="cuda").half()
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(4, 3)
    offsets, lens = ints([0, 6, 12, 18, 24]), ints([30, 31, 32, 33])
    bases = [24, 25, 26, 27]
    good = [0, 2, 5]
    for bad in ([0, 2, 2], [1, 0, 3], [-1, 2, 3], [0, 2, 6], [0, 1 << 30, 3], [-(1 << 31), 0, 1]):
        before = k.clone(), v.clone()
        lengths = ops.keep_tokens(k, v, table, offsets, lens, ints([good, bad, good, good]).view(4, 3), ints([3, 3, 3, 3]))
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        assert lengths.tolist() == [27, 31, 29, 30]
        held = table.tolist()
        paths = [good, [], good, good]
        assert torch.equal(k, kept(before[0], held, bases, paths, 16)) and torch.equal(v, kept(before[1], held, bases, paths, 16))
    for count in (-1, 4, 7, 1 << 30):  # past the path, past the tree
        before = k.clone()
        lengths = ops.keep_tokens(k, v, table, offsets, lens, ints([good] * 4).view(4, 3), ints([0, 0, count, 0]))
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        assert lengths.tolist() == [24, 25, 32, 27] and torch.equal(k, before)
    lens[3] = 1 << 20  # past its table
    lengths = ops.keep_tokens(k, v, table, offsets, lens, ints([good] * 4).view(4, 3), ints([0, 0, 0, 3]))
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE and lengths.tolist() == [24, 25, 26, 1 << 20]
    lens[3] = 33
    table[3, 2] = 12  # a page that is not there: that token does not move
    ops.keep_tokens(k, v, table, offsets, lens, ints([[0, 5, 5]] + [[0, 5, -1]] * 3).view(4, 3), ints([0, 0, 0, 2]))
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE


def test_keep_refusals():
    k = torch.zeros(2, 4, 2, 16, 64, device="cuda").half()
    table, offsets, lens = ints([0, 1]).view(1, 2), ints([0, 3]), ints([20])
    path, counts = ints([0, 2]).view(1, 2), ints([2])
    with pytest.raises(ValueError, match="path must be"):
        ops.keep_tokens(k, k.clone(), table, offsets, lens, path[0], counts)
    with pytest.raises(ValueError, match="counts"):
        ops.keep_tokens(k, k.clone(), table, offsets, lens, path, ints([2, 2]))
    with pytest.raises(ValueError, match="k_pages and v_pages"):
        ops.keep_tokens(k, k[:1].clone(), table, offsets, lens, path, counts)
    with pytest.raises(ValueError, match="contiguous"):
        ops.keep_tokens(k[:, 1:], k[:, 1:], table, offsets, lens, path, counts)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.keep_tokens(k, k.clone(), table, offsets, lens, path, counts, lengths=lens)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.keep_tokens(k, k.clone(), table, offsets, lens, path, counts, lengths=counts)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        ops.keep_tokens(k.float(), k.float(), table, offsets, lens, path, counts)


# ---- together -----------------------------------------------------------------------
def test_a_layer_of_a_verify_step():
    """Append, attention, acceptance and keep of two rounds: what a decoder that feeds the accepted tokens one by one has
    in its cache and gets for them."""
    heads, kv_heads, dim, page, dtype = 8, 2, 128, 16, torch.float16
    width = (heads + 2 * kv_heads) * dim
    g = torch.Generator("cuda").manual_seed(0)
    angles = torch.rand(400, dim // 2, generator=g, device="cuda") * 6
    extra = dict(heads=heads, rope_cos=angles.cos(), rope_sin=angles.sin())
    shape = (24, kv_heads, page, dim)
    k, v, slow_k, slow_v = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(4))
    table = torch.randperm(24, generator=g, device="cuda").to(torch.int32).view(2, 12)
    lens = ints([40, 3])
    context = torch.randn(43, width, generator=g, device="cuda")
    for pages in ((k, v), (slow_k, slow_v)):
        ops.paged_append(context, *pages, table, ints([0, 40, 43]), lens, **extra)
    for turn in range(2):
        trees = [draft(30, 4, seed=turn), draft(7, 2, seed=turn + 5)]
        targets, tokens = drafted(trees, 6, seed=turn)
        parents, offsets = ints([p for t in trees for p in t]), offsets_of(trees)
        qkv = torch.randn(37, width, generator=g, device="cuda")
        with_nodes = lens + ints([30, 7])
        q = ops.paged_append(qkv, k, v, table, offsets, with_nodes, parents=parents, **extra)
        out = ops.paged_tree_attention(q, k, v, table, offsets, with_nodes, parents)
        path, counts, _, _ = ops.accept_tree(ints(tokens), parents, offsets, targets=ints(targets), max_path=30)
        new = ops.keep_tokens(k, v, table, offsets, with_nodes, path, counts)
        for b in range(2):
            for i in range(int(counts[b])):  # one accepted token after the other
                row = int(offsets[b]) + int(path[b, i])
                at = lens[b:b + 1] + i + 1
                one = ops.paged_append(qkv[row:row + 1], slow_k, slow_v, table[b:b + 1], ints([0, 1]), at, **extra)
                assert torch.equal(one[0], q[row])
                want = ops.paged_attention(one, slow_k, slow_v, table[b:b + 1], ints([0, 1]), at)
                # two roundings of p and of the result (2^-11 each, of values below max|v|) on both sides
                assert (want[0].float() - out[row].float()).abs().max() <= 4 * 2.0 ** -11 * float(v.float().abs().max())
        assert torch.equal(new, lens + counts)
        lens = new
        for b in range(2):
            p = torch.arange(int(lens[b]), device="cuda")
            where = table[b, p // page].long(), p % page
            assert torch.equal(k[where[0], :, where[1]], slow_k[where[0], :, where[1]])
            assert torch.equal(v[where[0], :, where[1]], slow_v[where[0], :, where[1]])
    assert int(lens[0]) > 42 and _lib.device_status() == 0


def test_a_captured_step_follows_its_inputs():
    """Norm, append, attention, acceptance and keep in one graph, replayed with other trees, logits and lengths, on another
    stream than the tensors'."""
    heads, kv_heads, dim, page, vocab = 8, 2, 128, 16, 700
    width = (heads + 2 * kv_heads) * dim
    g = torch.Generator("cuda").manual_seed(1)
    weight = torch.rand(width, generator=g, device="cuda") + 0.5
    angles = torch.rand(400, dim // 2, generator=g, device="cuda") * 6
    rope = dict(rope_cos=angles.cos(), rope_sin=angles.sin())
    table = torch.randperm(40, generator=g, device="cuda").to(torch.int32).view(2, 20)
    offsets = ints([0, 40, 47])

    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        trees = [draft(40, 3, seed=seed), draft(7, 2, seed=seed + 1)]
        targets, tokens = drafted(trees, vocab, seed)
        logits = torch.randn(47, vocab, generator=g, device="cuda")
        logits.scatter_(1, torch.tensor(targets, device="cuda")[:, None], 9.0)
        pages = torch.randn(2, 40, kv_heads, page, dim, generator=g, device="cuda").half()
        return dict(x=torch.randn(47, width, generator=g, device="cuda"), delta=torch.randn(47, width, generator=g, device="cuda"),
                    parents=ints([p for t in trees for p in t]), tokens=ints(tokens), logits=logits,
                    lens=ints([40 + 31 * seed, 7 + 90 * seed]), k=pages[0].clone(), v=pages[1].clone())

    attend, accept = ops.paged_workspace(), ops.accept_workspace(47, 2)

    def step(s):
        x8, scales, sums = ops.rmsnorm_quantize_rows(s["x"], weight, 1e-6, delta=s["delta"])
        q = ops.paged_append(s["x"], s["k"], s["v"], table, offsets, s["lens"], heads=heads, parents=s["parents"], **rope)
        out = ops.paged_tree_attention(q, s["k"], s["v"], table, offsets, s["lens"], s["parents"], workspace=attend)
        path, counts, following, targets = ops.accept_tree(s["tokens"], s["parents"], offsets, s["logits"], max_path=9,
                                                           workspace=accept)
        lengths = ops.keep_tokens(s["k"], s["v"], table, offsets, s["lens"], path, counts)
        return [x8, scales, sums, s["x"], out, path, counts, following, targets, lengths, s["k"], s["v"]]

    want = {seed: [t.clone() for t in step(inputs(seed))] for seed in (1, 2, 3)}
    held = inputs(1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step(held)
    for seed in (2, 3, 1, 3):
        fresh = inputs(seed)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for name, t in held.items():
                t.copy_(fresh[name])
            graph.replay()
        stream.synchronize()
        for a, b in zip(got, want[seed]):
            assert torch.equal(a, b)
    assert _lib.device_status() == 0


def test_accept_and_keep_run_on_the_current_stream():
    trees = FORESTS["few"]
    targets, tokens = drafted(trees, 50, 3)
    logits = torch.zeros(13, 50, device="cuda")
    want = torch.zeros_like(logits).scatter_(1, torch.tensor(targets, device="cuda")[:, None], 9.0)
    k = torch.randn(1, 8, 1, 16, 64, device="cuda").half()
    v, table = k.clone(), torch.arange(5, dtype=torch.int32, device="cuda").view(5, 1)
    offsets, lens, parents = offsets_of(trees), ints([9, 1, 7, 0, 3]), ints([p for t in trees for p in t])
    ids = ints(tokens)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        workspace = ops.accept_workspace(13, 5)
        torch.cuda._sleep(20_000_000)
        logits.copy_(want)
        path, counts, following, _ = ops.accept_tree(ids, parents, offsets, logits, max_path=8, workspace=workspace)
        lengths = ops.keep_tokens(k, v, table, offsets, lens, path, counts)
    stream.synchronize()
    paths, numbers, tokens_after = follow(trees, tokens, targets, 8)
    assert (path.tolist(), counts.tolist(), following.tolist()) == (paths, numbers, tokens_after)
    assert lengths.tolist() == [n - len(t) + c for n, t, c in zip(lens.tolist(), trees, numbers)]
