"""The operators of a verify step of drafted token trees: what is measured, and their plain forms.

A draft proposes a tree of tokens for each sequence of a paged K/V cache; one
step of the model runs all its nodes and keeps the branch that agrees with it.
A sequence's nodes are rows q_offsets[b] .. q_offsets[b + 1] - 1 of the batch;
parents[row] is a node's parent within its sequence (-1: it follows the tokens
in the cache, of which there are kv_lens[b] - nodes). Node i lies in the cache
at context + i and stands at position context + depth.

norm       residual addition, RMSNorm and int8 rows with scales: what the
           int4 products of the step take
append     norm and rotate the nodes' q and k by their positions, write k and
           v to their places in the pages
attention  of the nodes over the pages: a node sees the context (optionally a
           window and a few first tokens of it), its ancestors and itself
accept     the model's greedy token of every row, and the branch that agrees
keep       the accepted nodes' K and V, moved behind the context in every layer

`run` computes them with elementary torch operations in 32 bits, or, where
`own` is set, with the framework's operators. `exact` is their definition in
64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
WORKSPACE_BYTES = 64 << 20
MAX_POSITION, ROPE_THETA, EPS = 40960, 1000000.0, 1e-6
MOST_NODES = 256


def listed():
    cache = {"dtype": "fp16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16}
    attention = dict(cache, op="attention", window=0, sinks=0, spread=4, roots=1)
    append = dict(cache, op="append", source="fp32", spread=4, roots=1)
    accept = {"op": "accept", "dtype": "fp32", "vocab": 151936, "spread": 4}
    keep = dict(cache, op="keep", layers=36, spread=4)
    return [
        # one user's drafted tokens, about a thousand tokens in: the latency of one layer's attention
        dict(attention, name="tree one", sequences=1, nodes=8, kv_min=1000, kv_max=1000, lens=1),
        # a chat server's verify step: 64 sequences of every length up to two thousand, 8 to 16 nodes each
        dict(attention, name="trees ragged", dtype="bf16", sequences=64, nodes=16, kv_min=1, kv_max=2100, lens=2),
        # long documents with 32 nodes each: the whole cache is read
        dict(attention, name="trees long", sequences=16, nodes=32, kv_min=32768, kv_max=32768, page=64, lens=3),
        # streaming sessions under a window, wide trees, 3 q heads a kv head
        dict(attention, name="trees window", dtype="bf16", heads=24, head_dim=64, sequences=24, nodes=61, kv_min=3000,
             kv_max=12000, page=32, window=2048, sinks=4, spread=30, roots=2, lens=4),
        # one layer's q, k and v of one user's tree, as the projection leaves them
        dict(append, name="append one", sequences=1, nodes=8, kv_min=1000, kv_max=1000, lens=5),
        # a large server's step: 128 sequences of 32 to 64 nodes
        dict(append, name="append many", dtype="bf16", sequences=128, nodes=64, kv_min=100, kv_max=1500, page=32, lens=6),
        # a chat server's 64 trees of 16 nodes: one norm of the step
        {"op": "norm", "name": "norm step", "dtype": "fp32", "delta": "fp32", "rows": 1024, "width": 2560},
        # a long prompt's rows on the way to the up projections' width, 16-bit residuals
        {"op": "norm", "name": "norm prompt", "dtype": "bf16", "delta": "bf16", "rows": 8192, "width": 9728},
        # one user's 8 nodes: the logits of a whole vocabulary each
        dict(accept, name="accept one", sequences=1, nodes=8, lens=7),
        # the chat server's: 64 trees of 8 to 16 nodes
        dict(accept, name="accept many", sequences=64, nodes=16, lens=8),
        # one user's accepted branch, in all layers
        dict(keep, name="keep one", sequences=1, nodes=8, kv_min=300, kv_max=300, lens=9),
        # the chat server's
        dict(keep, name="keep many", sequences=64, nodes=16, kv_min=1, kv_max=200, lens=10),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "norm", "accept", "keep"))
    if op == "norm":
        width = 8 * _log(rng, 4, 2048)
        return {"op": op, "dtype": rng.choice(("fp32", "fp16", "bf16")), "width": width,
                "delta": rng.choice(("none", "fp32", "fp16", "bf16")), "rows": _log(rng, 1, min(16384, (40 << 20) // width))}
    nodes = _log(rng, 1, MOST_NODES)
    spread = rng.choice((1, 2, 4, 16, nodes))
    if op == "accept":
        vocab = _log(rng, 100, 160000)
        most = min(128, (144 << 20) // (vocab * nodes))
        if most < 1:
            nodes, most = 64, 8
        return {"op": op, "dtype": rng.choice(("fp32", "fp16", "bf16")), "vocab": vocab, "nodes": nodes, "spread": spread,
                "sequences": _log(rng, 1, most), "lens": rng.randrange(1 << 20)}
    case = {"op": op, "dtype": rng.choice(("fp16", "bf16")), "kv_heads": rng.choice((1, 2, 4, 8)),
            "head_dim": rng.choice((64, 128, 128)), "page": rng.choice((16, 32, 64, 128)), "nodes": nodes,
            "spread": spread, "lens": rng.randrange(1 << 20)}
    case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 5, 8))
    if op == "keep":
        token_bytes = 4 * case["kv_heads"] * case["head_dim"]
        layers = _log(rng, 1, 40)
        sequences = _log(rng, 1, max(1, min(64, (1 << 30) // (token_bytes * layers * (nodes + 200)))))
        kv_max = nodes + rng.randrange(0, 150)
        return dict(case, layers=layers, sequences=sequences, kv_max=kv_max, kv_min=rng.randrange(0, kv_max + 1))
    if op == "append":
        sequences = _log(rng, 1, max(1, min(128, 8192 // nodes)))
        kv_max = nodes + _log(rng, 1, 4000)
        return dict(case, sequences=sequences, kv_max=kv_max, kv_min=rng.randrange(0, kv_max + 1),
                    source=rng.choice(("fp32", case["dtype"])), roots=rng.choice((1, 1, 2)))
    # the plain form's padded scores (sequences x heads x nodes x length) and keys are bounded
    sequences = _log(rng, 1, 64)
    most = min(MAX_POSITION, (1 << 29) // (sequences * case["heads"] * nodes), (1 << 19) // sequences)
    kv_max = max(nodes, _log(rng, nodes, max(nodes, most)))
    kv_min = kv_max if rng.random() < 0.3 else rng.randrange(0, kv_max + 1)
    windowed = rng.random() < 0.4
    return dict(case, sequences=sequences, kv_max=kv_max, kv_min=kv_min, roots=rng.choice((1, 1, 2)),
                window=_log(rng, 1, 8192) if windowed else 0, sinks=rng.choice((0, 1, 4, 16, 130)) if windowed else 0)


def _trees(case):
    """(parents of every sequence's nodes, tokens in the cache with them): the case's own, whatever the seed."""
    rng = random.Random(case["lens"])
    parents, total = [], []
    for _ in range(case["sequences"]):
        n = rng.randint((case["nodes"] + 1) // 2, case["nodes"])
        roots = min(case.get("roots", 1), n)
        parents.append([-1] * roots + [rng.randrange(max(0, i - case["spread"]), i) for i in range(roots, n)])
        total.append(n + max(0, rng.randint(case.get("kv_min", 0), case.get("kv_max", 0)) - n))
    return parents, total


def _paths(case, parents):
    """An accepted branch of every sequence: some first nodes that stay, then nodes that lie behind all of them."""
    rng = random.Random(case["lens"] + 1)
    paths = []
    for p in parents:
        count = rng.randint(1, max(1, min(len(p) // 2, 12)))
        stay = rng.randint(1, count)
        paths.append(list(range(stay)) + sorted(rng.sample(range(count, len(p)), count - stay)))
    return paths


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        return out.normal_(generator=g)

    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        return {"op": "norm", "x": normal(rows, width), "weight": 1 + 0.1 * normal(width, dtype=torch.float32),
                "delta": None if case["delta"] == "none" else 0.3 * normal(rows, width, dtype=DTYPES[case["delta"]]),
                "out": torch.empty(rows, width, dtype=dtype, device="cuda"),
                "values": torch.empty(rows, width, dtype=torch.float16, device="cuda")}

    parents, total = _trees(case)
    new = [len(p) for p in parents]
    rows = sum(new)
    state = {"op": case["op"], "dtype": dtype,
             "parents": torch.tensor([p for tree in parents for p in tree], dtype=torch.int32).cuda(),
             "q_offsets": torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda(),
             "max_query": max(new), "max_kv": max(total), "rows": rows}
    if case["op"] == "accept":
        # the model prefers one token of every row; a drafted token is its parent's preferred one, or a wrong one
        vocab = case["vocab"]
        logits = normal(rows, vocab)
        preferred = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        most = logits.amax(-1, keepdim=True)
        logits.scatter_(1, preferred[:, None], most + 1)
        first = torch.repeat_interleave(state["q_offsets"][:-1].long(), torch.tensor(new).cuda(), output_size=rows)
        right = torch.rand(rows, generator=g, device="cuda") < 0.6
        wrong = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        after = preferred[first + state["parents"].long().clamp(min=0)]
        state["tokens"] = torch.where(right, after, wrong).to(torch.int32)
        state.update(logits=logits, max_path=min(max(new), 16), workspace=torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda"))
        return state

    page, heads_dim = case["page"], (case["kv_heads"], case["page"], case["head_dim"])
    need = [-(-n // page) for n in total]
    pages = sum(need) + 7  # a few free ones
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(table.shape[1], device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[held] = ids[:sum(need)]
    state.update(page_table=table, kv_lens=torch.tensor(total, dtype=torch.int32, device="cuda"), heads=case["heads"])
    layers = (case["layers"],) if case["op"] == "keep" else ()
    state["k_pages"], state["v_pages"] = normal(*layers, pages, *heads_dim), normal(*layers, pages, *heads_dim)
    dim = case["head_dim"]
    if case["op"] == "keep":
        paths = _paths(case, parents)
        width = max(len(p) for p in paths)
        state["path"] = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).cuda()
        state["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
    elif case["op"] == "append":
        state["qkv"] = normal(rows, (case["heads"] + 2 * case["kv_heads"]) * dim, dtype=DTYPES[case["source"]]) * 3
        state["norm_q"] = 1 + 0.02 * normal(dim, dtype=torch.float32)
        state["norm_k"] = 1 + 0.02 * normal(dim, dtype=torch.float32)
        inv = 1.0 / ROPE_THETA ** (torch.arange(0, dim, 2, dtype=torch.float32, device="cuda") / dim)
        angles = torch.arange(MAX_POSITION, dtype=torch.float32, device="cuda")[:, None] * inv[None]
        state["cos"], state["sin"] = angles.cos(), angles.sin()
    else:
        state["q"] = normal(rows, case["heads"], dim) * 1.5  # normalised heads: scores of a few units
        state["window"], state["sinks"] = case["window"], case["sinks"]
        state["out"] = torch.empty_like(state["q"])
        state["lse"] = torch.empty(rows, case["heads"], dtype=torch.float32, device="cuda")
        state["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    return state


# ---- the plain forms ---------------------------------------------------------------
def _rows_of(s):
    """Of every row: its sequence and its index there."""
    offsets = s["q_offsets"].long()
    sequence = torch.repeat_interleave(torch.arange(offsets.numel() - 1, device="cuda"), offsets[1:] - offsets[:-1],
                                       output_size=s["rows"])
    return sequence, torch.arange(s["rows"], device="cuda") - offsets[sequence]


def _ancestors(s, sequence, index):
    """[sequences, nodes, nodes]: 1 where the second node is an ancestor of the first, or itself. With P the parents as
    a (strictly lower triangular) matrix that is I + P + P^2 + ..., the inverse of I - P."""
    batch, n = s["q_offsets"].numel() - 1, s["max_query"]
    parent = s["parents"].long()
    inner = parent >= 0
    eye = torch.eye(n, device="cuda").expand(batch, n, n)
    step = eye.clone()
    step[sequence[inner], index[inner], parent[inner]] = -1.0
    return torch.linalg.solve_triangular(step, eye, upper=False, unitriangular=True)


def _plain_norm(s):
    x = s["x"].float()
    if s["delta"] is not None:
        x = x + s["delta"].float()
    y = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * s["weight"]
    most = y.abs().amax(-1, keepdim=True).clamp(min=1e-5)
    codes = torch.round(y * (127.0 / most)).clamp(-127, 127)
    scales = most / 127.0
    return {"x": x.to(s["x"].dtype), "values": (codes * scales).half(), "scales": scales[:, 0]}


def _plain_append(s):
    heads, kv_heads, dim = s["heads"], s["k_pages"].shape[1], s["k_pages"].shape[3]
    sequence, index = _rows_of(s)
    context = s["kv_lens"].long() - (s["q_offsets"][1:] - s["q_offsets"][:-1])
    depth = _ancestors(s, sequence, index)[sequence, index].sum(-1).round().long() - 1
    x = s["qkv"].float().view(s["rows"], heads + 2 * kv_heads, dim)
    q, k, v = x.split((heads, kv_heads, kv_heads), dim=1)
    cos, sin = (s[name][context[sequence] + depth][:, None] for name in ("cos", "sin"))

    def turned(t, weight):
        t = t * (1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)) * weight
        a, b = t.chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)

    page, slot = s["k_pages"].shape[2], context[sequence] + index
    held, slot = s["page_table"][sequence, slot // page].long(), slot % page
    s["k_pages"][held, :, slot] = turned(k, s["norm_k"]).to(s["dtype"])
    s["v_pages"][held, :, slot] = v.to(s["dtype"])
    return {"q": turned(q, s["norm_q"]).to(s["dtype"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    rows, heads, dim = s["q"].shape
    kv_heads, page = s["k_pages"].shape[1:3]
    sequence, index = _rows_of(s)
    batch, longest, query = s["kv_lens"].numel(), s["max_kv"], s["max_query"]
    context = s["kv_lens"].long() - (s["q_offsets"][1:] - s["q_offsets"][:-1])
    ancestors = _ancestors(s, sequence, index)
    depth = ancestors.sum(-1).round().long() - 1                            # [batch, query]
    keys = torch.arange(longest, device="cuda")
    held = s["page_table"][:, keys // page].long().clamp(min=0)            # [batch, longest]
    k = s["k_pages"][held, :, keys % page].float()                          # [batch, longest, kv_heads, dim]
    v = s["v_pages"][held, :, keys % page].float()
    v = v.masked_fill_((keys[None] >= s["kv_lens"][:, None])[:, :, None, None], 0.0)
    q = torch.zeros(batch, query, heads, dim, dtype=torch.float32, device="cuda")
    q[sequence, index] = s["q"].float()
    node = (keys[None] - context[:, None]).clamp(min=0, max=query - 1)      # [batch, longest]
    drafted = keys[None] >= context[:, None]
    stands = torch.where(drafted, context[:, None] + depth.gather(1, node), keys[None])
    seen = torch.where(drafted[:, None], ancestors.gather(2, node[:, None].expand(-1, query, -1)) > 0.5, True)
    seen = seen & (keys[None] < s["kv_lens"][:, None])[:, None]
    if s["window"]:
        near = (context[:, None] + depth)[:, :, None] - stands[:, None] < s["window"]
        seen &= near | (stands < s["sinks"])[:, None]
    # q heads h * group + j share kv head h
    q = q.view(batch, query, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).view(batch, kv_heads, -1, query, longest)
    scores *= 1.0 / math.sqrt(dim)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(batch, kv_heads, -1, longest), v.permute(0, 2, 1, 3))
    out = out.view(batch, kv_heads, -1, query, dim) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, query, heads, dim)[sequence, index]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, query, heads)[sequence, index]
    return {"out": out.to(s["dtype"]), "lse": lse}


def _plain_accept(s):
    sequence, index = _rows_of(s)
    batch, n, width = s["q_offsets"].numel() - 1, s["max_query"], s["max_path"]
    first = s["q_offsets"][:-1].long()
    targets = s["logits"].float().argmax(-1)
    parent = s["parents"].long()
    # a node is reached if it is node 0, or its token is its parent's target, no earlier child's is, and its parent is
    # reached: with the edges that hold as a matrix, the ancestors of a node end at node 0
    match = (parent >= 0) & (s["tokens"].long() == targets[first[sequence] + parent.clamp(min=0)])
    place = sequence * n + parent.clamp(min=0)
    earliest = torch.full((batch * n,), n, dtype=torch.long, device="cuda")
    earliest.scatter_reduce_(0, place[match], index[match], "amin")
    match &= earliest[place] == index
    eye = torch.eye(n, device="cuda").expand(batch, n, n)
    step = eye.clone()
    step[sequence[match], index[match], parent[match]] = -1.0
    reached = torch.linalg.solve_triangular(step, eye, upper=False, unitriangular=True)  # along the edges that hold
    rank = reached.sum(-1).round().long() - 1                                # edges above a node
    on = reached[:, :, 0] > 0.5                                              # from node 0
    on &= rank < width
    path = torch.full((batch, width + 1), -1, dtype=torch.int32, device="cuda")
    nodes = torch.arange(n, dtype=torch.int32, device="cuda").expand(batch, n)
    path.scatter_(1, torch.where(on, rank, width), nodes)
    path = path[:, :width].contiguous()
    counts = on.sum(-1)
    last = path.gather(1, counts[:, None] - 1)[:, 0].long()
    return {"path": path, "counts": counts.to(torch.int32), "next": targets[first + last].to(torch.int32),
            "targets": targets.to(torch.int32)}


def _plain_keep(s):
    context = s["kv_lens"].long() - (s["q_offsets"][1:] - s["q_offsets"][:-1])
    page, width = s["k_pages"].shape[3], s["path"].shape[1]
    live = torch.arange(width, device="cuda") < s["counts"][:, None]
    sequence, place = live.nonzero(as_tuple=True)
    source, target = context[sequence] + s["path"][sequence, place], context[sequence] + place
    from_page, to_page = s["page_table"][sequence, source // page].long(), s["page_table"][sequence, target // page].long()
    s["k_pages"][:, to_page, :, target % page] = s["k_pages"][:, from_page, :, source % page]
    s["v_pages"][:, to_page, :, target % page] = s["v_pages"][:, from_page, :, source % page]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": (context + s["counts"]).to(torch.int32)}


def run(state):
    s = state
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "attention": _plain_attention, "accept": _plain_accept,
                "keep": _plain_keep}[s["op"]](s)
    from harsh4b_b200 import ops

    if s["op"] == "norm":
        x8, scales, _ = ops.rmsnorm_quantize_rows(s["x"], s["weight"], EPS, delta=s["delta"], out=s["out"])
        # the codes as the values that they stand for
        return {"x": s["x"] if s["delta"] is None else s["out"], "scales": scales,
                "values": torch.mul(x8, scales[:, None], out=s["values"])}
    if s["op"] == "append":
        q = ops.paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"],
                             heads=s["heads"], norm_q=s["norm_q"], norm_k=s["norm_k"], eps=EPS, rope_cos=s["cos"],
                             rope_sin=s["sin"], parents=s["parents"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["op"] == "attention":
        ops.paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"],
                                 s["parents"], max_query=s["max_query"], window=s["window"], sinks=s["sinks"],
                                 out=s["out"], lse=s["lse"], workspace=s["workspace"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["op"] == "accept":
        path, counts, following, targets = ops.accept_tree(s["tokens"], s["parents"], s["q_offsets"], s["logits"],
                                                           max_path=s["max_path"], workspace=s["workspace"])
        return {"path": path, "counts": counts, "next": following, "targets": targets}
    lengths = ops.keep_tokens(s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"], s["path"],
                              s["counts"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": lengths}


# ---- what they cannot do without, and their definitions ---------------------------------
def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        size, delta = (4 if t == "fp32" else 2 if t != "none" else 0 for t in (case["dtype"], case["delta"]))
        return {"bytes": n * (size + delta + (size if delta else 0) + 1) + 4 * case["width"] + 8 * case["rows"],
                "flops": 8 * n}
    parents, total = _trees(case)
    new = [len(p) for p in parents]
    rows = sum(new)
    if case["op"] == "accept":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": rows * case["vocab"] * size + 12 * rows + 12 * len(new), "flops": rows * case["vocab"]}
    dim = case["head_dim"]
    tables = 4 * sum(-(-t // case["page"]) for t in total) + 8 * len(new) + 4 * rows
    if case["op"] == "keep":
        moved = sum(n != i for path in _paths(case, parents) for i, n in enumerate(path))
        return {"bytes": 8 * moved * case["layers"] * case["kv_heads"] * dim + 12 * len(new), "flops": 0}
    if case["op"] == "append":
        wide = rows * (case["heads"] + 2 * case["kv_heads"]) * dim
        source = 4 if case["source"] == "fp32" else 2
        return {"bytes": wide * (source + 2) + 4 * rows + 12 * len(new), "flops": 8 * wide}
    pairs = keys = 0
    for p, t in zip(parents, total):
        context, depth = t - len(p), _depths(p)
        window = case["window"] or t + 1
        for d in depth:
            first = max(0, context + d - window + 1)
            held = min(first, context)
            pairs += context - held + min(case["sinks"], held) + min(d + 1, window)
        first = min(max(0, context - window + 1), context)
        keys += context - first + min(case["sinks"], first) + len(p)
    return {"bytes": 4 * rows * case["heads"] * dim + 4 * rows * case["heads"] + 4 * keys * case["kv_heads"] * dim + tables,
            "flops": 4 * dim * case["heads"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        if s["delta"] is not None:
            x += s["delta"].double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * s["weight"].double()
        scales = torch.maximum(y.abs().amax(-1), torch.full_like(y[:, 0], 1e-5)) / 127
        return {"x": x, "values": (y / scales[:, None]).round() * scales[:, None], "scales": scales}

    parents, total = _trees(case)
    offsets = s["q_offsets"].tolist()
    if case["op"] == "accept":
        targets = [int(row.double().argmax()) for row in s["logits"]]
        tokens = s["tokens"].tolist()
        paths, following = [], []
        for b, tree in enumerate(parents):
            path = [0]
            while len(path) < s["max_path"]:
                wanted = targets[offsets[b] + path[-1]]
                more = [i for i, p in enumerate(tree) if p == path[-1] and tokens[offsets[b] + i] == wanted]
                if not more:
                    break
                path.append(more[0])
            paths.append(path + [-1] * (s["max_path"] - len(path)))
            following.append(targets[offsets[b] + path[-1]])
        return {"path": torch.tensor(paths), "counts": torch.tensor([sum(i >= 0 for i in p) for p in paths]),
                "next": torch.tensor(following), "targets": torch.tensor(targets)}

    page, dim, kv_heads = case["page"], case["head_dim"], case["kv_heads"]
    table = s["page_table"].tolist()
    if case["op"] == "keep":
        if s["k_pages"].numel() > 1 << 30:
            return None
        paths = _paths(case, parents)
        pages = [s["k_pages"].double(), s["v_pages"].double()]
        for b, path in enumerate(paths):
            context = total[b] - len(parents[b])
            for i, n in enumerate(path):
                a, z = context + n, context + i
                for x in pages:
                    x[:, table[b][z // page], :, z % page] = x[:, table[b][a // page], :, a % page].clone()
        return {"k_pages": pages[0], "v_pages": pages[1],
                "lengths": torch.tensor([t - len(p) + len(path) for t, p, path in zip(total, parents, paths)])}

    group = case["heads"] // kv_heads
    if case["op"] == "append":
        x = s["qkv"].double().view(-1, case["heads"] + 2 * kv_heads, dim)
        q = torch.empty(x.shape[0], case["heads"], dim, dtype=torch.float64, device="cuda")
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        half = dim // 2

        def turned(rows_x, weight, positions):
            norm = rows_x / (rows_x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
            cos, sin = (s[name].double()[positions].unsqueeze(1) for name in ("cos", "sin"))
            out = torch.empty_like(norm)
            out[..., :half] = norm[..., :half] * cos - norm[..., half:] * sin
            out[..., half:] = norm[..., half:] * cos + norm[..., :half] * sin
            return out

        for b, tree in enumerate(parents):
            first, context = offsets[b], total[b] - len(tree)
            positions = torch.tensor([context + d for d in _depths(tree)], device="cuda")
            mine = x[first:first + len(tree)]
            q[first:first + len(tree)] = turned(mine[:, :case["heads"]], s["norm_q"], positions)
            k = turned(mine[:, case["heads"]:case["heads"] + kv_heads], s["norm_k"], positions)
            v = mine[:, case["heads"] + kv_heads:]
            i = 0
            while i < len(tree):  # page by page
                slot = (context + i) % page
                n = min(page - slot, len(tree) - i)
                held = table[b][(context + i) // page]
                k_pages[held, :, slot:slot + n] = k[i:i + n].transpose(0, 1)
                v_pages[held, :, slot:slot + n] = v[i:i + n].transpose(0, 1)
                i += n
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}

    out = torch.zeros(*s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, tree in enumerate(parents):
        first, n, context, depth = offsets[b], len(tree), total[b] - len(tree), _depths(tree)
        mine = [[False] * n for _ in range(n)]
        for i in range(n):
            j = i
            while j >= 0:
                mine[i][j] = True
                j = tree[j]
        at = torch.tensor([context + d for d in depth], device="cuda")
        where = torch.cat((torch.arange(context, device="cuda"), at))
        hidden = torch.cat((torch.zeros(n, context, dtype=torch.bool, device="cuda"), ~torch.tensor(mine, device="cuda")), 1)
        if case["window"]:
            hidden |= (where[None] <= at[:, None] - case["window"]) & (where[None] >= case["sinks"])
        held = torch.tensor(table[b][:-(-total[b] // page)], device="cuda")
        for h in range(kv_heads):
            k = s["k_pages"][held, h].reshape(-1, dim)[:total[b]].double()
            v = s["v_pages"][held, h].reshape(-1, dim)[:total[b]].double()
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][first:first + n, j].double() @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                lse[first:first + n, j] = torch.logsumexp(score, -1)
                out[first:first + n, j] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}
