"""The paged K/V cache operators: what is measured, and their plain forms.

A serving process keeps the K/V of its sequences in pages of `page` tokens,
[pages][kv_heads][page][head_dim] per layer, and a table of page ids per
sequence. Four operators work on it:

append     norm and rotate the new tokens' q and k, write k and v into the pages
attention  of a ragged batch of new tokens (one to thousands a sequence) over
           the pages: causal, optionally with a sliding window and a few first
           tokens that stay visible
copy       pages to other pages in every layer: the private last page of a
           forked sequence, or the moves that compact the cache

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


def listed():
    attention = {"op": "attention", "dtype": "fp16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
                 "window": 0, "sinks": 0, "chunks": 0, "q": 1}
    append = {"op": "append", "dtype": "fp16", "source": "fp32", "heads": 32, "kv_heads": 8, "head_dim": 128,
              "page": 16, "chunks": 0, "q": 1}
    copy = {"op": "copy", "dtype": "fp16", "kv_heads": 8, "head_dim": 128}
    return [
        # one user's next token, about a thousand tokens in: the latency of one layer's attention
        dict(attention, name="decode one", sequences=1, kv_min=1000, kv_max=1000, lens=1),
        # a chat server's decode step: 64 sequences of every length up to two thousand
        dict(attention, name="decode ragged", sequences=64, kv_min=1, kv_max=2100, lens=2),
        # long documents, decoded 32 at a time: the whole cache is read
        dict(attention, name="decode long", sequences=32, kv_min=32768, kv_max=32768, page=64, lens=3),
        # streaming sessions far past their window, the first four tokens still visible
        dict(attention, name="decode window", dtype="bf16", sequences=48, kv_min=9000, kv_max=40000, page=32,
             window=4096, sinks=4, lens=4),
        # a long prompt in one pass, nothing cached before it
        dict(attention, name="prompt", sequences=1, chunks=1, q=8192, kv_min=8192, kv_max=8192, page=64, lens=5),
        # two prompts' next 500-odd tokens over a long cached history
        dict(attention, name="chunk on history", dtype="bf16", sequences=2, chunks=2, q=512, kv_min=15000,
             kv_max=16411, lens=6),
        # continuous batching: three prompts' chunks and 21 decoding sequences in one step, 3 q heads a kv head
        dict(attention, name="mixed step", dtype="bf16", heads=24, head_dim=64, sequences=24, chunks=3, q=255,
             kv_min=300, kv_max=4100, lens=7),
        # prompt chunks of a model whose layers see a window, with 16 first tokens kept
        dict(attention, name="chunk window", sequences=4, chunks=4, q=1024, kv_min=5000, kv_max=6500, page=64,
             window=1024, sinks=16, lens=8),
        # one layer's new q, k and v of a decode step, as the projection leaves them
        dict(append, name="append step", sequences=64, kv_min=1, kv_max=1000, lens=9),
        # the same for a long prompt
        dict(append, name="append prompt", sequences=1, chunks=1, q=8192, kv_min=8192, kv_max=8192, lens=10),
        # four forks of a sequence: each gets its own copy of the last, partly filled page
        dict(copy, name="fork", layers=36, page=16, pages=64, moves=4),
        # compaction after many sequences ended: 400 pages move to the front
        dict(copy, name="compact", layers=36, page=16, pages=900, moves=400),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "copy"))
    case = {"op": op, "dtype": rng.choice(("fp16", "bf16")), "kv_heads": rng.choice((1, 2, 4, 8)),
            "head_dim": rng.choice((64, 128, 128)), "page": rng.choice((16, 32, 64, 128))}
    if op == "copy":
        page_bytes = 2 * case["kv_heads"] * case["head_dim"] * case["page"] * 2
        layers = _log(rng, 1, 40)
        moves = _log(rng, 1, max(1, min(2000, (900 << 20) // (page_bytes * layers))))
        return dict(case, layers=layers, moves=moves, pages=2 * moves + rng.randrange(1, 50))
    case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 5, 8))
    kind = rng.choice(("decode", "chunk", "mixed"))
    if kind == "decode":
        chunks, q = 0, 1
        sequences = _log(rng, 1, 128)
        kv_max = _log(rng, 1, min(MAX_POSITION, (32 << 15) // sequences))
    else:
        q = _log(rng, 2, 4096)
        chunks = _log(rng, 1, max(1, 8192 // q))
        sequences = chunks if kind == "chunk" else chunks + _log(rng, 1, 32)
        # the padded scores of the plain form: sequences x heads x q x kv, at most 1 G values
        most = (1 << 30) // (sequences * case["heads"] * q)
        if most < q:
            chunks = sequences = 1
            q = min(q, int(math.sqrt((1 << 30) // case["heads"])))
            most = (1 << 30) // (case["heads"] * q)
        kv_max = max(q, _log(rng, q, max(q, min(MAX_POSITION, most))))
    kv_min = kv_max if rng.random() < 0.3 else rng.randrange(1, kv_max + 1)
    case.update(sequences=sequences, chunks=chunks, q=q, kv_min=kv_min, kv_max=kv_max, lens=rng.randrange(1 << 20))
    if op == "append":
        return dict(case, source=rng.choice(("fp32", case["dtype"])))
    windowed = rng.random() < 0.4
    return dict(case, window=_log(rng, 1, 8192) if windowed else 0, sinks=rng.choice((0, 1, 4, 16, 130)) if windowed else 0)


def _lengths(case):
    """(new tokens, tokens in all) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["lens"])
    new, total = [], []
    for i in range(case["sequences"]):
        n = (case["q"] if i == 0 else rng.randint((case["q"] + 1) // 2, case["q"])) if i < case["chunks"] else 1
        new.append(n)
        total.append(max(n, rng.randint(case["kv_min"], case["kv_max"])))
    return new, total


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        return out.normal_(generator=g)

    heads_dim = (case["kv_heads"], case["page"], case["head_dim"])
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], *heads_dim)
        ids = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        return {"op": "copy", "k_pages": normal(*shape), "v_pages": normal(*shape), "src": ids[:case["moves"]].clone(),
                "dst": ids[case["moves"]:2 * case["moves"]].clone()}

    new, total = _lengths(case)
    page, rows = case["page"], sum(new)
    need = [-(-n // page) for n in total]
    pages = sum(need) + 7  # a few free ones
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    counts = torch.tensor(need, device="cuda")
    held = torch.arange(table.shape[1], device="cuda")[None] < counts[:, None]
    table[held] = ids[:sum(need)]
    offsets = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    state = {"op": case["op"], "dtype": dtype, "k_pages": normal(pages, *heads_dim), "v_pages": normal(pages, *heads_dim),
             "page_table": table, "q_offsets": offsets,
             "kv_lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "max_query": max(new),
             "max_kv": max(total), "heads": case["heads"]}
    dim = case["head_dim"]
    if case["op"] == "append":
        source = DTYPES[case["source"]]
        state["qkv"] = normal(rows, (case["heads"] + 2 * case["kv_heads"]) * dim, dtype=source) * 3
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


def _token_rows(s):
    """Of every new token: its sequence and its position."""
    offsets = s["q_offsets"].long()
    new = offsets[1:] - offsets[:-1]
    sequence = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=s["rows"])
    index = torch.arange(s["rows"], device="cuda") - offsets[sequence]
    return sequence, index, s["kv_lens"].long()[sequence] - new[sequence] + index


def _plain_append(s):
    heads, kv_heads, dim = s["heads"], s["k_pages"].shape[1], s["k_pages"].shape[3]
    s = dict(s, rows=s["qkv"].shape[0])
    sequence, _, position = _token_rows(s)
    x = s["qkv"].float().view(s["rows"], heads + 2 * kv_heads, dim)
    q, k, v = x.split((heads, kv_heads, kv_heads), dim=1)

    def turned(t, weight):
        t = t * (1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)) * weight
        a, b = t.chunk(2, dim=-1)
        cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)

    page = s["k_pages"].shape[2]
    where = s["page_table"][sequence, position // page].long(), position % page
    s["k_pages"][where[0], :, where[1]] = turned(k, s["norm_k"]).to(s["dtype"])
    s["v_pages"][where[0], :, where[1]] = v.to(s["dtype"])
    return {"q": turned(q, s["norm_q"]).to(s["dtype"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    rows, heads, dim = s["q"].shape
    kv_heads, page = s["k_pages"].shape[1:3]
    s = dict(s, rows=rows)
    sequence, index, position = _token_rows(s)
    batch, longest, query = s["kv_lens"].numel(), s["max_kv"], s["max_query"]
    keys = torch.arange(longest, device="cuda")
    held = s["page_table"][:, keys // page].long().clamp(min=0)            # [batch, longest]
    k = s["k_pages"][held, :, keys % page].float()                          # [batch, longest, kv_heads, dim]
    v = s["v_pages"][held, :, keys % page].float()
    v = v.masked_fill_((keys[None] >= s["kv_lens"][:, None])[:, :, None, None], 0.0)
    q = torch.zeros(batch, query, heads, dim, dtype=torch.float32, device="cuda")
    q[sequence, index] = s["q"].float()
    at = torch.full((batch, query), -1, dtype=torch.long, device="cuda")
    at[sequence, index] = position
    # q heads h * group + j share kv head h
    q = q.view(batch, query, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).view(batch, kv_heads, -1, query, longest)
    scores *= 1.0 / math.sqrt(dim)
    seen = keys <= at[:, :, None]
    if s["window"]:
        seen &= (keys > at[:, :, None] - s["window"]) | (keys < s["sinks"])
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


def _plain_copy(s):
    s["k_pages"][:, s["dst"].long()] = s["k_pages"][:, s["src"].long()]
    s["v_pages"][:, s["dst"].long()] = s["v_pages"][:, s["src"].long()]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "copy": _plain_copy}[s["op"]](s)
    from harsh4b_b200 import ops

    if s["op"] == "append":
        q = ops.paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"],
                             heads=s["heads"], norm_q=s["norm_q"], norm_k=s["norm_k"], eps=EPS, rope_cos=s["cos"],
                             rope_sin=s["sin"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["op"] == "attention":
        ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"],
                            max_query=s["max_query"], window=s["window"], sinks=s["sinks"], out=s["out"],
                            lse=s["lse"], workspace=s["workspace"])
        return {"out": s["out"], "lse": s["lse"]}
    ops.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _seen(case, n, total):
    """(pairs of a new token and a key that it sees, keys that some new token sees) of one sequence."""
    window, sinks = case["window"] or total, case["sinks"]
    pairs = 0
    for p in range(total - n, total):
        first = max(0, p - window + 1)
        pairs += p + 1 - first + min(sinks, first)
    first = max(0, total - n - window + 1)
    return pairs, total - first + min(sinks, first)


def work(case):
    if case["op"] == "copy":
        page = case["kv_heads"] * case["page"] * case["head_dim"] * 2
        return {"bytes": 4 * case["moves"] * case["layers"] * page + 8 * case["moves"], "flops": 0}
    new, total = _lengths(case)
    rows, dim = sum(new), case["head_dim"]
    tables = 4 * sum(-(-t // case["page"]) for t in total) + 8 * len(new)
    if case["op"] == "append":
        wide = rows * (case["heads"] + 2 * case["kv_heads"]) * dim
        source = 4 if case["source"] == "fp32" else 2
        # tables: a cos and a sin row of every position that occurs, and one page id of every new token's page
        return {"bytes": wide * (source + 2) + rows * 4 * dim + 8 * len(new) + 4 * sum(-(-n // case["page"]) for n in new),
                "flops": 8 * wide}
    seen = [_seen(case, n, t) for n, t in zip(new, total)]
    keys = sum(k for _, k in seen)
    return {"bytes": 4 * rows * case["heads"] * dim + 4 * rows * case["heads"] + 4 * keys * case["kv_heads"] * dim + tables,
            "flops": 4 * dim * case["heads"] * sum(p for p, _ in seen)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        if s["k_pages"].numel() > 1 << 28:
            return None
        k, v = s["k_pages"].double(), s["v_pages"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = k[:, a].clone(), v[:, a].clone()
        return {"k_pages": k, "v_pages": v}

    offsets, totals, table = s["q_offsets"].tolist(), s["kv_lens"].tolist(), s["page_table"].tolist()
    page, dim, kv_heads = case["page"], case["head_dim"], case["kv_heads"]
    group = case["heads"] // kv_heads
    if case["op"] == "append":
        rows = s["qkv"].shape[0]
        x = s["qkv"].double().view(rows, case["heads"] + 2 * kv_heads, dim)
        q = torch.empty(rows, case["heads"], dim, dtype=torch.float64, device="cuda")
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        half = dim // 2

        def turned(rows_x, weight, positions):
            norm = rows_x / (rows_x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
            cos, sin = (s[name].double()[positions].unsqueeze(1) for name in ("cos", "sin"))
            out = torch.empty_like(norm)
            out[..., :half] = norm[..., :half] * cos - norm[..., half:] * sin
            out[..., half:] = norm[..., half:] * cos + norm[..., :half] * sin
            return out

        for b, total in enumerate(totals):
            first, last = offsets[b], offsets[b + 1]
            positions = torch.arange(total - (last - first), total, device="cuda")
            q[first:last] = turned(x[first:last, :case["heads"]], s["norm_q"], positions)
            k = turned(x[first:last, case["heads"]:case["heads"] + kv_heads], s["norm_k"], positions)
            v = x[first:last, case["heads"] + kv_heads:]
            start, i = total - (last - first), 0
            while i < last - first:  # page by page
                slot = (start + i) % page
                n = min(page - slot, last - first - i)
                held = table[b][(start + i) // page]
                k_pages[held, :, slot:slot + n] = k[i:i + n].transpose(0, 1)
                v_pages[held, :, slot:slot + n] = v[i:i + n].transpose(0, 1)
                i += n
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}

    out = torch.zeros(*s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, total in enumerate(totals):
        first, last = offsets[b], offsets[b + 1]
        held = torch.tensor(table[b][:-(-total // page)], device="cuda")
        for h in range(kv_heads):
            k = s["k_pages"][held, h].reshape(-1, dim)[:total].double()
            v = s["v_pages"][held, h].reshape(-1, dim)[:total].double()
            for j in range(h * group, (h + 1) * group):
                for low in range(first, last, 4096):
                    high = min(last, low + 4096)
                    at = torch.arange(total - last + low, total - last + high, device="cuda")[:, None]
                    key = torch.arange(total, device="cuda")[None]
                    hidden = key > at
                    if case["window"]:
                        hidden |= (key <= at - case["window"]) & (key >= case["sinks"])
                    score = (s["q"][low:high, j].double() @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                    lse[low:high, j] = torch.logsumexp(score, -1)
                    out[low:high, j] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}
