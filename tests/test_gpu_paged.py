"""The paged K/V cache operators against their definitions in 64 bits.

Attention tolerance, derived before the first run. With u the rounding unit of
the 16-bit type (2^-11 fp16, 2^-8 bf16) and A = softmax(S) |V|:
  * p is rounded once for the p v products:         u A
  * the result is rounded once:                     u |o|
  * S in fp32, |error| <= D 2^-24 scale sum|q k|, about 2^-14 for the inputs
    here; p, o and l in fp32, ex2 to 2^-22:         2^-13 A
  * an fp16 p = 2^(s - m + 8), m within 7 of the maximum, below 2^-14 is
    rounded absolutely, by 2^-25 (l >= 2):          n 2^-26 max|v|
and the sum times 1.1 for the second-order terms. The log-sum-exp carries the
error of S: 2e-4.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib, ops  # noqa: E402

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Batch:
    """A layer's pages and a ragged batch over them, with everything that no
    call may read set to NaN: free pages, page tails, freed pages' ids -1."""

    def __init__(self, new, total, *, heads, kv_heads, dim, page, dtype, window=0, sinks=0, seed=0, spare=3,
                 stale=float("nan"), keep_hidden=False):
        g = torch.Generator("cuda").manual_seed(seed)
        self.new, self.total, self.window, self.sinks = list(new), list(total), window, sinks
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        need = [-(-n // page) for n in total]
        pages = sum(need) + spare
        self.k_pages = torch.full((pages, kv_heads, page, dim), stale, dtype=dtype, device="cuda")
        self.v_pages = self.k_pages.clone()
        ids = torch.randperm(pages, generator=g, device="cuda")
        table = torch.full((len(new), max(need, default=0) + 2), -1, dtype=torch.int32)
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(total):
            k = torch.empty(n, kv_heads, dim, dtype=dtype, device="cuda").normal_(generator=g)
            v = torch.empty(n, kv_heads, dim, dtype=dtype, device="cuda").normal_(generator=g)
            self.k.append(k)
            self.v.append(v)
            first_seen = max(0, n - self.new[b] - window + 1) if window else 0
            for j in range(need[b]):
                low, high = j * page, min(n, (j + 1) * page)
                hidden = not keep_hidden and window and low >= sinks and high <= first_seen
                held = int(ids[at + j])
                if not hidden:  # a page that no row sees any more stays -1
                    table[b, j] = held
                    self.k_pages[held, :, :high - low] = k[low:high].transpose(0, 1)
                    self.v_pages[held, :, :high - low] = v[low:high].transpose(0, 1)
            at += need[b]
        self.table = table.cuda()
        self.offsets = torch.tensor([0] + self.new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        self.lens = torch.tensor(self.total, dtype=torch.int32, device="cuda").reshape(-1)
        self.rows = sum(self.new)
        self.q = torch.empty(self.rows, heads, dim, dtype=dtype, device="cuda").normal_(generator=g) * 1.5

    def call(self, q=None, **kwargs):
        kwargs.setdefault("lse", torch.full((self.rows, self.heads), 7.0, device="cuda"))
        out = ops.paged_attention(self.q if q is None else q, self.k_pages, self.v_pages, self.table, self.offsets,
                                  self.lens, window=self.window, sinks=self.sinks, **kwargs)
        return out, kwargs["lse"]

    def expected(self):
        """out, lse and the error bound of out, in 64 bits."""
        group = self.heads // self.kv_heads
        out = torch.zeros(self.rows, self.heads, self.dim, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        lse = torch.full((self.rows, self.heads), -math.inf, dtype=torch.float64, device="cuda")
        u, at = UNIT[self.dtype], 0
        for b, (n, total) in enumerate(zip(self.new, self.total)):
            if n == 0:
                continue
            p = torch.arange(total - n, total, device="cuda")[:, None]
            j = torch.arange(total, device="cuda")[None]
            seen = j <= p
            if self.window:
                seen &= (j > p - self.window) | (j < self.sinks)
            for h in range(self.heads):
                if total == 0:
                    break
                k, v = self.k[b][:, h // group].double(), self.v[b][:, h // group].double()
                s = (self.q[at:at + n, h].double() @ k.T / math.sqrt(self.dim)).masked_fill(~seen, -math.inf)
                some = seen.any(-1)
                lse[at:at + n, h] = torch.logsumexp(s, -1)
                w = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
                o, a = w @ v, w @ v.abs()
                out[at:at + n, h] = o
                bound[at:at + n, h] = 1.1 * (u * (a + o.abs()) + 2.0 ** -13 * a) + total * 2.0 ** -26 * v.abs().max()
            at += n
        return out, lse, bound

    def check(self, **kwargs):
        out, lse = self.call(**kwargs)
        want, want_lse, bound = self.expected()
        assert torch.isfinite(out).all()
        worst = ((out.double() - want).abs() - bound).max().item() if out.numel() else 0.0
        assert worst <= 0, f"out passes its bound by {worst}"
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert (out[empty] == 0).all()
        if (~empty).any():
            assert (lse.double() - want_lse)[~empty].abs().max().item() <= 2e-4
        assert _lib.device_status() == 0


SHAPES = [  # heads, kv_heads, dim, page, dtype
    (32, 8, 128, 16, torch.float16), (8, 2, 128, 64, torch.bfloat16), (6, 2, 64, 32, torch.float16),
    (5, 1, 128, 16, torch.bfloat16), (4, 4, 64, 128, torch.bfloat16), (16, 2, 128, 256, torch.float16),
    (24, 2, 64, 16, torch.bfloat16), (32, 1, 128, 32, torch.float16)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
def test_decode_lengths(heads, kv_heads, dim, page, dtype):
    total = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000, 1023, 2049]
    Batch([1] * len(total), total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
def test_ragged_chunks(heads, kv_heads, dim, page, dtype):
    new = [1, 0, 7, 33, 130, 64, 1, 0]
    total = [90, 50, 7, 200, 131, 64, 1, 0]
    Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seed=1).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 17), (128, 130), (5000, 3)])
def test_window_and_sinks(heads, kv_heads, dim, page, dtype, window, sinks):
    new, total = [1, 1, 40, 150, 3, 1], [700, 1, 400, 517, 100, 129]
    Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, window=window, sinks=sinks,
          seed=2).check()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES[:3])
@pytest.mark.parametrize("hint", [1, 2, 4, 40, 1000])
def test_every_kernel_answers_every_chunk(heads, kv_heads, dim, page, dtype, hint):
    """max_query picks the kernel only: too small or too large, the result stands."""
    new, total = [1, 5, 70, 300, 0], [260, 5, 513, 300, 9]
    Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seed=3).check(max_query=hint)


@pytest.mark.parametrize("hint", [1, 8, 64])
def test_rows_that_see_nothing(hint):
    """More new tokens than tokens: those before position 0 get zeros and -inf."""
    batch = Batch([1, 4, 90], [3, 4, 100], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    batch.total = [0, 2, 30]  # lengths that leave rows without a key
    batch.lens.copy_(torch.tensor(batch.total, dtype=torch.int32))
    batch.k = [k[:n] for k, n in zip(batch.k, batch.total)]
    batch.v = [v[:n] for v, n in zip(batch.v, batch.total)]
    batch.check(max_query=hint)


@pytest.mark.parametrize("hint", [1, 64])
def test_many_sequences(hint):
    """More sequences than threads, most of them short, and one long one among them."""
    total = [1 + (37 * i) % 90 for i in range(700)]
    total[311] = 9000
    Batch([1] * 700, total, heads=4, kv_heads=1, dim=128, page=16, dtype=torch.float16, seed=4).check(max_query=hint)


@pytest.mark.parametrize("new,total", [([1], [33000]), ([3], [20011]), ([64], [12345])])
def test_long_contexts_are_split(new, total):
    Batch(new, total, heads=8, kv_heads=2, dim=128, page=64, dtype=torch.bfloat16, seed=5).check()


def test_scores_far_apart():
    """Rising scores move the running maximum again and again."""
    batch = Batch([1, 80], [900, 700], heads=4, kv_heads=1, dim=128, page=16, dtype=torch.float16, seed=6)
    ramp = torch.linspace(0.1, 4.0, 900, device="cuda", dtype=torch.float32)
    for b in range(2):
        n = batch.total[b]
        direction = batch.q[-1, 0].float() / batch.q[-1, 0].float().norm()
        batch.k[b] = (batch.k[b].float() + 8 * ramp[:n, None, None] * direction).to(torch.float16)
        for j in range(n):
            held = int(batch.table[b, j // 16])
            batch.k_pages[held, :, j % 16] = batch.k[b][j]
    batch.check()


def test_strided_queries_and_outputs():
    batch = Batch([1, 40], [77, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16)
    wide = torch.randn(batch.rows, 12 * 128, device="cuda").to(torch.bfloat16)  # q of a fused q, k, v row
    wide[:, :1024] = batch.q.reshape(batch.rows, 1024)
    out = torch.zeros(batch.rows, 2, 8, 128, dtype=torch.bfloat16, device="cuda")
    plain, _ = batch.call()
    strided, _ = batch.call(q=wide[:, :1024].unflatten(1, (8, 128)), out=out[:, 1])
    assert torch.equal(strided, plain) and torch.equal(out[:, 1], plain)
    assert (out[:, 0] == 0).all()


def test_same_bits_every_time_and_workspace_left_ready():
    batch = Batch([1, 1, 200], [5000, 9001, 4000], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    workspace = ops.paged_workspace()
    first = [t.clone() for t in batch.call(workspace=workspace)]
    for _ in range(5):
        again = batch.call(workspace=workspace)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    few = Batch([1], [700], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    few.check(workspace=workspace)


def test_captured_graph_follows_the_tables():
    batch = Batch([1, 1], [400, 90], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    workspace = ops.paged_workspace()
    out, lse = batch.call(workspace=workspace, max_query=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        batch.call(workspace=workspace, max_query=1, out=out, lse=lse)
    other = Batch([1, 1], [17, 333], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16, seed=9)
    batch.lens.copy_(other.lens)
    batch.q.copy_(other.q)
    batch.table.fill_(-1)
    for b in range(2):  # the other batch's tokens in the pages that this one owns
        need = -(-other.total[b] // 16)
        held = torch.arange(b * 5, b * 5 + need, device="cuda", dtype=torch.int32)
        batch.table[b, :need] = held
        batch.k_pages[held.long()] = other.k_pages[other.table[b, :need].long()]
        batch.v_pages[held.long()] = other.v_pages[other.table[b, :need].long()]
    graph.replay()
    torch.cuda.synchronize()
    want, _, bound = other.expected()
    assert ((out.double() - want).abs() <= bound).all()


def test_captured_chunks():
    """Long chunks, some of them across CTAs, replay to the same bits (two launches a call)."""
    batch = Batch([300, 1, 64], [3000, 90, 9000], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16)
    workspace = ops.paged_workspace()
    want = [t.clone() for t in batch.call(workspace=workspace)]
    out, lse = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        batch.call(workspace=workspace, out=out, lse=lse)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES)
def test_few_long_chunks_among_many_short(heads, kv_heads, dim, page, dtype):
    """The short sequences of such a step go through a launch of their own; two
    to four new tokens are on either side of that bound."""
    new = [1] * 12 + [200] + [2, 3, 4] * 4 + [0, 90] + [1] * 6
    total = [17 * i + n for i, n in enumerate(new)]
    Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, window=150, sinks=5,
          seed=11).check()


def test_runs_on_the_current_stream():
    batch = Batch([1, 30], [500, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    want, _ = batch.call()
    q = batch.q.clone()
    batch.q.zero_()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        batch.q.copy_(q)
        got, _ = batch.call()
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("chunk", [1, 80])
def test_offsets_past_32_bits(chunk):
    """Pages whose values lie past 2^31 elements into the buffers."""
    pages = (1 << 31) // (8 * 64 * 128) + 40
    batch = Batch([chunk], [2000], heads=32, kv_heads=8, dim=128, page=64, dtype=torch.float16)
    k_pages = torch.empty(pages, 8, 64, 128, dtype=torch.float16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    held, used = batch.table[0, :32].long(), pages - 32 + torch.arange(32, device="cuda")
    k_pages[used], v_pages[used] = batch.k_pages[held], batch.v_pages[held]
    batch.table[0, :32] = used.to(torch.int32)
    batch.k_pages, batch.v_pages = k_pages, v_pages
    batch.check()


@pytest.mark.parametrize("chunk", [1, 80])
def test_bad_tables_are_reported_and_harmless(chunk):
    batch = Batch([chunk, chunk], [200, 300], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    good, _ = batch.call()
    batch.table[0, 3] = 1 << 20
    out, _ = batch.call()
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert torch.equal(out[chunk:], good[chunk:])
    batch.lens[0] = 1 << 28  # past its table: counts as empty
    out, lse = batch.call()
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert (out[:chunk] == 0).all() and (lse[:chunk] == -math.inf).all()
    assert torch.equal(out[chunk:], good[chunk:])


def test_refusals():
    batch = Batch([1], [40], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    args = (batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens)
    with pytest.raises(ValueError, match="q must be torch.float16"):
        ops.paged_attention(batch.q.float(), *args)
    with pytest.raises(ValueError, match="multiple of its kv heads"):
        ops.paged_attention(batch.q[:, :3], *args)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_attention(batch.q, *args, window=-1)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_attention(batch.q, *args, sinks=4)  # sinks without a window
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_attention(batch.q, *args, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.paged_attention(batch.q.cpu(), *args)
    with pytest.raises(ValueError, match="lse must be"):
        ops.paged_attention(batch.q, *args, lse=torch.zeros(1, 7, device="cuda"))
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        ops.paged_attention(batch.q, batch.k_pages.float(), batch.v_pages.float(), *args[2:])
    odd = torch.zeros(4, 2, 24, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="invalid argument"):  # 24 tokens a page
        ops.paged_attention(batch.q, odd, odd, *args[2:])
    thin = torch.zeros(4, 2, 16, 96, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="not supported"):
        ops.paged_attention(batch.q[..., :96].contiguous(), thin, thin, *args[2:])
    with pytest.raises(ValueError, match="page_table"):
        ops.paged_attention(batch.q, *args[:2], batch.table[:, 0], *args[3:])
    with pytest.raises(ValueError, match="as many page ids"):
        ops.copy_pages(*args[:2], batch.lens, batch.offsets)
    qkv = torch.zeros(1, 12 * 128, device="cuda")
    with pytest.raises(ValueError, match="qkv must be"):
        ops.paged_append(qkv, *args, heads=4)
    with pytest.raises(ValueError, match="qkv must be float32 or"):
        ops.paged_append(qkv.double(), *args, heads=8)
    with pytest.raises(ValueError, match="invalid argument"):
        ops.paged_append(qkv, *args, heads=8, norm_q=torch.ones(128, device="cuda"))


def test_empty_batches():
    batch = Batch([0, 0], [40, 3], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    batch.check()
    nobody = Batch([], [], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    nobody.check()
    for b in (batch, nobody):
        q = ops.paged_append(torch.zeros(0, 12 * 128, device="cuda"), b.k_pages, b.v_pages, b.table, b.offsets, b.lens, heads=8)
        assert q.shape == (0, 8, 128)


def test_another_keys_infinity_stays_out_of_the_scores():
    """An infinite k of a later token of the chunk is selected away in the rows that do not see it."""
    batch = Batch([40], [100], heads=4, kv_heads=1, dim=128, page=16, dtype=torch.float16, seed=8)
    want, _, bound = batch.expected()
    for hint in (1, 40):
        batch.k_pages[int(batch.table[0, 5]), :, 10:] = float("inf")  # tokens 90..95; row i stands at 60 + i
        batch.k_pages[int(batch.table[0, 6]), :, :4] = float("nan")   # 96..99
        out, lse = batch.call(max_query=hint)
        assert ((out.double() - want).abs() <= bound)[:30].all()
        assert torch.isfinite(lse[:30]).all()


# ---- append -----------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SHAPES[:6])
@pytest.mark.parametrize("source", ["fp32", "same"])
@pytest.mark.parametrize("turned", [True, False])
def test_append(heads, kv_heads, dim, page, dtype, source, turned):
    """fp32 arithmetic of a few operations (norm, two products and a sum), then
    one rounding: u |x| + 2^-19 (|cos| + |sin|) max|x|; untouched slots keep their bits."""
    batch = Batch([1, 0, 50, 3, 1], [9, 4, 130, 3, 64], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                  stale=5.0)
    g = torch.Generator("cuda").manual_seed(3)
    width = (heads + 2 * kv_heads) * dim
    wide = torch.empty(batch.rows, width + 64, device="cuda").normal_(generator=g) * 3
    wide = wide if source == "fp32" else wide.to(dtype)
    qkv = wide[:, :width]  # strided rows
    norm_q, norm_k = (1 + 0.1 * torch.empty(dim, device="cuda").normal_(generator=g) for _ in range(2))
    angles = torch.rand(256, dim // 2, generator=g, device="cuda") * 6
    cos, sin = angles.cos(), angles.sin()
    before = batch.k_pages.clone(), batch.v_pages.clone()
    extra = dict(norm_q=norm_q, norm_k=norm_k, eps=1e-5, rope_cos=cos, rope_sin=sin) if turned else {}
    q = ops.paged_append(qkv, batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens, heads=heads, **extra)
    x = qkv.double().view(batch.rows, heads + 2 * kv_heads, dim)
    position = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(batch.new, batch.total)])

    def expected(t, weight):
        if not turned:
            return t
        t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
        a, b = t.chunk(2, -1)
        c, s = cos.double()[position][:, None], sin.double()[position][:, None]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    def close(got, want):
        bound = UNIT[dtype] * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert ((got.double() - want).abs() <= bound).all()

    close(q, expected(x[:, :heads], norm_q))
    touched = torch.zeros(before[0].shape[0], page, dtype=torch.bool, device="cuda")
    at = 0
    for b, (n, t) in enumerate(zip(batch.new, batch.total)):
        p = torch.arange(t - n, t, device="cuda")
        where = batch.table[b, p // page].long(), p % page
        touched[where] = True
        close(batch.k_pages[where[0], :, where[1]], expected(x[:, heads:heads + kv_heads], norm_k)[at:at + n])
        close(batch.v_pages[where[0], :, where[1]], x[at:at + n, heads + kv_heads:])
        at += n
    keep = ~touched[:, None, :, None]
    assert torch.equal(batch.k_pages * keep, before[0] * keep) and torch.equal(batch.v_pages * keep, before[1] * keep)
    assert _lib.device_status() == 0


def test_append_many_tokens_and_sequences():
    """A long chunk (one CTA a token) among many sequences, against the same tokens fed one by one."""
    new, total = [1] * 90 + [1500] + [1] * 10, [5 + i for i in range(90)] + [1600] + [40] * 10
    batch = Batch(new, total, heads=4, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    qkv = torch.randn(batch.rows, 8 * 128, device="cuda")
    args = batch.k_pages, batch.v_pages, batch.table
    q = ops.paged_append(qkv, *args, batch.offsets, batch.lens, heads=4)
    assert torch.equal(q.view(batch.rows, -1), qkv[:, :512].half())
    held = batch.table[90, torch.arange(100, 1600, device="cuda") // 16].long()
    slot = torch.arange(100, 1600, device="cuda") % 16
    assert torch.equal(batch.k_pages[held, :, slot].reshape(1500, -1), qkv[90:1590, 512:768].half())
    assert torch.equal(batch.v_pages[held, :, slot].reshape(1500, -1), qkv[90:1590, 768:].half())


def test_append_bad_tables_are_reported_and_harmless():
    batch = Batch([1, 2], [20, 30], heads=4, kv_heads=2, dim=128, page=16, dtype=torch.float16, stale=5.0)
    before = batch.k_pages.clone()
    batch.table[0, 1] = -1
    qkv = torch.randn(3, 8 * 128, device="cuda")
    args = batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens
    ops.paged_append(qkv, *args, heads=4)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    changed = (batch.k_pages != before).any(-1).any(1).sum().item()
    assert changed == 2
    ones = torch.ones(8, 64, device="cuda")
    ops.paged_append(qkv, *args, heads=4, rope_cos=ones, rope_sin=ones)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE | _lib.STATUS_BAD_POSITION


# ---- page copies --------------------------------------------------------------------
@pytest.mark.parametrize("layers,kv_heads,page,dim,dtype", [
    (1, 1, 16, 64, torch.float16), (3, 8, 16, 128, torch.bfloat16), (2, 3, 256, 128, torch.float16),
    (36, 2, 32, 128, torch.float32)])
@pytest.mark.parametrize("moves", [0, 1, 7])
def test_copy_pages(layers, kv_heads, page, dim, dtype, moves):
    k = torch.randn(layers, 20, kv_heads, page, dim, device="cuda").to(dtype)
    v = torch.randn(layers, 20, kv_heads, page, dim, device="cuda").to(dtype)
    ids = torch.randperm(20, device="cuda").to(torch.int32)
    src, dst = ids[:moves].contiguous(), ids[moves:2 * moves].contiguous()
    want_k, want_v = k.clone(), v.clone()
    want_k[:, dst.long()], want_v[:, dst.long()] = k[:, src.long()], v[:, src.long()]
    ops.copy_pages(k, v, src, dst)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_copy_pages_skips_bad_ids():
    k = torch.randn(2, 6, 2, 16, 64, device="cuda").half()
    v = torch.randn_like(k)
    want_k, want_v = k.clone(), v.clone()
    want_k[:, 3], want_v[:, 3] = k[:, 1], v[:, 1]
    ops.copy_pages(k, v, torch.tensor([1, 6, 2], dtype=torch.int32, device="cuda"),
                   torch.tensor([3, 0, -1], dtype=torch.int32, device="cuda"))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
