"""The paged operators at their limits: what test_gpu_paged.py's batches do not
reach, with its definitions in 64 bits and its tolerance."""
import copy
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_paged import Batch  # noqa: E402

from harsh4b_b200 import _lib, ops  # noqa: E402

FORMS = [([1, 1, 1], [700, 64, 1]), ([200, 1, 40], [300, 90, 513])]  # few rows, long chunks


# ---- the scale of the scores ------------------------------------------------------
@pytest.mark.parametrize("new,total", FORMS)
@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.bfloat16)])
@pytest.mark.parametrize("scale", [1e-30, 0.01, 0.2])
def test_scale(new, total, dim, dtype, scale):
    """Scores of another scale: the error of S, and with it the bound, grows by
    its ratio to 1 / sqrt(D) where that is above one."""
    batch = Batch(new, total, heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype, window=150, sinks=3, seed=21)
    ratio = scale * math.sqrt(dim)
    as_default = copy.copy(batch)
    as_default.q = batch.q.double() * ratio
    out, lse = batch.call(scale=scale)
    want, want_lse, bound = as_default.expected()
    assert ((out.double() - want).abs() <= max(1.0, ratio) * bound).all()
    assert (lse.double() - want_lse).abs().max().item() <= 2e-4 * max(1.0, ratio)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("new,total", FORMS)
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, math.nan, math.inf, -math.inf, 1e-46, 3e38])
def test_scales_that_are_refused(new, total, scale):
    """A scale that is not positive, or neither it nor its base-2 form a finite fp32."""
    batch = Batch(new, total, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    with pytest.raises(ValueError, match="scale|invalid argument"):
        batch.call(scale=scale)


# ---- devices ----------------------------------------------------------------------
def test_tensors_of_another_device_are_refused(monkeypatch):
    batch = Batch([1], [40], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    workspace, ids = ops.paged_workspace(), torch.zeros(1, dtype=torch.int32, device="cuda")
    args = batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: ops.paged_attention(batch.q, *args, workspace=workspace),
                 lambda: ops.paged_append(torch.zeros(1, 12 * 128, device="cuda:0"), *args, heads=8),
                 lambda: ops.copy_pages(*args[:2], ids, ids + 1)):
        with pytest.raises(ValueError, match="current device, cuda:1"):
            call()


# ---- append: values that are not rotated ---------------------------------------------
@pytest.mark.parametrize("source", ["fp32", "same"])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("past", [False, True])
def test_unrotated_values_do_not_meet_their_partners(source, normed, past):
    """Without a rotation (none asked for, or a position past its rows) dim d's
    value is its own: an infinity or NaN in dim d + D / 2 does not reach it."""
    batch = Batch([3, 1], [40, 9], heads=4, kv_heads=2, dim=128, page=16, dtype=torch.float16, stale=5.0)
    qkv = torch.randn(4, 8, 128, device="cuda")
    qkv[0, 0, 70] = qkv[1, 4, 3] = math.inf
    qkv[2, 5, 127], qkv[3, 1, 64] = math.nan, -math.inf
    qkv[3, 7, 10] = math.nan  # a v head
    qkv = qkv if source == "fp32" else qkv.half()
    extra, want = {}, qkv.double()
    if normed:
        ones = torch.ones(128, device="cuda")
        extra.update(norm_q=ones, norm_k=ones)
        want[:, :6] = want[:, :6] / (want[:, :6].pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    if past:
        extra.update(rope_cos=torch.zeros(8, 64, device="cuda"), rope_sin=torch.ones(8, 64, device="cuda"))
    q = ops.paged_append(qkv.view(4, -1), batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens, heads=4,
                         **extra)
    position, row = torch.tensor([37, 38, 39, 8], device="cuda"), torch.tensor([0, 0, 0, 1], device="cuda")
    held, slot = batch.table[row, position // 16].long(), position % 16
    got = torch.cat([q, batch.k_pages[held, :, slot], batch.v_pages[held, :, slot]], 1).double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~finite].nan_to_num(7.0), want[~finite].nan_to_num(7.0))
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -18 * 4)[finite].all()
    assert _lib.device_status() == (_lib.STATUS_BAD_POSITION if past else 0)


# ---- integers past 32 bits --------------------------------------------------------------
@pytest.mark.parametrize("name", ["window", "sinks", "max_query"])
@pytest.mark.parametrize("value", [1 << 31, (1 << 32) + 1, (1 << 32) + 16, -(1 << 32) + 1, 1 << 70])
def test_integers_past_32_bits_are_refused(name, value):
    batch = Batch([1], [40], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    options = {"window": 8, "sinks": 1, "max_query": 1, name: value}
    batch.window, batch.sinks = options["window"], options["sinks"]
    with pytest.raises(ValueError, match="32 bits|invalid argument"):
        batch.call(max_query=options["max_query"])


# ---- append: long chunks, two warps a token, several passes over the heads --------------
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(32, 8, 128, torch.float16), (24, 8, 64, torch.bfloat16),
                                                      (40, 1, 128, torch.bfloat16), (3, 1, 128, torch.float16)])
@pytest.mark.parametrize("source", ["fp32", "same"])
def test_append_long_chunks(heads, kv_heads, dim, dtype, source):
    """1024 tokens and more, with norms and rotation. The bound is that of
    test_gpu_paged.py's append: one rounding of a few fp32 operations."""
    new, total = [1, 1030, 0, 200, 1], [40, 1100, 7, 200, 1]
    batch = Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=32, dtype=dtype, stale=5.0)
    g = torch.Generator("cuda").manual_seed(5)
    qkv = torch.empty(batch.rows, (heads + 2 * kv_heads) * dim, device="cuda").normal_(generator=g) * 3
    qkv = qkv if source == "fp32" else qkv.to(dtype)
    norm_q, norm_k = (1 + 0.1 * torch.empty(dim, device="cuda").normal_(generator=g) for _ in range(2))
    angles = torch.rand(1100, dim // 2, generator=g, device="cuda") * 6
    cos, sin = angles.cos(), angles.sin()
    q = ops.paged_append(qkv, batch.k_pages, batch.v_pages, batch.table, batch.offsets, batch.lens, heads=heads,
                         norm_q=norm_q, norm_k=norm_k, eps=1e-5, rope_cos=cos, rope_sin=sin)
    x = qkv.double().view(batch.rows, heads + 2 * kv_heads, dim)
    position = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(new, total)])
    row = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))

    def turned(t, weight):
        t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
        a, b = t.chunk(2, -1)
        c, s = cos.double()[position][:, None], sin.double()[position][:, None]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    held, slot = batch.table[row, position // 32].long(), position % 32
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for got, want in ((q, turned(x[:, :heads], norm_q)),
                      (batch.k_pages[held, :, slot], turned(x[:, heads:heads + kv_heads], norm_k)),
                      (batch.v_pages[held, :, slot], x[:, heads + kv_heads:])):
        bound = unit * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert ((got.double() - want).abs() <= bound).all()
    assert _lib.device_status() == 0


# ---- values that are not finite reach the rows that see them, and no others --------------
SPECIAL = [math.inf, -math.inf, math.nan]


def check_reach(new, total, hint, *, heads, kv_heads, dim, page, dtype, window=0, sinks=0, seed=0):
    """v values that are not finite in every seventh key or so: a row's dims
    are finite where no key that it sees has one there, and within the bound."""
    batch = Batch(new, total, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, window=window, sinks=sinks,
                  seed=seed)
    clean, _, bound = batch.expected()
    g = torch.Generator().manual_seed(seed)
    reached = torch.zeros(batch.rows, heads, dim, dtype=torch.bool, device="cuda")
    group, at, wild = heads // kv_heads, 0, 0
    for b, (n, t) in enumerate(zip(new, total)):
        p = torch.arange(t - n, t, device="cuda")
        # mostly where the chunk's rows see different keys: its own tokens, the window's edge; a few elsewhere
        keys = [j for j in range(max(0, t - n), t, 5)] + [j for j in range(max(0, t - n - window), max(0, t - window), 3)]
        for j in set(keys) if window else set(keys[:len(keys) // 2]):
            held = int(batch.table[b, j // page])
            if held < 0:
                continue
            h, d = int(torch.randint(kv_heads, (1,), generator=g)), int(torch.randint(dim, (1,), generator=g))
            batch.v_pages[held, h, j % page, d] = SPECIAL[wild % 3]
            wild += 1
            seen = j <= p
            if window:
                seen &= (j > p - window) | (j < sinks)
            reached[at:at + n, h * group:(h + 1) * group, d] |= seen[:, None]
        at += n
    out, lse = batch.call(max_query=hint)
    assert torch.equal(torch.isfinite(out), ~reached)
    assert ((out.double() - clean).abs() <= bound)[~reached].all()
    assert torch.isfinite(lse).all() and wild > 0 and reached.any()
    assert _lib.device_status() == 0


REACH = [dict(heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16),
         dict(heads=6, kv_heads=2, dim=64, page=64, dtype=torch.bfloat16),
         dict(heads=5, kv_heads=1, dim=128, page=256, dtype=torch.bfloat16),
         dict(heads=32, kv_heads=1, dim=64, page=16, dtype=torch.float16)]


@pytest.mark.parametrize("shape", REACH)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5), (3, 0)])
def test_values_reach_the_rows_that_see_them_few_rows(shape, window, sinks):
    check_reach([4, 2, 7, 3], [200, 2, 70, 129], 1, window=window, sinks=sinks, seed=1, **shape)
    check_reach([3], [5000], 1, window=window, sinks=sinks, seed=2, **shape)


@pytest.mark.parametrize("shape", REACH)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5), (300, 130), (3, 0)])
def test_values_reach_the_rows_that_see_them_long_chunks(shape, window, sinks):
    check_reach([150, 2, 64, 300], [200, 2, 70, 900], 1000, window=window, sinks=sinks, seed=1, **shape)
    check_reach([90], [6000], 1000, window=window, sinks=sinks, seed=2, **shape)  # items across CTAs


def test_values_reach_the_rows_that_see_them_mixed_step():
    """Chunks and decoded tokens in one step, each kernel with its share of them."""
    check_reach([1] * 20 + [200, 90], [50 + i for i in range(20)] + [500, 90], 200, window=60, sinks=3, seed=3, **REACH[0])


def test_an_item_after_such_values_is_as_before():
    """Where one sequence's v values are not finite, the others keep their bits."""
    batch = Batch([200] * 8, [1000] * 8, heads=32, kv_heads=8, dim=128, page=16, dtype=torch.float16, seed=4)
    want, want_lse = batch.call()
    batch.v_pages[int(batch.table[2, 60]), :, 3, ::7] = math.nan  # token 963 of sequence 2: rows from 163 on
    out, lse = batch.call()
    same = torch.ones(batch.rows, dtype=torch.bool, device="cuda")
    same[2 * 200 + 163:3 * 200] = False
    assert torch.equal(out[same], want[same]) and torch.equal(lse, want_lse)
    assert torch.isnan(out[~same][..., ::7]).all()
    rest = torch.arange(128, device="cuda") % 7 != 0
    assert torch.equal(out[~same][..., rest], want[~same][..., rest])


# ---- steps of few long chunks among many short sequences: one launch or two -------------
@pytest.mark.parametrize("sequences", [19, 20, 39, 40, 70])
@pytest.mark.parametrize("shape", REACH + [dict(heads=32, kv_heads=8, dim=128, page=16, dtype=torch.bfloat16)])
def test_mixed_steps_on_both_sides_of_the_rule(sequences, shape):
    new = [1] * 6 + [130] + [2] * 3 + [0, 70] + [1] * (sequences - 12)
    total = [n + (37 * i) % 400 for i, n in enumerate(new)]
    Batch(new, total, window=150, sinks=5, seed=13, **shape).check()
    assert check_reach(new, total, None, window=150, sinks=5, seed=13, **shape) is None


# ---- scores far past fp32's fractions ----------------------------------------------------
@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("dim,dtype,power", [(128, torch.float16, 8), (128, torch.float16, 12), (64, torch.float16, 13),
                                             (128, torch.float16, 14), (64, torch.float16, 15), (128, torch.bfloat16, 12),
                                             (128, torch.bfloat16, 16), (64, torch.bfloat16, 20), (128, torch.bfloat16, 60)])
@pytest.mark.parametrize("below", [False, True])
def test_huge_scores(hint, dim, dtype, power, below):
    """q and k of one dim each, of few bits: their products are exact in fp32
    and equal scores stay equal, so the weights are known whatever their size."""
    new, total = [1, 3, 60, 130], [700, 65, 500, 130]
    batch = Batch(new, total, heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype, seed=31)
    batch.q.zero_()
    batch.q[:, :, 5] = 1.375 * 2.0 ** power
    g = torch.Generator().manual_seed(power)
    for b, t in enumerate(total):
        k = torch.zeros_like(batch.k[b])
        # rising by factors of two along the sequence, each with many equal and some opposite ones
        size = torch.arange(t, device="cuda").float().mul(4.0 / t).floor() - 3
        sign = torch.randint(-1, 2, (t,), generator=g).float().cuda()
        sign[0] = 1
        if below:  # none but hugely negative ones
            sign = -torch.ones_like(sign)
        k[:, :, 5] = (sign * 1.625 * torch.exp2(size + power))[:, None].to(dtype)
        batch.k[b] = k
        for j in range(t):
            batch.k_pages[int(batch.table[b, j // 16]), :, j % 16] = k[j]
    out, lse = batch.call(max_query=hint)
    want, want_lse, bound = batch.expected()
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= bound).all()
    # a score's own rounding, and the product with the scale's
    assert ((lse.double() - want_lse).abs() <= 2e-4 + 2.0 ** -22 * want_lse.abs()).all()
    assert _lib.device_status() == 0
