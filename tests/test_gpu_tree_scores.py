"""Attention of drafted trees with scores at fp32's limits: rows of huge scores
beside others, and keys with an infinite value."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib  # noqa: E402
from test_gpu_tree import Trees, draft  # noqa: E402


# ---- rows of huge scores beside others ---------------------------------------------------
def mixed_scores(batch, first):
    """Head 0 scores all keys alike, `first` (exact in fp32); head 1 scores the first half of them 0 and the rest far
    above 2^20; heads 2 and 3 all 0. v is 1 in the first half and -1 in the rest, so a row's result shows the weights
    of the two halves against each other."""
    batch.q.zero_()
    batch.q[:, 0, 5], batch.q[:, 1, 7] = first, 4096.0
    for b, total in enumerate(batch.total):
        half = total // 2
        for j in range(total):
            k = torch.zeros_like(batch.k[b][j])
            k[:, 5] = 2048.0
            k[:, 7] = 0.0 if j < half else 16384.0
            v = torch.full_like(batch.v[b][j], 1.0 if j < half else -1.0)
            batch.k[b][j], batch.v[b][j] = k, v
            held = int(batch.table[b, j // batch.page])
            batch.k_pages[held, :, j % batch.page], batch.v_pages[held, :, j % batch.page] = k, v


def check_mixed_scores(batch, **kwargs):
    out, lse = batch.call(**kwargs)
    want, want_lse, bound = batch.expected()
    worst = ((out.double() - want).abs() - bound).amax(dim=(0, 2))
    assert (worst <= 0).all(), worst.tolist()
    # score, scale, base and sum are rounded once each
    assert ((lse.double() - want_lse).abs() <= 4 * 2.0 ** -24 * want_lse.abs() + 2e-4).all()
    assert _lib.device_status() == 0


# q of head 0 (of 8 bits each): its scores in base-2 units, times log2(e) / sqrt(dim), lie in 2^19 .. 2^20, where fp32's
# neighbours are 2^-4 apart, and are off by nearly half of that when they are rounded, the first downwards
FIRST = {128: [3584.0, 2560.0], 64: [1544.0, 2656.0]}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,total", [(2, 200), (8, 200), (8, 380), (40, 300), (40, 900), (8, 5000)])
def test_rows_beside_huge_ones(n, total, dim, dtype):
    """Whole items and items that are cut: the huge scores come into some of the parts only."""
    for first in FIRST[dim]:
        trees = Trees([draft(n, 3)], [total], heads=4, kv_heads=1, dim=dim, page=16, dtype=dtype)
        mixed_scores(trees, first)
        check_mixed_scores(trees)
        wide = torch.full((1, trees.table.shape[1] + 256), -1, dtype=torch.int32, device="cuda")
        wide[:, :trees.table.shape[1]] = trees.table
        trees.table = wide
        check_mixed_scores(trees)


# ---- infinite keys ------------------------------------------------------------------------
@pytest.mark.parametrize("n", [2, 4, 40])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_an_infinite_key_by_the_sign_of_its_scores(n, dim, value):
    """One dim of a key is infinite, so its score is by the sign of a row's value there: inf leaves nothing of a row but
    NaN, -inf leaves the row as if the key were not there. Rows that do not see it keep their bits."""
    for window in (0, 100):
        trees = Trees([draft(n, 3, roots=2), draft(n, 3, seed=1)], [300, 211], heads=8, kv_heads=2, dim=dim, page=16,
                      dtype=torch.float16, window=window, sinks=2 if window else 0)
        clean, clean_lse = [t.clone() for t in trees.call()]
        touched = torch.zeros(trees.rows, 8, dtype=torch.bool, device="cuda")
        up = touched.clone()
        for b, j in ((0, 300 - n + 1), (1, 211 - n - 99)):  # a node that some nodes see; at the windows' edges
            k = trees.k[b][j].clone()
            k[:, 9] = value
            trees.set_key(b, j, k=k)
            sees = trees.seen(b)[:, j]
            rows = slice(b * n, (b + 1) * n)
            touched[rows] |= sees[:, None]
            up[rows] |= sees[:, None] & (trees.q[rows, :, 9].float() * value > 0)
        out, lse = trees.call()
        want, want_lse, bound = trees.expected()
        assert touched.any() and up.any() and (touched & ~up).any() and not (touched & (trees.q[:, :, 9] == 0)).any()
        assert torch.equal(out[~touched], clean[~touched]) and torch.equal(lse[~touched], clean_lse[~touched])
        assert torch.isnan(out[up]).all() and not torch.isfinite(lse[up]).any()
        low = touched & ~up
        assert ((out.double() - want).abs() <= bound)[low].all()
        assert ((lse.double() - want_lse).abs() <= 2e-4)[low].all()
        assert _lib.device_status() == 0
