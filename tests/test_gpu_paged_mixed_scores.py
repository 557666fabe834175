"""Paged attention where some rows' scores are huge and others' are not: every
row's weights are formed in one way."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_paged import Batch  # noqa: E402
from test_gpu_tree_scores import FIRST, check_mixed_scores, mixed_scores  # noqa: E402


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,total", [([1], [400]), ([8], [700]), ([60], [900]), ([130], [700]), ([40], [6000])])
def test_rows_beside_huge_ones(new, total, dim, hint):
    for first in FIRST[dim]:
        batch = Batch(new, total, heads=4, kv_heads=1, dim=dim, page=16, dtype=torch.float16)
        mixed_scores(batch, first)
        check_mixed_scores(batch, max_query=hint)
