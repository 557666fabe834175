"""The attentions' workspace: one for both, in turn, or the plain one's alone."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib, ops  # noqa: E402
from test_gpu_paged import Batch  # noqa: E402
from test_gpu_tree import Trees, draft  # noqa: E402


def test_the_plain_attention_takes_its_smaller_workspace():
    """Trees keep twice the items' records of the plain attention, which needs none of that room."""
    new, total = [1, 3, 60, 130], [700, 65, 500, 130]
    batch = Batch(new, total, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    trees = Trees([draft(20, 3)], [900], heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16)
    full = ops.paged_workspace(128)
    small = torch.zeros(full.numel() - 4096, dtype=torch.uint8, device="cuda")
    want, want_tree = batch.call(workspace=full)[0], trees.call(workspace=full)[0]
    for hint in (1, 1000):
        assert torch.equal(batch.call(workspace=small, max_query=hint)[0], batch.call(workspace=full, max_query=hint)[0])
    with pytest.raises(ValueError, match="invalid argument"):
        batch.call(workspace=small[:-16])
    with pytest.raises(ValueError, match="invalid argument"):
        trees.call(workspace=small)
    for _ in range(2):  # one workspace for both, in turn
        assert torch.equal(batch.call(workspace=full)[0], want) and torch.equal(trees.call(workspace=full)[0], want_tree)
    assert _lib.device_status() == 0
