"""The move of the accepted tokens where pages are missing."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from harsh4b_b200 import _lib, ops  # noqa: E402
from test_gpu_tree_steps import ints, kept, offsets_of  # noqa: E402


@pytest.mark.parametrize("layers,kv_heads,dim,page,dtype", [(1, 8, 128, 16, torch.float16), (3, 2, 64, 16, torch.bfloat16)])
def test_keep_without_a_page_leaves_its_sequence(layers, kv_heads, dim, page, dtype):
    """Nothing of a sequence moves where a page of its path is missing, whichever token needs it."""
    path = [0, 1, 5, 20, 33, 47]  # of 48 nodes from place 20 on: pages 1 (0 .. 5), 2, 3 and 4
    bases, count = [20, 20, 20], len(path)
    k = torch.randn(layers, 18, kv_heads, page, dim, device="cuda").to(dtype)
    v = torch.randn(layers, 18, kv_heads, page, dim, device="cuda").to(dtype)
    whole = torch.arange(18, dtype=torch.int32, device="cuda").view(3, 6)
    offsets, lens = offsets_of([[0] * 48] * 3), ints([68] * 3)
    paths = ints([path] * 3).view(3, count)
    for missing in (1, 2, 3, 4):
        for bad in (-1, 18, 1 << 30):
            table = whole.clone()
            table[1, missing] = bad
            ours_k, ours_v = k.clone(), v.clone()
            lengths = ops.keep_tokens(ours_k if layers > 1 else ours_k[0], ours_v if layers > 1 else ours_v[0], table, offsets,
                                      lens, paths, ints([count] * 3))
            assert _lib.device_status() == _lib.STATUS_BAD_PAGE
            assert lengths.tolist() == [20 + count, 68, 20 + count]
            held = whole.tolist()
            for got, was in ((ours_k, k), (ours_v, v)):
                assert torch.equal(got, kept(was, held, bases, [path, [], path], page))
    table = whole.clone()
    table[1, 0], table[1, 5] = -1, -1  # pages that no token of the path needs
    ours_k, ours_v = k.clone(), v.clone()
    lengths = ops.keep_tokens(ours_k if layers > 1 else ours_k[0], ours_v if layers > 1 else ours_v[0], table, offsets, lens,
                              paths, ints([count] * 3))
    assert _lib.device_status() == 0 and lengths.tolist() == [20 + count] * 3
    assert torch.equal(ours_k, kept(k, whole.tolist(), bases, [path] * 3, page))
