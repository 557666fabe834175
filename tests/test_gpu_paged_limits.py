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
