"""What the paged entry points refuse before any GPU work: shapes whose values
within a row or a page the kernels could not count in 32 bits. No device is
needed (without one a call that is not refused ends in a CUDA error)."""
import ctypes

import pytest

from harsh4b_b200 import _lib

pytest.importorskip("torch")

BIG = 1 << 31


@pytest.fixture(scope="module")
def library():
    if not _lib.LIBRARY.exists():
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load_library()


def batch(kv_heads=8, page_size=16, head_dim=128, tokens=0):
    """A batch without tokens: a call that accepts it has nothing to do."""
    at = ctypes.addressof(ctypes.create_string_buffer(64)) & ~63
    return _lib.PagedKvDesc(at or 64, at or 64, 64, 64, 64, 1, 1, page_size, kv_heads, head_dim, 1, 1, tokens)


def append(library, kv, heads):
    return library.h4b_paged_append(ctypes.byref(kv), 64, 0, BIG * 4, heads, None, None, 1e-6, None, None, 0, 64, BIG * 4,
                                    None)


def attention(library, kv, heads):
    return library.h4b_paged_attention(ctypes.byref(kv), 64, BIG * 4, heads, 0.1, 0, 0, 1, 64, BIG * 4, None, 64, 1 << 40,
                                       None)


@pytest.mark.parametrize("call", [append, attention])
@pytest.mark.parametrize("kv_heads,page_size,head_dim", [(16384, 1024, 128), (BIG // 1024, 16, 64), (BIG - 1, 1024, 128)])
def test_pages_past_32_bits_are_refused(library, call, kv_heads, page_size, head_dim):
    kv = batch(kv_heads, page_size, head_dim)
    assert call(library, kv, kv_heads) == _lib.H4B_EUNSUPPORTED


@pytest.mark.parametrize("heads,kv_heads", [(BIG // 128 - 16, 8), (BIG // 128, 1 << 20), (BIG - 8, 8)])
def test_rows_past_32_bits_are_refused(library, heads, kv_heads):
    assert append(library, batch(kv_heads), heads) == _lib.H4B_EUNSUPPORTED


def test_query_rows_past_32_bits_are_refused(library):
    assert attention(library, batch(600000), 32 * 600000) == _lib.H4B_EUNSUPPORTED


@pytest.mark.parametrize("call", [append, attention])
def test_large_shapes_that_fit_are_taken(library, call):
    assert call(library, batch(8191, 1024, 128), 8191) == 0
    assert call(library, batch(8), 256) == 0
