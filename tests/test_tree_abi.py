"""What the entry points of drafted token trees refuse before any GPU work. No
device is needed (without one a call that is not refused ends in a CUDA error)."""
import ctypes

import pytest

from harsh4b_b200 import _lib

pytest.importorskip("torch")

BIG = 1 << 31
EINVAL, EUNSUPPORTED = _lib.H4B_EINVAL, _lib.H4B_EUNSUPPORTED


@pytest.fixture(scope="module")
def library():
    if not _lib.LIBRARY.exists():
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load_library()


def batch(tokens=4, sequences=1, kv_heads=8, page_size=16, head_dim=128, dtype=1):
    """Tables and pages at made-up addresses: none is read by a call that is refused."""
    return _lib.PagedKvDesc(1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24, dtype, 4, page_size, kv_heads, head_dim, sequences, 1,
                            tokens)


def append(library, kv, parents=64, heads=8):
    return library.h4b_paged_append_tree(ctypes.byref(kv), parents, 64, 0, 1 << 20, heads, None, None, 1e-6, None, None, 0, 64,
                                         1 << 20, None)


def attention(library, kv, parents=64, heads=8, max_query=4, window=0, sinks=0, scale=0.1, stride=1 << 20):
    return library.h4b_paged_tree_attention(ctypes.byref(kv), parents, 64, stride, heads, scale, window, sinks, max_query, 64,
                                            stride, None, 64, 1 << 40, None)


def test_trees_without_parents_are_refused(library):
    assert append(library, batch(), parents=None) == EINVAL
    assert attention(library, batch(), parents=None) == EINVAL


def test_batches_without_nodes_have_nothing_to_do(library):
    for kv in (batch(tokens=0), batch(sequences=0)):
        assert append(library, kv) == 0 and attention(library, kv) == 0
    assert append(library, batch(tokens=0), parents=None) == 0


@pytest.mark.parametrize("change", [dict(max_query=0), dict(window=-1), dict(sinks=3), dict(scale=0.0), dict(scale=float("nan")),
                                    dict(heads=9), dict(stride=1020)])
def test_attention_refuses(library, change):
    assert attention(library, batch(), **change) == EINVAL


@pytest.mark.parametrize("kv,heads", [(batch(head_dim=96), 8), (batch(dtype=3), 8), (batch(kv_heads=1), 33),
                                      (batch(kv_heads=BIG // 1024, head_dim=64), BIG // 1024)])
def test_attention_supports_no_such_shape(library, kv, heads):
    assert attention(library, kv, heads=heads) == EUNSUPPORTED


def accept(library, logits=64, dtype=0, stride=1000, vocab=1000, tokens=64, parents=64, offsets=64, rows=4, sequences=2,
           max_path=3, targets=64, path=64, counts=64, following=64, workspace=64, nbytes=1 << 20):
    return library.h4b_tree_accept(logits, dtype, stride, vocab, tokens, parents, offsets, rows, sequences, max_path, targets,
                                   path, counts, following, workspace, nbytes, None)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(sequences=-1), dict(max_path=0), dict(vocab=0), dict(stride=999),
                                    dict(logits=66), dict(tokens=None), dict(parents=None), dict(offsets=None),
                                    dict(targets=None), dict(path=None), dict(counts=None), dict(following=None),
                                    dict(workspace=None), dict(workspace=68), dict(nbytes=100), dict(logits=None, targets=None)])
def test_accept_refuses(library, change):
    assert accept(library, **change) == EINVAL


def test_accept_supports_no_such_shape(library):
    assert accept(library, dtype=3) == EUNSUPPORTED
    assert accept(library, vocab=BIG - 1, stride=BIG) == EUNSUPPORTED
    assert accept(library, sequences=0) == 0


def test_accept_workspace(library):
    nbytes = library.h4b_tree_accept_workspace_bytes
    assert nbytes(-1, 1) == EINVAL and nbytes(1, -1) == EINVAL
    assert 0 < nbytes(1, 1) < 1 << 16
    assert accept(library, sequences=5000, nbytes=nbytes(4, 5000) - 1) == EINVAL


def keep(library, kv=None, layers=2, layer_bytes=4 * 8 * 16 * 128 * 2, path=64, max_path=3, counts=64, lengths=1 << 12):
    return library.h4b_tree_keep(ctypes.byref(kv if kv is not None else batch()), layers, layer_bytes, path, max_path, counts,
                                 lengths, None)


@pytest.mark.parametrize("change", [dict(layers=0), dict(max_path=0), dict(layer_bytes=16), dict(path=None), dict(counts=None),
                                    dict(lengths=None), dict(lengths=1 << 24), dict(lengths=64),
                                    dict(layer_bytes=4 * 8 * 16 * 128 * 2 + 8), dict(kv=batch(page_size=24))])
def test_keep_refuses(library, change):
    assert keep(library, **change) == EINVAL


def test_keep_supports_no_such_shape(library):
    assert keep(library, batch(head_dim=96)) == EUNSUPPORTED
    assert keep(library, layers=65536) == EUNSUPPORTED
    assert keep(library, batch(sequences=0)) == 0


def norm(library, x=64, x_dtype=0, x_stride=64, delta=64, delta_dtype=0, delta_stride=64, out=64, out_stride=64, weight=64,
         x8=64, scales=64, sums=64, rows=2, width=64):
    return library.h4b_rmsnorm_quantize_rows(x, x_dtype, x_stride, delta, delta_dtype, delta_stride, out, out_stride, weight,
                                             1e-6, x8, scales, sums, rows, width, None)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(width=0), dict(width=60), dict(x=None), dict(weight=None), dict(x8=None),
                                    dict(scales=None), dict(sums=None), dict(out=None), dict(x=72), dict(delta=72), dict(out=72),
                                    dict(weight=72), dict(x8=68), dict(x_stride=56), dict(x_stride=68), dict(delta_stride=56),
                                    dict(delta_stride=68), dict(out_stride=68)])
def test_norm_refuses(library, change):
    assert norm(library, **change) == EINVAL


def test_norm_supports_no_such_type(library):
    assert norm(library, x_dtype=3) == EUNSUPPORTED and norm(library, delta_dtype=-1) == EUNSUPPORTED
    assert norm(library, rows=0) == 0


def test_the_models_step_needs_parents(library):
    assert library.h4b_forward_paged_tree(None, None, None, None) == EINVAL
    assert library.h4b_forward_paged_tree(None, None, 64, None) == EINVAL


@pytest.mark.parametrize("below", [65, 100, 255, 300, 592, 600, 9000])
@pytest.mark.parametrize("rows,dtype", [(1, 1), (4, 0), (1 << 20, 2)])
def test_logits_whose_parts_pass_32_bits_are_refused(library, below, rows, dtype):
    """The ends of a row's parts lie up to 16 values a part behind the row's."""
    assert accept(library, vocab=BIG - 1 - below, stride=BIG, rows=rows, dtype=dtype, nbytes=1 << 30) == EUNSUPPORTED


# ---- sizes that a C int cuts off ---------------------------------------------------------
CUT = (1 << 32) + 8  # 8, cut off


def meta(*shape, dtype=None):
    import torch

    return torch.empty(shape, dtype=dtype or torch.int32, device="meta")


def test_sizes_past_32_bits_are_refused_not_cut_off(library):
    import torch

    from harsh4b_b200 import ops

    half, full = torch.float16, torch.float32
    for rows, width in ((CUT, 8), (1, CUT)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.rmsnorm_quantize_rows(meta(rows, width, dtype=half), meta(width, dtype=full), 1e-6)
    for rows, sequences, vocab in ((CUT, 1, 8), (8, CUT, 8), (8, 1, CUT)):
        batch = meta(rows), meta(rows), meta(sequences + 1)
        with pytest.raises(ValueError, match="32 bits"):
            ops.accept_tree(*batch, meta(rows, vocab, dtype=half))
        if vocab == 8:
            with pytest.raises(ValueError, match="32 bits"):
                ops.accept_tree(*batch, targets=meta(rows))
            with pytest.raises(ValueError, match="32 bits"):
                ops.accept_workspace(rows, sequences, "meta")


@pytest.mark.parametrize("at", [1 << 22, 1 << 23, (1 << 23) + 4, 1 << 24, 1 << 12, (1 << 12) + 8, 1 << 14])
def test_keep_refuses_lengths_over_what_it_reads(library, at):
    """The table, the offsets, the lengths, path and counts of one sequence: other CTAs read them while one writes."""
    assert keep(library, path=1 << 12, counts=1 << 14, lengths=at) == EINVAL
