"""The host side of the paged cache: pages held, shared, freed, trimmed and
compacted (the copies are recorded, not run)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from harsh4b_b200 import paged  # noqa: E402


@pytest.fixture
def cache(monkeypatch):
    made = paged.PagedCache(2, 2, 64, pages=12, page_size=16, device="cpu")
    made.moves = []

    def record(k_pages, v_pages, src, dst):
        pairs = list(zip(src.tolist(), dst.tolist()))
        assert not {a for a, _ in pairs} & {b for _, b in pairs}
        assert len({b for _, b in pairs}) == len(pairs)
        for a, b in pairs:
            k_pages[:, b], v_pages[:, b] = k_pages[:, a].clone(), v_pages[:, a].clone()
        made.moves.extend(pairs)

    monkeypatch.setattr(paged.ops, "copy_pages", record)
    return made


def grow(cache, sequence, count):
    """Append `count` tokens whose value is their position + 100 * sequence."""
    cache.reserve({sequence: count})
    start = cache.length(sequence)
    for p in range(start, start + count):
        cache.k_pages[:, cache.table(sequence)[p // 16], :, p % 16] = p + 100 * sequence
    cache.advance(sequence, count)


def read(cache, sequence):
    return [int(cache.k_pages[0, cache.table(sequence)[p // 16], 0, p % 16, 0]) for p in range(cache.length(sequence))]


def consistent(cache):
    held = [p for s in cache._tables for p in cache.table(s) if p >= 0]
    counts = np.bincount(held, minlength=cache.pages)
    assert np.array_equal(counts, cache._shared)
    assert sorted(cache._free) == np.flatnonzero(counts == 0).tolist()


def test_grow_and_free(cache):
    a = cache.new_sequence()
    grow(cache, a, 40)
    assert len(cache.table(a)) == 3 and cache.free_pages == 9
    grow(cache, a, 8)
    assert len(cache.table(a)) == 3
    grow(cache, a, 1)
    assert len(cache.table(a)) == 4
    consistent(cache)
    cache.free(a)
    assert cache.free_pages == 12
    consistent(cache)


def test_fork_shares_until_written(cache):
    a = cache.new_sequence()
    grow(cache, a, 40)
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 9
    grow(cache, b, 1)
    assert cache.moves == [(cache.table(a)[2], cache.table(b)[2])]
    assert cache.table(b)[:2] == cache.table(a)[:2]
    consistent(cache)
    assert read(cache, b) == list(range(40)) + [40 + 100 * b] and read(cache, c) == list(range(40))
    grow(cache, a, 1)  # c still holds the old page
    grow(cache, c, 1)  # and now alone
    assert len(cache.moves) == 2
    assert read(cache, a)[-1] == 40 + 100 * a and read(cache, c)[-1] == 40 + 100 * c
    consistent(cache)


def test_forks_reserved_together_copy_once_less(cache):
    a = cache.new_sequence()
    grow(cache, a, 20)
    b, c = cache.fork(a), cache.fork(a)
    cache.reserve({a: 1, b: 1, c: 1})
    assert len(cache.moves) == 2  # the last one keeps the page
    assert len({cache.table(s)[1] for s in (a, b, c)}) == 3
    consistent(cache)


def test_fork_at_a_page_boundary_copies_nothing(cache):
    a = cache.new_sequence()
    grow(cache, a, 32)
    b = cache.fork(a)
    grow(cache, b, 5)
    assert cache.moves == []
    assert read(cache, a) == list(range(32))
    consistent(cache)


def test_out_of_pages_changes_nothing(cache):
    a, b = cache.new_sequence(), cache.new_sequence()
    grow(cache, a, 100)
    before = cache.table(a), cache.table(b), cache.free_pages
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.reserve({a: 10, b: 100})
    assert (cache.table(a), cache.table(b), cache.free_pages) == before
    consistent(cache)


def test_trim_and_truncate(cache):
    a = cache.new_sequence()
    grow(cache, a, 100)
    # the next token stands at 100 and sees 81..100 and 0..3
    assert cache.trim(a, window=20, sinks=4) == 4
    assert cache.table(a)[0] >= 0 and cache.table(a)[1:5] == [-1] * 4 and min(cache.table(a)[5:]) >= 0
    assert cache.trim(a, window=20, sinks=4) == 0
    consistent(cache)
    cache.truncate(a, 97)
    cache.truncate(a, 96)
    assert len(cache.table(a)) == 6
    consistent(cache)
    with pytest.raises(ValueError):
        cache.truncate(a, 97)
    b = cache.fork(a)
    cache.free(a)
    consistent(cache)
    grow(cache, b, 3)
    cache.free(b)
    assert cache.free_pages == 12


def test_appending_to_a_trimmed_page_is_refused(cache):
    a = cache.new_sequence()
    grow(cache, a, 20)
    cache._drop(cache._tables[a][1])
    cache._tables[a][1] = -1
    with pytest.raises(RuntimeError, match="trimmed"):
        cache.reserve({a: 1})


def test_compact(cache):
    a, b, c = (cache.new_sequence() for _ in range(3))
    for s in (a, b, c):
        grow(cache, s, 50)
    d = cache.fork(c)
    cache.free(a)
    cache.free(b)
    assert cache.compact() == 4
    assert sorted(cache.table(c)) == [0, 1, 2, 3] and cache.table(c) == cache.table(d)
    assert read(cache, c) == [p + 100 * c for p in range(50)]
    assert cache.compact() == 0
    consistent(cache)


def test_batch_tables(cache):
    a, b = cache.new_sequence(), cache.new_sequence()
    grow(cache, a, 40)
    cache.reserve({b: 3})
    table, offsets, lengths = cache.batch_tables([b, a], [3, 1])
    assert table.tolist() == [cache.table(b) + [-1, -1], cache.table(a)]
    assert offsets.tolist() == [0, 3, 4] and lengths.tolist() == [3, 41]


def test_refusals():
    make = paged.PagedCache
    for kwargs in (dict(page_size=24), dict(page_size=8), dict(dtype="float32"), dict(head_dim=96), dict(pages=0)):
        args = dict(layers=1, kv_heads=1, head_dim=64, pages=4, device="cpu")
        args.update(kwargs)
        with pytest.raises(ValueError):
            make(**args)
    cache = make(1, 1, 64, pages=4, device="cpu")
    a = cache.new_sequence()
    with pytest.raises(ValueError):
        cache.reserve({a: -1})
    with pytest.raises(ValueError):
        cache.advance(a, 1)
    with pytest.raises(ValueError):
        cache.trim(a, 0)
