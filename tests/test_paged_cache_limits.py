"""The host side of the paged cache where its promises could break: forks over
reserved room (the copies are recorded, not run)."""
import pytest

from test_paged_cache import cache, consistent, grow, read  # noqa: F401 (cache is a fixture)

torch = pytest.importorskip("torch")


def write(cache, sequence, value):
    """One token into the reserved room."""
    p = cache.length(sequence)
    cache.k_pages[:, cache.table(sequence)[p // 16], :, p % 16] = value
    cache.advance(sequence, 1)


@pytest.mark.parametrize("length", [0, 5, 16, 20, 32])
def test_fork_leaves_reserved_room_to_its_owner(cache, length):  # noqa: F811
    a = cache.new_sequence()
    cache.reserve({a: length + 40})
    for p in range(length):
        write(cache, a, p)
    own = cache.table(a)
    b = cache.fork(a)
    cache.reserve({a: 1, b: 1})
    consistent(cache)
    assert not set(cache.table(a)[length // 16:]) & set(cache.table(b)[length // 16:])
    write(cache, a, 70)
    write(cache, b, 71)
    assert read(cache, a) == list(range(length)) + [70] and read(cache, b) == list(range(length)) + [71]
    assert len(cache.table(a)) == len(own)  # a's room is still there


@pytest.mark.parametrize("length", [5, 16, 20])
def test_reserved_room_outlives_a_fork(cache, length):  # noqa: F811
    """The owner goes on in its room without reserving anew."""
    a = cache.new_sequence()
    cache.reserve({a: length + 30})
    for p in range(length):
        write(cache, a, p)
    b = cache.fork(a)
    for p in range(length, length + 10):
        write(cache, a, p)
    grow(cache, b, 20)
    for p in range(length + 10, length + 30):
        write(cache, a, p)
    assert read(cache, a) == list(range(length + 30))
    assert read(cache, b) == list(range(length)) + [p + 100 * b for p in range(length, length + 20)]
    consistent(cache)
