"""Host logic of a paged cache: the book of free and shared pages."""
import numpy as np
import pytest

from kandle_b200.paged import PagePool


def test_pages_are_taken_shared_and_released():
    p = PagePool(6)
    a = p.take(3)
    assert a.tolist() == [0, 1, 2] and p.free == 3
    p.share(a[:2])
    p.release(a)
    assert p.free == 4 and p.held.tolist() == [1, 1, 0, 0, 0, 0]
    b = p.take(2)
    assert b.tolist() == [2, 3]
    p.release([0, 1])
    assert p.take(4).tolist() == [0, 1, 4, 5]
    with pytest.raises(ValueError, match="overflow"):
        p.take(1)
    p.release([3, 3][:1])
    assert p.free == 1 and p.take(0).size == 0


def test_misuse_is_refused_and_changes_nothing():
    p = PagePool(4)
    p.take(2)
    before = p.held.copy()
    for call, pages in ((p.release, [2]), (p.release, [0, 0]), (p.share, [3]), (p.release, [-1]), (p.release, [4]), (p.share, [9]), (p.keep, [7])):
        with pytest.raises(ValueError):
            call(pages)
        assert np.array_equal(p.held, before) and p.free == 2


def test_a_page_that_several_release_at_once_is_free_once():
    p = PagePool(3)
    a = p.take(1)
    p.share([0])
    p.release([0, 0])
    assert p.free == 3 and p.take(3).tolist() == [0, 1, 2] and a.tolist() == [0]


def test_compaction_moves_the_last_pages_into_the_holes():
    rng = np.random.default_rng(0)
    for _ in range(50):
        n = int(rng.integers(1, 40))
        p = PagePool(n)
        p.keep(rng.integers(0, n, int(rng.integers(0, n + 1))))
        held, count = p.held.copy(), int((p.held > 0).sum())
        src, dst = p.compact()
        assert len(src) == len(dst) and not set(src) & set(dst) and len(set(dst)) == len(dst)
        held[dst], held[src] = held[src], 0
        assert np.array_equal(held, p.held) and (p.held[:count] > 0).all() and not p.held[count:].any() and p.free == n - count
        assert p.take(p.free).tolist() == list(range(count, n))


def test_what_the_tables_say_is_held():
    p = PagePool(8)
    p.keep(np.array([[1, 2, 5], [1, 2, 6]]))
    assert p.held.tolist() == [0, 2, 2, 0, 0, 1, 1, 0] and p.free == 4 and p.take(2).tolist() == [0, 3]
