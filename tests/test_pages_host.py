"""The book of a cache's pages, on the CPU: sharing, copies on write, compaction, refusals that change nothing."""

from __future__ import annotations

import pytest
import torch


@pytest.fixture
def book(fcv):
    class Book(fcv.CachePages):
        def __init__(self, n):
            super().__init__(torch.zeros(1, n, 1))
            self.moves = []

        def _copy(self, src, dst):
            assert len(set(dst)) == len(dst) and not set(src) & set(dst)
            self.moves += list(zip(src, dst))

    return Book


def test_rows_are_in_order_and_pages_the_lowest(book):
    b = book(10)
    s = b.open()
    assert b.extend([s], [70]).tolist() == list(range(70))
    assert b.extend([s], [0]).tolist() == []
    t = b.open()
    assert b.extend([t, s], [2, 60]).tolist() == [128, 129] + list(range(70, 128)) + [192, 193]
    assert b.table([s, t]).tolist() == [[0, 1, 3], [2, -1, -1]]
    assert b.table([t], 2).tolist() == [[2, -1]]
    assert b.lengths([t, s]).tolist() == [2, 130]
    assert b.free == 6 and b.moves == []


def test_forks_share_until_they_write(book):
    b = book(10)
    s = b.open()
    b.extend([s], [100])
    kids = [b.fork(s) for _ in range(3)]
    assert b.free == 8
    assert b.extend([kids[0], kids[1]], [1, 1]).tolist() == [2 * 64 + 36, 3 * 64 + 36]
    assert b.moves == [(1, 2), (1, 3)]
    # the last two that share the page: one copies, the other then has it alone
    assert b.extend([kids[2], s], [1, 1]).tolist() == [4 * 64 + 36, 64 + 36]
    assert b.moves[2:] == [(1, 4)]
    assert b.extend([s], [1]).tolist() == [64 + 37]
    for k in kids:
        b.close(k)
    assert b.free == 8
    b.close(s)
    assert b.free == 10


def test_a_full_last_page_is_not_copied(book):
    b = book(4)
    s = b.open()
    b.extend([s], [64])
    k = b.fork(s)
    assert b.extend([k, s], [1, 1]).tolist() == [64, 128]
    assert b.moves == []


def test_a_pool_that_is_full_changes_nothing(book):
    b = book(3)
    s = b.open()
    b.extend([s], [100])
    k = b.fork(s)
    before = (b.table([s, k]).tolist(), b.lengths([s, k]).tolist(), b.free)
    with pytest.raises(RuntimeError, match="2 pages are needed, 1 of 3"):
        b.extend([k, s], [1, 64])
    assert (b.table([s, k]).tolist(), b.lengths([s, k]).tolist(), b.free) == before and not b.moves
    assert b.extend([k], [1]).tolist() == [2 * 64 + 36]


def test_compaction(book):
    b = book(12)
    sessions = [b.open() for _ in range(5)]
    b.extend(sessions, [64, 128, 64, 70, 64])
    kid = b.fork(sessions[3])
    b.close(sessions[0])
    b.close(sessions[1])
    assert b.compact() == 3  # pages 3 .. 6 are in use, 0 .. 2 free
    assert b.moves == [(4, 0), (5, 1), (6, 2)]
    held = b.table([sessions[2], sessions[3], kid, sessions[4]]).tolist()
    assert held[1] == held[2]
    assert sorted({p for row in held for p in row if p >= 0}) == [0, 1, 2, 3]
    assert b.free == 8 and b.compact() == 0
    b.close(kid)
    assert b.free == 8
    assert b.extend([sessions[2]], [64]).tolist()[0] == 4 * 64


def test_refusals(book, fcv):
    b = book(4)
    s = b.open()
    for bad in (lambda: b.extend([s, s], [1, 1]), lambda: b.extend([s], [1, 2]), lambda: b.extend([s], [-1]),
                lambda: b.extend([99], [1]), lambda: b.fork(99), lambda: b.close(99), lambda: b.lengths([99]),
                lambda: b.table([99])):
        with pytest.raises(ValueError):
            bad()
    b.extend([s], [65])
    with pytest.raises(ValueError, match="2 pages, the table 1"):
        b.table([s], 1)
    with pytest.raises(ValueError, match="layers, pages"):
        fcv.CachePages(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="GPU"):
        fcv.copy_pages(torch.zeros(1, 4, 16), [0], [1])
