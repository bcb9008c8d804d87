"""What ``copy_pages`` hands the library, on the CPU: as many page numbers as it says."""

from __future__ import annotations

import ctypes

import pytest


class Pool:
    """As much of a pool on the GPU as ``copy_pages`` looks at."""

    is_cuda, shape, device = True, (2, 8, 64), type("device", (), {"index": 0})

    def dim(self):
        return 3

    def element_size(self):
        return 1

    def stride(self, i=None):
        return (512, 64, 1) if i is None else (512, 64, 1)[i]

    def data_ptr(self):
        return 1 << 40


@pytest.fixture
def calls(fcv, monkeypatch):
    got = []
    module = __import__("faster_cosyvoice_amd.pages", fromlist=["x"])

    def launch(fn, index, *args):
        src, dst, count = args[-3:]
        got.append((count, [list((ctypes.c_int32 * count).from_address(a)) if count else [] for a in (src, dst)]))

    monkeypatch.setattr(module, "_launch", launch)
    return got


def test_lists(fcv, calls):
    fcv.copy_pages(Pool(), [0, 1], (6, 7))
    fcv.copy_pages(Pool(), range(3), iter([5, 6, 7]))
    fcv.copy_pages(Pool(), [], [])
    assert calls == [(2, [[0, 1], [6, 7]]), (3, [[0, 1, 2], [5, 6, 7]]), (0, [[], []])]


@pytest.mark.parametrize("src,dst", [(b"\1\0\0\0", b"\2\0\0\0"), (bytearray(4), [2, 3, 4, 5]), (b"\0\0\0\0", [5]),
                                     ("0", "1"), ([0], [1, 2]), (range(2), iter([5])), (5, 6)])
def test_refusals(fcv, calls, src, dst):
    """Bytes are the machine's integers to an array: four of them are one page number, not four."""
    with pytest.raises(ValueError):
        fcv.copy_pages(Pool(), src, dst)
    assert calls == []


def test_a_copy_that_fails_changes_nothing(fcv):
    """The book stays as it was where the pages cannot be copied (here: a pool that is not on the GPU)."""
    import torch

    book = fcv.CachePages(torch.zeros(1, 12, 16))
    voice, other = book.open(), book.open()
    book.extend([other, voice], [64, 100])
    kids = [book.fork(voice) for _ in range(2)]
    everyone = [voice, other, *kids]
    before = (book.table(everyone).tolist(), book.lengths(everyone).tolist(), book.free)
    for sessions, counts in (([kids[0]], [1]), ([other, kids[0], kids[1], voice], [70, 1, 200, 2])):
        with pytest.raises(ValueError, match="GPU"):
            book.extend(sessions, counts)
        assert (book.table(everyone).tolist(), book.lengths(everyone).tolist(), book.free) == before
    assert book.extend([other], [2]).tolist() == [3 * 64, 3 * 64 + 1]  # pages 0 to 2 are in use
    book.close(kids[0])
    book.close(kids[1])
    assert book.extend([voice], [1]).tolist() == [2 * 64 + 36] and book.free == 8
    book.close(other)
    before = (book.table([voice]).tolist(), book.free)
    with pytest.raises(ValueError, match="GPU"):
        book.compact()
    assert (book.table([voice]).tolist(), book.free) == before
