"""Pages of a key/value cache: copies of them in all layers (include/fcv_fp4.h), and the book of which session
has which.

A scheduler decides on the host which session gets which page; what the GPU does about it are copies.  A
session forked from another (a request from its voice's prompt) shares its pages until one of the two
writes into the last, partly filled one, which is then copied.
"""

from __future__ import annotations

import heapq
from array import array

import torch

from . import _lib
from .lm import _launch

PAGE = 64  # FCV_FP4_PAGE, tokens of a page


def copy_pages(pages: torch.Tensor, src: list[int], dst: list[int]) -> None:
    """Copies page ``src[i]`` of every layer to page ``dst[i]``, in place.

    ``pages`` is ``[layers, n_pages, ...]`` on the GPU, of any type, each page's bytes contiguous: a pool of
    ``new_fp4_pages``, or 16-bit caches laid out so.  ``src`` and ``dst`` are numbers on the host; a page
    may be a source more than once, but no page is a destination twice, or both a source and a
    destination (``ValueError``).  Asynchronous on the current stream; a captured call copies the
    same pages on every replay."""
    if pages.dim() < 3 or not pages.is_cuda:
        raise ValueError("pages must be a tensor [layers, pages, ...] on the GPU, got "
                         f"{tuple(pages.shape)} on {pages.device}")
    layers, n_pages = pages.shape[:2]
    size = pages.element_size()
    step = 1
    for n, stride in zip(reversed(pages.shape[2:]), reversed(pages.stride()[2:])):
        if n > 1 and stride != step:
            raise ValueError(f"a page's bytes must be contiguous, got strides {pages.stride()}")
        step *= n
    if isinstance(src, (bytes, bytearray)) or isinstance(dst, (bytes, bytearray)):
        raise ValueError("src and dst must be lists of page numbers, not bytes")  # an array's own integers
    try:
        lists = array("i", src), array("i", dst)
    except OverflowError as e:
        raise ValueError(f"a page is outside the pool of {n_pages}") from e
    except TypeError as e:
        raise ValueError(f"src and dst must be lists of page numbers: {e}") from e
    if len(lists[0]) != len(lists[1]):
        raise ValueError(f"{len(lists[0])} sources and {len(lists[1])} destinations")
    _launch(_lib.load().fcv_copy_pages, pages.device.index, pages.data_ptr(), layers,
            pages.stride(0) * size, n_pages, pages.stride(1) * size if n_pages > 1 else step * size,
            step * size, lists[0].buffer_info()[0], lists[1].buffer_info()[0], len(lists[0]))


class CachePages:
    """The book of a pool of pages ``[layers, n_pages, ...]``: sessions, their lengths and their pages.

        book = CachePages(pages)
        voice = book.open()
        rows = book.extend([voice], [prompt_length])   # where qk_norm_rope_fp4 puts the prompt's tokens
        request = book.fork(voice)                     # shares the prompt's pages
        rows = book.extend([request, ...], [1, ...])   # copies a shared last page before it is written
        table, lengths = book.table([request, ...]), book.lengths([request, ...])
        book.close(request); book.compact()

    Copies run on the current stream when a method needs them: calls on one stream are in order.  A pool
    that is full raises ``RuntimeError`` and changes nothing, as any error does.  Driven from one thread."""

    def __init__(self, pages: torch.Tensor):
        if pages.dim() < 3:
            raise ValueError(f"pages must be [layers, pages, ...], got {tuple(pages.shape)}")
        self.pages = pages
        self._free = list(range(pages.shape[1]))  # a heap: the lowest page first
        self._users = [0] * pages.shape[1]
        self._held: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    def _copy(self, src: list[int], dst: list[int]) -> None:
        if src:
            copy_pages(self.pages, src, dst)

    def _session(self, session: int) -> list[int]:
        held = self._held.get(session)
        if held is None:
            raise ValueError(f"no session {session}")
        return held

    @property
    def free(self) -> int:
        """How many pages no session has."""
        return len(self._free)

    def open(self) -> int:
        """A new, empty session."""
        session, self._next = self._next, self._next + 1
        self._held[session], self._length[session] = [], 0
        return session

    def fork(self, session: int) -> int:
        """A new session with the same tokens; the pages are shared."""
        held = self._session(session)
        new = self.open()
        for page in held:
            self._users[page] += 1
        self._held[new], self._length[new] = list(held), self._length[session]
        return new

    def extend(self, sessions: list[int], counts: list[int]) -> torch.Tensor:
        """Room for ``counts[i]`` more tokens of ``sessions[i]``: their cache rows, int32, session after
        session, on the pool's device.  A last page that is shared and partly filled is copied first."""
        if len(sessions) != len(counts) or len(set(sessions)) != len(sessions):
            raise ValueError("one count for each of different sessions")
        plan, need = [], 0
        left: dict[int, int] = {}  # users of a shared last page, without those that copy it
        for session, count in zip(sessions, counts):
            held, length = self._session(session), self._length[session]
            if count < 0:
                raise ValueError(f"a negative count: {count}")
            copied = False
            if count and length % PAGE:
                users = left.get(held[-1], self._users[held[-1]])
                copied = users > 1
                left[held[-1]] = users - copied
            more = (length + count + PAGE - 1) // PAGE - len(held)
            plan.append((session, count, copied, more))
            need += copied + more
        if need > len(self._free):
            raise RuntimeError(f"{need} pages are needed, {len(self._free)} of {len(self._users)} "
                               "are free")
        taken = [heapq.heappop(self._free) for _ in range(need)]
        try:  # nothing else changes before the copy is on its way and the rows are there
            fresh = iter(taken)
            src, dst, rows, held_now = [], [], [], []
            for session, count, copied, more in plan:
                held, length = list(self._held[session]), self._length[session]
                if copied:
                    src.append(held[-1])
                    held[-1] = next(fresh)
                    dst.append(held[-1])
                held += [next(fresh) for _ in range(more)]
                rows += [held[i // PAGE] * PAGE + i % PAGE for i in range(length, length + count)]
                held_now.append(held)
            self._copy(src, dst)
            out = torch.tensor(rows, dtype=torch.int32, device=self.pages.device)
        except BaseException:
            for page in taken:
                heapq.heappush(self._free, page)
            raise
        for (session, count, _, _), held in zip(plan, held_now):
            self._held[session] = held
            self._length[session] += count
        for page in src:
            self._users[page] -= 1
        for page in taken:
            self._users[page] = 1
        return out

    def close(self, session: int) -> None:
        """Ends a session; pages that no other has are free again."""
        for page in self._session(session):
            self._users[page] -= 1
            if self._users[page] == 0:
                heapq.heappush(self._free, page)
        del self._held[session], self._length[session]

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; how many were moved.  Tables and rows given
        out before no longer hold."""
        used = len(self._users) - len(self._free)
        dst = sorted(page for page in self._free if page < used)
        src = [page for page in range(used, len(self._users)) if self._users[page]]
        self._copy(src, dst)
        to = dict(zip(src, dst))
        for held in self._held.values():
            held[:] = [to.get(page, page) for page in held]
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(used, len(self._users)))
        return len(src)

    def lengths(self, sessions: list[int]) -> torch.Tensor:
        """The sessions' token counts, int32 on the pool's device."""
        for session in sessions:
            self._session(session)
        return torch.tensor([self._length[s] for s in sessions], dtype=torch.int32,
                            device=self.pages.device)

    def table(self, sessions: list[int], width: int | None = None) -> torch.Tensor:
        """The sessions' pages, int32 ``[len(sessions), width]`` on the pool's device, -1 behind the last;
        ``width`` defaults to the most pages that one has."""
        held = [self._session(s) for s in sessions]
        most = max((len(h) for h in held), default=0)
        if width is None:
            width = max(most, 1)
        elif most > width:
            raise ValueError(f"a session has {most} pages, the table {width}")
        return torch.tensor([h + [-1] * (width - len(h)) for h in held], dtype=torch.int32,
                            device=self.pages.device).view(len(held), width)
