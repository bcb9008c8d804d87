"""``copy_pages`` and ``CachePages`` on the GPU."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def expect(pages, src, dst):
    want = pages.clone()
    for a, b in zip(src, dst):
        want[:, b] = pages[:, a]
    return want


@pytest.mark.parametrize("shape,dtype", [
    ((1, 5, 16), torch.uint8), ((3, 40, 2, 4288), torch.uint8), ((2, 9, 7), torch.uint8),
    ((4, 12, 3, 5, 64), torch.bfloat16), ((2, 700, 1, 4288), torch.uint8), ((5, 6, 33), torch.float32),
    ((1, 3, 100003), torch.uint8), ((300, 4, 32), torch.uint8), ((2, 8, 1), torch.float16)])
def test_copies(fcv, shape, dtype):
    say(f"[pages] {shape} {dtype}")
    g = torch.Generator().manual_seed(1)
    pages = torch.randint(0, 120, shape, generator=g).to(dtype).to(DEV)
    order = torch.randperm(shape[1], generator=g).tolist()
    half = len(order) // 2
    for src, dst in ((order[:half], order[half:2 * half]), ([order[0]] * (len(order) - 1), order[1:]),
                     ([order[-1]], [order[0]]), ([], [])):
        want = expect(pages, src, dst)
        fcv.copy_pages(pages, src, dst)
        assert torch.equal(pages, want)


def test_strides(fcv):
    """Layers inside pages, pages with gaps between them, starts off 16-byte boundaries."""
    g = torch.Generator().manual_seed(2)
    buf = torch.randint(0, 200, (9, 4, 100), generator=g, dtype=torch.uint8).to(DEV)
    for view in (buf.transpose(0, 1), buf.transpose(0, 1)[:, :, 3:81], buf[::2], buf.transpose(0, 1)[1:3]):
        whole, want = buf.clone(), view.clone()
        n = view.shape[1]
        want = expect(want, [0], [n - 1])
        fcv.copy_pages(view, [0], [n - 1])
        assert torch.equal(view, want)
        changed = (buf != whole).sum()
        assert int(changed) <= view.shape[0] * view.shape[2]


def test_captured(fcv):
    pages = torch.zeros(2, 6, 4288, dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fcv.copy_pages(pages, [0, 1], [4, 5])
    for seed in range(3):
        pages.copy_(torch.randint(0, 256, pages.shape, generator=torch.Generator().manual_seed(seed),
                                  dtype=torch.uint8))
        want = expect(pages, [0, 1], [4, 5])
        graph.replay()
        assert torch.equal(pages, want)


def test_refusals(fcv):
    pages = torch.zeros(2, 6, 64, dtype=torch.uint8, device=DEV)
    for a, match in [((pages, [0], [6]), "outside"), ((pages, [-1], [2]), "outside"),
                     ((pages, [0, 1], [2, 2]), "twice"), ((pages, [0, 1], [1, 2]), "both"),
                     ((pages, [3], [3]), "both"), ((pages, [0, 1], [2]), "2 sources"),
                     ((pages, [1 << 40], [2]), "outside"), ((pages, [0.5], [2]), "page numbers"),
                     ((pages[0], [0], [1]), "layers, pages"), ((pages.cpu(), [0], [1]), "GPU"),
                     ((pages[:, :, ::2], [0], [1]), "contiguous"),
                     ((pages[:1].expand(3, -1, -1), [0], [1]), "overlap"),
                     ((pages[:, :1].expand(-1, 4, -1), [0], [1]), "overlap")]:
        before = pages.clone()
        with pytest.raises(ValueError, match=match):
            fcv.copy_pages(*a)
        assert torch.equal(pages, before)


def test_book(fcv):
    """A voice's prompt, forks that write on, closed sessions and a compaction: every session's bytes are
    those that it was given."""
    pages = torch.zeros(3, 40, 2, 4288, dtype=torch.uint8, device=DEV)
    book = fcv.CachePages(pages)
    truth: dict[int, list[int]] = {}
    stamp = 0

    def write(session, count):
        nonlocal stamp
        rows = book.extend([session], [count]).tolist()
        for row in rows:  # a token's mark: byte `place` of its page in every layer
            stamp = stamp % 250 + 1
            pages[:, row // 64, :, row % 64] = stamp
            truth[session].append(stamp)

    def look():
        for session, marks in truth.items():
            held = book.table([session])[0].tolist()
            got = [int(pages[2, held[i // 64], 1, i % 64]) for i in range(len(marks))]
            assert got == marks, session
            assert book.lengths([session]).tolist() == [len(marks)]

    voice = book.open()
    truth[voice] = []
    write(voice, 100)
    kids = [book.fork(voice) for _ in range(5)]
    for kid in kids:
        truth[kid] = list(truth[voice])
    assert book.free == 38
    for kid in kids:
        write(kid, 3)
    write(voice, 70)
    look()
    for kid in kids[1:4]:
        book.close(kid)
        del truth[kid]
    other = book.open()
    truth[other] = []
    write(other, 200)
    book.close(voice)
    del truth[voice]
    look()
    assert book.compact() > 0
    look()
    used = 40 - book.free
    assert all(max(book.table([s])[0].tolist()) < used for s in truth)
    write(other, 60)
    look()


@pytest.mark.parametrize("d", [64, 128])
def test_offsets_that_pass_32_bits(fcv, d):
    """Pages and heads gigabytes apart: every operator as over a dense pool."""
    hk, hq, n = 2, 8, 6
    g = torch.Generator().manual_seed(d)
    dense = fcv.new_fp4_pages(n, hk, d, device=DEV)
    size = dense.shape[2]
    flat = torch.empty(5 * 2 ** 30 + 2 ** 29 + size, dtype=torch.uint8, device=DEV)
    far = flat.as_strided((n, hk, size), (2 ** 30, 2 ** 29, 1))
    far.zero_()
    tokens = 300
    qkv = torch.randn(tokens, (hq + 2 * hk) * d, generator=g).to(DEV, torch.bfloat16)
    rows = (torch.randperm(n * 64, generator=g)[:tokens]).int().to(DEV)
    angle = torch.rand(tokens, d // 2, generator=g).to(DEV)
    cos, sin = angle.cos(), angle.sin()
    pos = torch.arange(tokens, dtype=torch.int32, device=DEV)
    q = [fcv.qk_norm_rope_fp4(qkv, pos, cos, sin, pool, rows, n_heads=hq) for pool in (dense, far)]
    assert torch.equal(q[0], q[1]) and torch.equal(dense, far)
    for a, b in zip(fcv.read_fp4_pages(dense, rows, dtype=torch.bfloat16),
                    fcv.read_fp4_pages(far, rows, dtype=torch.bfloat16)):
        assert torch.equal(a, b)
    table = torch.tensor([[5, 0, 4, 1, 3, 2]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([n * 64 - 5], dtype=torch.int32, device=DEV)
    for count in (1, 3, tokens):  # each form of the attention
        many = q[0][:count].repeat(1 if count < tokens else 24, 1, 1)
        batch = 1 if count < tokens else 24
        got = [fcv.paged_attention_fp4(many, pool, table.expand(batch, -1), lengths.expand(batch).contiguous())
               for pool in (dense, far)]
        assert torch.equal(got[0], got[1])
    fcv.copy_pages(far.transpose(0, 1), [5, 0], [1, 4])  # a head as a layer: its bytes lie together
    assert torch.equal(far[1], dense[5]) and torch.equal(far[4], dense[0])
