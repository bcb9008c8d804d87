"""The 4-bit operators together, as a server's decoder layers use them: a voice's prompt, requests forked from
it, single-token steps, a compaction, a captured step."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4_oracle as F
from oracle import lm_oracle as O
from tests import fp4_bars, lm_bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HK, D, LAYERS = 4, 2, 64, 2
WIDTH = HQ * D


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Model:
    """Two decoder layers' 4-bit operators, and every intermediate result of the last call."""

    def __init__(self, fcv, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.fcv, self.dtype = fcv, dtype
        self.cos, self.sin = (t.to(DEV) for t in fcv.rope_tables(700, D, D))

        def weight(n, k):
            return fcv.quantize_fp4((torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).to(DEV))

        self.layers = [dict(qkv=weight((HQ + 2 * HK) * D, WIDTH), out=weight(WIDTH, WIDTH),
                            up=weight(2 * WIDTH, WIDTH), down=weight(WIDTH, 2 * WIDTH),
                            qw=torch.ones(D, dtype=dtype, device=DEV),
                            kw=torch.ones(D, dtype=dtype, device=DEV)) for _ in range(LAYERS)]
        self.pages = fcv.new_fp4_pages(40, HK, D, layers=LAYERS, device=DEV)
        self.book = fcv.CachePages(self.pages)

    def __call__(self, x, positions, rows, table, lengths, cu=None):
        f, self.trace = self.fcv, []
        for i, w in enumerate(self.layers):
            qkv = f.fused_linear_fp4(x, *w["qkv"])
            q = f.qk_norm_rope_fp4(qkv, positions, self.cos, self.sin, self.pages[i], rows, n_heads=HQ,
                                   q_weight=w["qw"], k_weight=w["kw"])
            o = f.paged_attention_fp4(q, self.pages[i], table, lengths, cu_q=cu)
            y = f.fused_linear_fp4(o.flatten(1), *w["out"], residual=x)
            h = f.fused_linear_fp4(y, *w["up"], activation="silu")
            z = f.fused_linear_fp4(h, *w["down"], residual=y)
            self.trace.append((x, qkv, q, o, y, h, z))
            x = z
        return x

    def check(self, positions, rows, table, lengths, cu=None):
        """Every operator's result against its formula on its own inputs."""
        for i, (w, (x, qkv, q, o, y, h, z)) in enumerate(zip(self.layers, self.trace)):
            for got, a, name, act, r in ((qkv, x, "qkv", None, None), (y, o.flatten(1), "out", None, x),
                                         (h, y, "up", "silu", None), (z, h, "down", None, y)):
                wt = F.weights(*w[name], a.shape[1], a.dtype)
                want, arg, mass = O.linear(a, wt, None, act, r)
                lm_bars.assert_within(got, want, lm_bars.linear(want, arg, mass, r, a.shape[1], act,
                                                                self.dtype), f"layer {i} {name}")
            at = positions.long().cpu()
            heads = qkv.view(-1, HQ + 2 * HK, D).cpu()
            c, s = self.cos.cpu()[at], self.sin.cpu()[at]
            want, size = O.norm_rope(heads[:, :HQ], w["qw"], 1e-6, c, s, False)
            lm_bars.assert_within(q, want, lm_bars.norm_rope(want, size, D, True, self.dtype), "q")
            k, _ = O.norm_rope(heads[:, HQ:HQ + HK], w["kw"], 1e-6, c, s, False)
            got = self.fcv.read_fp4_pages(self.pages[i], rows, dtype=self.dtype)
            assert torch.equal(got[0].cpu(), F.quantized(k, self.dtype, 32).to(self.dtype))
            assert torch.equal(got[1].cpu(), F.quantized(heads[:, HQ + HK:].double(),
                                                         self.dtype).to(self.dtype))
            want, _, mass, score, keys = F.attention(q, self.pages[i], table, lengths, cu)
            lm_bars.assert_within(o, want, fp4_bars.attention(want, mass, score, keys, D, self.dtype), "o")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_voice_and_its_requests(fcv, dtype):
    say(f"[fp4 step] {dtype}")
    model = Model(fcv, dtype)
    book = model.book
    g = torch.Generator().manual_seed(5)

    def hidden(n):
        return torch.randn(n, WIDTH, generator=g).to(dtype).to(DEV)

    def call(sessions, counts):
        before = book.lengths(sessions).tolist()
        rows = book.extend(sessions, counts)
        at = ints([p for b, c in zip(before, counts) for p in range(b, b + c)])
        cu = ints([0, *torch.tensor(counts).cumsum(0).tolist()])
        args = (at, rows, book.table(sessions), book.lengths(sessions), cu)
        out = model(hidden(sum(counts)), *args)
        model.check(*args)
        return out

    voice = book.open()
    call([voice], [100])                          # the prompt
    kids = [book.fork(voice) for _ in range(3)]
    call(kids, [20, 1, 7])                        # texts of several lengths: the shared page is copied
    for _ in range(2):
        call(kids, [1, 1, 1])                     # speech tokens, one each
    book.close(kids[0])
    late = book.fork(voice)
    book.close(voice)
    assert book.compact() > 0
    out = call([kids[1], late, kids[2]], [1, 5, 1])
    assert bool(out.isfinite().all())


def test_a_captured_step(fcv):
    """One step captured with tables of a fixed width, replayed token after token beside eager steps."""
    model, twin = Model(fcv, torch.bfloat16), Model(fcv, torch.bfloat16)
    g = torch.Generator().manual_seed(6)
    sessions = []
    for m in (model, twin):
        s = [m.book.open(), m.book.open()]
        rows = m.book.extend(s, [70, 60])
        m(torch.randn(130, WIDTH, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV),
          ints([*range(70), *range(60)]), rows, m.book.table(s, 8), m.book.lengths(s), ints([0, 70, 130]))
        sessions.append(s)
    x = torch.zeros(2, WIDTH, dtype=torch.bfloat16, device=DEV)
    at, rows, lengths = ints([0, 0]), ints([-1, -1]), ints([0, 0])
    table = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    model(x, at, rows, table, lengths)  # nothing is appended: rows are negative
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model(x, at, rows, table, lengths)
    for step in range(6):
        new = torch.randn(2, WIDTH, generator=g).bfloat16().to(DEV)
        got = []
        for m, s in zip((model, twin), sessions):
            before = m.book.lengths(s)
            r = m.book.extend(s, [1, 1])
            if m is model:
                x.copy_(new), at.copy_(before), rows.copy_(r), lengths.copy_(m.book.lengths(s))
                table.copy_(m.book.table(s, 8))
                graph.replay()
                got.append(out)
            else:
                got.append(m(new, before, r, m.book.table(s, 8), m.book.lengths(s)))
        torch.cuda.synchronize()
        assert torch.equal(*got), step
        assert torch.equal(model.pages, twin.pages), step
