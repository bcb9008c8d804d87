"""The language model operators together, as a decoder layer runs them: a voice's prompt is prefilled
once, requests append their texts, then tokens, eagerly and from a captured graph."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests.gpu_helpers import rel_l2, say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HK, DIM, WIDTH, FF = 14, 2, 64, 896, 1300
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def weights(dtype, seed=11):
    g = torch.Generator().manual_seed(seed)

    def w(n, k):
        return (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).to(DEV)

    qkv = (HQ + 2 * HK) * DIM
    return {"qkv": w(qkv, WIDTH), "qkv_b": (0.2 * torch.randn(qkv, generator=g)).to(dtype).to(DEV),
            "out": w(WIDTH, HQ * DIM), "up": w(FF, WIDTH), "down": w(WIDTH, FF),
            "qn": (1 + 0.2 * torch.randn(DIM, generator=g)).to(DEV),
            "kn": (1 + 0.2 * torch.randn(DIM, generator=g)).to(DEV)}


def layer(fcv, w, x, tables, pos, rows, caches, lengths, **attn):
    """One layer (without its norms) on the rows ``x``."""
    k, v = caches
    qkv = fcv.fused_linear(x, w["qkv"], w["qkv_b"])
    q = fcv.qk_norm_rope(qkv, pos, *tables, k, v, rows, n_heads=HQ, q_weight=w["qn"],
                         k_weight=w["kn"], eps=EPS)
    o = fcv.prefix_attention(q, k, v, lengths, **attn)
    x = fcv.fused_linear(o.flatten(1), w["out"], residual=x)
    h = fcv.fused_linear(x, w["up"], activation="gelu_tanh")
    return fcv.fused_linear(h, w["down"], residual=x)


def exact_layer(w, x, cos, sin, pos, past):
    """The same for one sequence in 64 bits on all of its tokens so far: ``past`` are earlier keys and
    values, returned with the new ones behind."""
    d = {n: t.double().cpu() for n, t in w.items()}
    t = x.shape[0]
    qkv = (x @ d["qkv"].t() + d["qkv_b"]).view(t, HQ + 2 * HK, DIM)
    c, s = cos.cpu()[pos], sin.cpu()[pos]
    q, _ = O.norm_rope(qkv[:, :HQ], d["qn"], EPS, c, s, False)
    k, _ = O.norm_rope(qkv[:, HQ:HQ + HK], d["kn"], EPS, c, s, False)
    k, v = torch.cat((past[0], k)), torch.cat((past[1], qkv[:, HQ + HK:]))
    n = k.shape[0]
    visible = torch.arange(n) <= (n - t + torch.arange(t))[:, None]
    o = torch.stack([O.attention(q[:, h], k[:, h // (HQ // HK)], v[:, h // (HQ // HK)], visible,
                                 DIM ** -0.5)[0] for h in range(HQ)], 1)
    x = x + o.flatten(1) @ d["out"].t()
    return x + O.activate(x @ d["up"].t(), "gelu_tanh") @ d["down"].t(), (k, v)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_prefill_append_decode(fcv, dtype):
    """Every output within 8 half steps relative L2 (six roundings to the type on a row's way, each
    of at most half a step, through matrices of unit gain) of the 64-bit layer."""
    say(f"[layer] {dtype}")
    bar = 8 * torch.finfo(dtype).eps / 2
    w, p, cap = weights(dtype), 83, 64
    tables = tuple(t.to(DEV) for t in fcv.rope_tables(300, DIM, DIM))
    g = torch.Generator().manual_seed(3)

    def rows_of(n):
        return torch.randn(n, WIDTH, generator=g).to(dtype)

    zero = (torch.zeros(0, HK, DIM, dtype=torch.float64),) * 2
    # the voice's prompt, into a cache of one session
    voice_x = rows_of(p)
    voice = tuple(torch.zeros(1, p, HK, DIM, dtype=dtype, device=DEV) for _ in range(2))
    at = torch.arange(p, dtype=torch.int32, device=DEV)
    got = layer(fcv, w, voice_x.to(DEV), tables, at, at, voice, ints([p]))
    want, past = exact_layer(w, voice_x.double(), *tables, at.cpu().long(), zero)
    assert rel_l2(got, want) <= bar
    prefix = dict(prefix_k=voice[0][0], prefix_v=voice[1][0])

    # three requests append their texts
    news, slots = [7, 1, 20], [2, 0, 3]
    caches = tuple(torch.full((4, cap, HK, DIM), float("nan"), dtype=dtype, device=DEV)
                   for _ in range(2))
    xs = [rows_of(n) for n in news]
    pos = torch.cat([p + torch.arange(n) for n in news])
    rows = torch.cat([s * cap + torch.arange(n) for n, s in zip(news, slots)])
    got = layer(fcv, w, torch.cat(xs).to(DEV), tables, pos.int().to(DEV), rows.int().to(DEV), caches,
                ints(news), cu_q=ints([0, 7, 8, 28]), max_q=20, slots=ints(slots), **prefix)
    pasts, first = [], 0
    for x, n in zip(xs, news):
        want, own = exact_layer(w, x.double(), *tables, p + torch.arange(n), past)
        assert rel_l2(got[first:first + n], want) <= bar
        pasts.append(own)
        first += n

    # and two tokens each: eagerly, then the same from a graph captured once and replayed
    state = {"x": torch.zeros(3, WIDTH, dtype=dtype, device=DEV), "pos": ints([0] * 3),
             "rows": ints([-1] * 3), "lengths": ints([0] * 3)}
    slot_t = ints(slots)

    def step():
        return layer(fcv, w, state["x"], tables, state["pos"], state["rows"], caches,
                     state["lengths"], slots=slot_t, max_length=cap, **prefix)

    def feed(x, lengths):
        state["x"].copy_(x)
        state["pos"].copy_(ints([p + n - 1 for n in lengths]))
        state["rows"].copy_(ints([s * cap + n - 1 for n, s in zip(lengths, slots)]))
        state["lengths"].copy_(ints(lengths))

    graph = None
    for i in range(4):
        x = rows_of(3)
        lengths = [n + i + 1 for n in news]
        feed(x, lengths)
        eager = step().clone()
        if graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = step()
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager), f"replay {i}"
        for j in range(3):
            want, pasts[j] = exact_layer(w, x[j:j + 1].double(), *tables,
                                         torch.tensor([p + lengths[j] - 1]), pasts[j])
            assert rel_l2(eager[j:j + 1], want) <= bar, (i, j)


def test_two_streams_and_two_graphs(fcv):
    """Calls in flight on two streams at once, and two captured graphs replayed in turn, give the
    bits of calls one after the other."""
    dtype = torch.bfloat16
    w = weights(dtype)
    g = torch.Generator(device=DEV).manual_seed(9)

    def case(n):
        caches = [torch.randn(n, 700, HK, DIM, generator=g, device=DEV).to(dtype) for _ in range(2)]
        prefix = [torch.randn(900, HK, DIM, generator=g, device=DEV).to(dtype) for _ in range(2)]
        q = torch.randn(n, HQ, DIM, generator=g, device=DEV).to(dtype)
        x = torch.randn(40, WIDTH, generator=g, device=DEV).to(dtype)
        return q, caches, prefix, ints([700 - 3 * i for i in range(n)]), x

    cases = [case(5), case(9)]

    def run(c):
        q, (k, v), (pk, pv), lengths, x = c
        return (fcv.prefix_attention(q, k, v, lengths, prefix_k=pk, prefix_v=pv),
                fcv.fused_linear(fcv.fused_linear(x, w["up"], activation="silu"), w["down"],
                                 residual=x))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(c))
    for i in range(6):
        for o in outs:
            for t in o:
                t.zero_()
        for j in ((0, 1), (1, 0))[i % 2]:
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        if i % 3 == 0:
            run(cases[0])  # eager work between replays
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), i
