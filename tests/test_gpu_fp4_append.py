"""``qk_norm_rope_fp4`` and ``read_fp4_pages`` against their formulas in 64 bits: the queries within roundings,
the appended numbers exactly."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4_oracle as F
from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def make(tokens, hq, hk, d, dtype, seed=0, rope=None, normed=False, side=None, n_pages=None, table=600):
    g = torch.Generator().manual_seed(seed + tokens + 17 * hq)
    rope = d if rope is None else rope
    n_pages = n_pages or tokens // F.PAGE + 3
    angle = torch.rand(table, rope // 2, generator=g) * 6.28
    rows = torch.randperm(n_pages * F.PAGE, generator=g)[:tokens].int()
    st = dict(qkv=torch.randn(tokens, (hq + 2 * hk) * d, generator=g).to(dtype),
              positions=torch.randint(0, table, (tokens,), generator=g).int(), cos=angle.cos(),
              sin=angle.sin(), rows=rows,
              qw=(1 + 0.2 * torch.randn(d, generator=g)).to(side or dtype) if normed else None,
              kw=(1 + 0.2 * torch.randn(d, generator=g)).to(side or dtype) if normed else None,
              pages=torch.randint(0, 254, (n_pages, hk, F.PAGE * (d + d // 32 + 1)), generator=g,
                                  dtype=torch.uint8))
    return {k: v if v is None else v.to(DEV) for k, v in st.items()}


def append(fcv, st, hq, **kw):
    return fcv.qk_norm_rope_fp4(st["qkv"], st["positions"], st["cos"], st["sin"], st["pages"], st["rows"],
                                n_heads=hq, q_weight=st["qw"], k_weight=st["kw"], **kw)


def want(st, hq, hk, d, eps, interleaved):
    """(q, size of q's terms, keys' numbers, values' numbers)"""
    x = st["qkv"].cpu().view(-1, hq + 2 * hk, d)
    at = st["positions"].long().cpu().clamp(0, st["cos"].shape[0] - 1)
    c, s = st["cos"].cpu()[at], st["sin"].cpu()[at]
    q, size = O.norm_rope(x[:, :hq], st["qw"], eps, c, s, interleaved)
    k, _ = O.norm_rope(x[:, hq:hq + hk], st["kw"], eps, c, s, interleaved)
    dtype = st["qkv"].dtype
    return q, size, F.quantized(k, dtype, 32), F.quantized(x[:, hq + hk:].double(), dtype)


def check(fcv, st, hq, hk, d, eps=1e-6, interleaved=False, what=""):
    before = st["pages"].clone()
    q = append(fcv, st, hq, eps=eps, interleaved=interleaved)
    y, size, k, v = want(st, hq, hk, d, eps, interleaved)
    dtype = st["qkv"].dtype
    bars.assert_within(q, y, bars.norm_rope(y, size, d, st["qw"] is not None, dtype), what + " q")
    rows = st["rows"].long().cpu()
    good = (rows >= 0) & (rows < st["pages"].shape[0] * F.PAGE)
    pk, pv = F.split(st["pages"], d)
    page, place = rows[good] // F.PAGE, rows[good] % F.PAGE
    for got, w, name in ((pk[page, :, place], k[good], "keys"), (pv[page, :, place], v[good], "values")):
        same = (got == w) | (got.isnan() & w.isnan())
        assert bool(same.all()), f"{what} {name}: {int((~same).sum())} numbers differ"
    # nothing else was written
    k0, v0 = F.split(before, d)
    pk[page, :, place], pv[page, :, place] = k0[page, :, place], v0[page, :, place]
    assert torch.equal(pk.nan_to_num(7.7), k0.nan_to_num(7.7))
    assert torch.equal(pv.nan_to_num(7.7), v0.nan_to_num(7.7))
    # and the reader gives the numbers in the type
    rk, rv = fcv.read_fp4_pages(st["pages"], st["rows"], dtype=dtype)
    for got, w in ((rk, k), (rv, v)):
        w = torch.where(good[:, None, None], w, torch.zeros_like(w)).to(dtype)
        same = (got.cpu() == w) | (got.cpu().isnan() & w.isnan())
        assert bool(same.all()), what
    return q


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hq,hk,d,rope", [
    (1, 14, 2, 64, 64), (3, 4, 4, 64, 32), (64, 32, 8, 128, 128), (67, 8, 1, 128, 64), (130, 3, 3, 64, 16),
    (5, 6, 2, 128, 96), (33, 2, 1, 128, 16), (9, 5, 5, 64, 48), (300, 12, 12, 128, 112)])
def test_sizes(fcv, tokens, hq, hk, d, rope, dtype, normed, interleaved):
    say(f"[append fp4] {tokens} x {hq}/{hk} x {d} rope {rope} {dtype} {normed} {interleaved}")
    st = make(tokens, hq, hk, d, dtype, rope=rope, normed=normed)
    check(fcv, st, hq, hk, d, interleaved=interleaved)


def test_fp32_weights_and_eps(fcv):
    for dtype in (torch.bfloat16, torch.float16):
        st = make(40, 4, 2, 64, dtype, normed=True, side=torch.float32)
        check(fcv, st, 4, 2, 64, eps=1e-2)
        st["qkv"][7] = 0
        check(fcv, st, 4, 2, 64, eps=1e-6)


def test_a_prefill_in_order(fcv):
    """Tokens one behind the other: whole pages, from the middle of one."""
    say("[append fp4] prefill")
    for first, d in ((0, 64), (37, 128)):
        st = make(1000, 4, 2, d, torch.bfloat16, normed=True, n_pages=20)
        ids = torch.randperm(20, generator=torch.Generator().manual_seed(1))[:18]
        at = torch.arange(first, first + 1000)
        st["rows"] = (ids[at // 64] * 64 + at % 64).int().to(DEV)
        check(fcv, st, 4, 2, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_on_borders(fcv, dtype):
    """Position 0 rotates by nothing: every element is its own, with ties and group maxima on the border."""
    st = make(8, 1, 1, 64, dtype)
    st["cos"][0], st["sin"][0] = 1, 0
    st["positions"].zero_()
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x = torch.zeros(8, 3, 64)
    for t in range(8):
        scale = 2.0 ** (2 * t - 8)
        x[t, :, :8] = grid * scale
        x[t, :, 32:40] = -grid * scale
        x[t, :, 9] = (7.0 if t % 2 else 6.96875) * scale
        x[t, 1:, 20] = 1e-4 * scale
        x[t, 1:, 63] = 8.0 * scale if t == 3 else 0
    st["qkv"] = x.reshape(8, -1).to(dtype).to(DEV)
    check(fcv, st, 1, 1, 64)


def test_values_that_are_not_finite_and_extremes(fcv):
    for dtype in (torch.bfloat16, torch.float16):
        big = torch.finfo(dtype).max
        st = make(10, 2, 2, 64, dtype)
        x = st["qkv"].view(10, 6, 64)
        st["cos"][0], st["sin"][0] = 1, 0
        st["positions"].zero_()
        x[0, 2, 40], x[1, 5, 3], x[2, 3, 10] = math.inf, math.nan, -math.inf
        x[3, 4] = math.inf
        x[4, 2:], x[5, 2:, ::2] = big, -big
        x[6, 2:] = 0
        x[7, 2:] = torch.finfo(dtype).tiny
        x[:, :2] = 1
        before = st["pages"].clone()
        append(fcv, st, 2)
        k, v = fcv.read_fp4_pages(st["pages"], st["rows"], dtype=dtype)
        # 0 times an infinite sine's partner is NaN: a key's pair of an infinity is one, its group is
        wk = F.quantized(x[:, 2:4].double().cpu() * 1, dtype, 32)
        partner = x[:, 2:4].double().cpu().roll(32, -1)
        wk[((partner * 0).isnan()).unflatten(-1, (2, 32)).any(-1).repeat_interleave(32, -1)] = math.nan
        wv = F.quantized(x[:, 4:].double().cpu(), dtype)
        for got, w in ((k, wk), (v, wv)):
            w = w.to(dtype)
            assert bool(((got.cpu() == w) | (got.cpu().isnan() & w.isnan())).all()), dtype
        assert not torch.equal(before, st["pages"])


def test_large_and_small_heads_are_normed(fcv):
    """Squares of bf16's largest values pass fp32, those of its smallest vanish there."""
    st = make(6, 2, 2, 128, torch.bfloat16, normed=True)
    x = st["qkv"].view(6, 6, 128)
    x[0] *= 1e36
    x[1] *= 1e-36
    x[2, :, ::3] = 3e38
    check(fcv, st, 2, 2, 128, eps=0.0)


def test_rows_and_positions_outside(fcv):
    """Negative rows, rows past the pool: nothing is written; positions outside the tables are clipped."""
    st = make(20, 4, 2, 64, torch.float16)
    st["rows"][::3] = -1
    st["rows"][1::3] = torch.tensor([st["pages"].shape[0] * 64, 2 ** 31 - 1, -2 ** 31, -64, -63, 1 << 20, 1 << 28])[:7].int().to(DEV)
    st["positions"][4], st["positions"][5] = -5, 100000
    check(fcv, st, 4, 2, 64)


def test_strides(fcv):
    """Wide rows of qkv and of the queries, a pool whose heads come before its pages, a layer of a pool."""
    st = make(70, 6, 2, 64, torch.bfloat16, normed=True)
    ref = {k: v.clone() if v is not None else None for k, v in st.items()}
    q = check(fcv, ref, 6, 2, 64)
    wide = torch.zeros(70, st["qkv"].shape[1] + 24, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:8 + st["qkv"].shape[1]] = st["qkv"]
    st["qkv"] = wide[:, 8:8 + st["qkv"].shape[1]]
    n, h, size = st["pages"].shape
    pool = torch.zeros(3, h, n + 1, size + 32, dtype=torch.uint8, device=DEV)
    pages = pool[1].transpose(0, 1)[:n, :, :size]
    pages.copy_(st["pages"])
    st["pages"] = pages
    out = torch.zeros(70, 8, 64, dtype=torch.bfloat16, device=DEV)
    got = append(fcv, st, 6, out=out[:, 1:7])
    assert torch.equal(got, q) and bool((out[:, 0] == 0).all()) and bool((out[:, 7] == 0).all())
    assert torch.equal(st["pages"], ref["pages"])
    assert int(pool[0].sum()) + int(pool[2].sum()) + int(pool[1, :, n].sum()) == 0


def test_queries_in_place(fcv):
    """The queries' own columns of qkv as the output: keys and values read theirs."""
    for d, hq, hk in ((64, 6, 2), (128, 4, 4)):
        st = make(130, hq, hk, d, torch.bfloat16, normed=True)
        ref = {k: v.clone() for k, v in st.items()}
        want = append(fcv, ref, hq)
        got = append(fcv, st, hq, out=st["qkv"].view(130, hq + 2 * hk, d)[:, :hq])
        assert torch.equal(got, want) and torch.equal(st["pages"], ref["pages"])
        assert torch.equal(st["qkv"][:, hq * d:], ref["qkv"][:, hq * d:])


def test_captured_and_no_tokens(fcv):
    st = make(16, 4, 2, 128, torch.bfloat16, normed=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = append(fcv, st, 4)
    for seed in range(3):
        new = make(16, 4, 2, 128, torch.bfloat16, seed=seed, normed=True)
        for name in ("qkv", "positions", "rows"):
            st[name].copy_(new[name])
        st["pages"].zero_()
        graph.replay()
        new["pages"].zero_()
        new |= {"cos": st["cos"], "sin": st["sin"], "qw": st["qw"], "kw": st["kw"]}
        want_q = append(fcv, new, 4)
        assert torch.equal(q, want_q) and torch.equal(st["pages"], new["pages"])
    st["qkv"], st["rows"], st["positions"] = st["qkv"][:0], st["rows"][:0], st["positions"][:0]
    assert append(fcv, st, 4).shape == (0, 4, 128)
    assert fcv.read_fp4_pages(st["pages"], st["rows"], dtype=torch.float16)[0].shape == (0, 2, 128)


def test_refusals(fcv):
    st = make(4, 4, 2, 64, torch.float16, normed=True)

    def call(**kw):
        a = {**st, **{k: v for k, v in kw.items() if k in st}}
        rest = {k: v for k, v in kw.items() if k not in st}
        return append(fcv, a, rest.pop("hq", 4), **rest)

    flat = torch.zeros(st["pages"].numel() + 4096, dtype=torch.uint8, device=DEV)
    over = flat[:st["pages"].numel()].view(st["pages"].shape)
    for bad, match in [
        (dict(hq=3), "qkv must be"), (dict(pages=st["pages"][..., :4000]), "pages must be"),
        (dict(pages=st["pages"].int()), "pages must be"), (dict(pages=st["pages"].cpu()), "pages must be"),
        (dict(rows=st["rows"].long()), "int32"), (dict(positions=st["positions"][:3]), "int32"),
        (dict(kw=None), "together"), (dict(cos=st["cos"].half()), "float32 table"),
        (dict(cos=st["cos"][:, :4].contiguous(), sin=st["sin"][:, :4].contiguous()), "rope_dim"),
        (dict(out=st["qkv"].view(4, 8, 64)[:, 1:5]), "out overlaps qkv"),
        (dict(pages=over, out=over.view(-1)[:2048].view(torch.float16).view(4, 4, 64)), "out overlaps pages"),
        (dict(pages=st["pages"][:1].expand(5, -1, -1)), "none over another"),
        (dict(eps=-1.0), "eps"), (dict(qkv=st["qkv"].float()), "float16 or bfloat16"),
        (dict(pages=flat[8:8 + st["pages"].numel()].view(st["pages"].shape)), "16-byte"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**bad)
    for bad, match in [((st["pages"], st["rows"].long(), torch.float16), "int32"),
                       ((st["pages"], st["rows"], torch.float32), "float16 or bfloat16"),
                       ((st["pages"].cpu(), st["rows"], torch.float16), "GPU")]:
        with pytest.raises(ValueError, match=match):
            fcv.read_fp4_pages(bad[0], bad[1], dtype=bad[2])
    with pytest.raises(ValueError, match="head dim"):
        fcv.new_fp4_pages(4, 2, 96)
    assert fcv.new_fp4_pages(4, 2, 64, layers=3).shape == (3, 4, 2, 4288)
