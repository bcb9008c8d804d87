"""``paged_attention_fp4`` against its formula in 64 bits: sizes, head layouts, ragged lengths, rows without keys,
missing and shared pages, what lies behind a sequence, captures and refusals."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4_oracle as F
from tests import fp4_bars, lm_bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def make(news, keys, heads, n_kv, d, dtype, seed=0, spare=3, extra_rows=0, q_scale=1.5):
    """q, pages, table, lengths, cu_q of a batch whose pages sit anywhere; -1 behind the last."""
    g = torch.Generator().manual_seed(seed + 31 * sum(keys) + len(keys) + heads)
    counts = [(k + F.PAGE - 1) // F.PAGE for k in keys]
    n = sum(counts) + spare
    ids = torch.randperm(n, generator=g).tolist()
    table = torch.full((len(keys), max(max(counts), 1)), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor([ids.pop() for _ in range(c)], dtype=torch.int32)
    cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32)
    q = (torch.randn(int(cu[-1]) + extra_rows, heads, d, generator=g) * q_scale).to(dtype)
    pages = fp4_bars.random_pages(n, n_kv, d, seed + 1, dtype)
    return dict(q=q, pages=pages, table=table, lengths=torch.tensor(keys, dtype=torch.int32), cu_q=cu)


def run(fcv, st, **kw):
    a = {k: v.to(DEV) for k, v in st.items()}
    return fcv.paged_attention_fp4(a["q"], a["pages"], a["table"], a["lengths"], cu_q=a["cu_q"], **kw)


def check(fcv, st, what="", scale=None, **kw):
    out, lse = run(fcv, st, scale=scale, return_lse=True, **kw)
    compare(out, lse, st, what, scale)
    return out, lse


def compare(out, lse, st, what="", scale=None):
    want, wl, mass, score, keys = F.attention(st["q"], st["pages"], st["table"], st["lengths"],
                                              st["cu_q"], scale)
    rows, d = int(st["cu_q"][-1]), st["q"].shape[2]
    tol = fp4_bars.attention(want, mass, score, keys, d, st["q"].dtype)
    lm_bars.assert_within(out[:rows], want[:rows], tol[:rows], what + " out")
    seen = keys[:rows] > 0
    got = lse[:rows].double().cpu()
    assert bool((got[~seen] == -math.inf).all()) and bool((out[:rows].cpu()[~seen] == 0).all()), what
    lm_bars.assert_within(got[seen], wl[:rows][seen], lm_bars.lse(score, keys, d, wl)[:rows][seen],
                          what + " lse")


HEADS = [(14, 2, 64), (4, 4, 64), (16, 4, 64), (32, 8, 128), (16, 1, 128), (3, 3, 128), (40, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,n_kv,d", HEADS)
def test_single_tokens(fcv, heads, n_kv, d, dtype):
    say(f"[attend fp4] tokens {heads}/{n_kv} x {d} {dtype}")
    keys = [1, 63, 64, 65, 200, 2, 1000]
    check(fcv, make([1] * len(keys), keys, heads, n_kv, d, dtype), "tokens")
    check(fcv, make([1], [3000], heads, n_kv, d, dtype), "one long")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,n_kv,d", HEADS)
def test_several_tokens(fcv, heads, n_kv, d, dtype):
    say(f"[attend fp4] appends {heads}/{n_kv} x {d} {dtype}")
    check(fcv, make([3, 1, 7, 70, 2], [130, 64, 7, 70, 900], heads, n_kv, d, dtype), "appends")


@pytest.mark.parametrize("heads,n_kv,d,dtype", [(14, 2, 64, torch.bfloat16), (8, 2, 128, torch.float16),
                                                (4, 4, 128, torch.bfloat16)])
def test_long_appends(fcv, heads, n_kv, d, dtype):
    say(f"[attend fp4] long appends {heads}/{n_kv} x {d}")
    check(fcv, make([333, 150, 257], [700, 150, 1300], heads, n_kv, d, dtype), "long")


def test_without_cu_q(fcv):
    st = make([2, 2, 2], [70, 2, 300], 8, 2, 64, torch.bfloat16)
    a = {k: v.to(DEV) for k, v in st.items()}
    out, lse = fcv.paged_attention_fp4(a["q"], a["pages"], a["table"], a["lengths"], return_lse=True)
    compare(out, lse, st)


def test_bounds_that_a_batch_passes(fcv):
    """max_q and max_length shape the launch only."""
    st = make([1, 90, 5], [900, 300, 1500], 8, 2, 128, torch.bfloat16)
    for max_q, max_length in ((1, 64), (90, 1500), (1000, 100), (2, 100000), (1, 0)):
        check(fcv, st, f"{max_q} {max_length}", max_q=max_q, max_length=max_length)


def test_rows_without_keys(fcv):
    """Lengths of zero, fewer keys than queries, negative lengths, lengths past the table."""
    st = make([1, 4, 3, 1, 2], [1, 4, 3, 60, 130], 8, 2, 64, torch.float16)
    st["lengths"] = torch.tensor([0, 2, -5, 100000, 130], dtype=torch.int32)
    check(fcv, st, "short")
    st["lengths"].zero_()
    out, lse = run(fcv, st, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_missing_pages(fcv):
    """A page that is negative or past the pool has no keys; the others of the sequence count."""
    st = make([1, 3, 2, 80], [300, 200, 64, 400], 8, 2, 128, torch.bfloat16)
    n = st["pages"].shape[0]
    st["table"][0, 1], st["table"][1, 0], st["table"][2, 0] = -1, n, 2 ** 31 - 1
    st["table"][3, 2], st["table"][3, 6] = -2 ** 31, n + 5
    check(fcv, st, "missing")


def test_shared_pages(fcv):
    """Sequences that share a prompt's pages, and one page twice in a table."""
    st = make([1] * 5, [500, 400, 300, 128, 200], 14, 2, 64, torch.bfloat16)
    st["table"][1:4, :2] = st["table"][0, :2]
    st["table"][4, 1] = st["table"][4, 0]
    check(fcv, st, "shared")


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 60, 3]])
def test_what_lies_behind_the_last_key_is_hidden(fcv, news):
    """Codes and scales behind a sequence's last key, NaN scales among them, do not touch its result; nor do
    pages behind it in the table."""
    st = make(news, [100, 70, 191], 8, 2, 64, torch.bfloat16)
    want, lse0 = check(fcv, st, "clean")
    d = 64
    for b, length in enumerate(st["lengths"].tolist()):
        page = st["pages"][st["table"][b, length // 64]]
        first = length % 64
        kv = page.view(2, -1)
        kv[:, F.PAGE * d // 2:F.PAGE * d].view(2, d // 2, 64)[:, :, first:] = 0x77
        kv[:, :F.PAGE * d // 2].view(2, 64, d // 2)[:, first:] = 0x7f
        kv[:, F.PAGE * d:F.PAGE * d + 128].view(2, 64, 2)[:, first:] = 255
        kv[:, F.PAGE * d + 128:][:, first:] = 255
    out, lse = run(fcv, st, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, lse0)


def test_nan_groups_that_are_seen(fcv):
    """A NaN key or value makes the queries NaN that see it, and no others."""
    for d, part in ((64, "key"), (128, "value")):
        st = make([6, 1], [100, 70], 4, 2, d, torch.float16)
        clean, _ = check(fcv, st)
        at = 97  # seen by the last three of the first sequence's queries (keys 94 .. 99 are theirs)
        page = st["pages"][st["table"][0, at // 64]][1]
        if part == "key":
            page[F.PAGE * d + (at % 64) * (d // 32)] = 255
        else:
            page[F.PAGE * (d + d // 32) + at % 64] = 255
        out = run(fcv, st).cpu()
        nan = out.isnan()
        assert bool(nan[3:6, 2:].all()), part
        assert torch.equal(out[:3], clean[:3].cpu()) and torch.equal(out[:, :2], clean[:, :2].cpu())
        assert torch.equal(out[6:], clean[6:].cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_extreme_values_and_scores(fcv, dtype):
    """The type's largest values, keys of many sizes, and scores of hundreds."""
    lo, hi = F.LIMITS[dtype]
    g = torch.Generator().manual_seed(3)
    st = make([2, 1], [150, 64], 4, 2, 64, dtype)
    n = st["pages"].shape[0]
    k = torch.randn(n, 2, 64, 64, generator=g)
    v = torch.full((n, 2, 64, 64), 6.0 * 2.0 ** hi if dtype == torch.bfloat16 else 49152.0)
    st["pages"] = fp4_bars.pack(k, v, dtype)
    out, _ = check(fcv, st, "largest values")
    assert bool(out.isfinite().all())
    v = torch.randn(n, 2, 64, 64, generator=g) * 2.0 ** torch.randint(-12, 9, (n, 2, 64, 1), generator=g)
    st["pages"] = fp4_bars.pack(k * 8, v, dtype)
    check(fcv, st, "scores of hundreds", scale=1.0)
    check(fcv, st, "one scale", scale=1e-4)


def test_rows_behind_the_last_sequence_stay(fcv):
    for news in ([1, 1], [40, 60]):
        st = make(news, [100, 70], 8, 2, 64, torch.bfloat16, extra_rows=5)
        rows = sum(news)
        out = torch.full(st["q"].shape, 3.0, dtype=torch.bfloat16, device=DEV)
        run(fcv, st, out=out)
        assert bool((out[rows:] == 3).all())
        assert torch.equal(out[:rows], run(fcv, st)[:rows])


def test_strides_and_in_place(fcv):
    st = make([1, 30, 2], [100, 130, 700], 8, 2, 128, torch.float16)
    want = run(fcv, st)
    a = {k: v.to(DEV) for k, v in st.items()}
    t = a["q"].shape[0]
    wide = torch.zeros(8, t, 144, dtype=torch.float16, device=DEV)       # heads before tokens
    q = wide.transpose(0, 1)[:, :, 8:136]
    q.copy_(a["q"])
    n, h, size = a["pages"].shape
    pool = torch.zeros(2, h, n, size + 16, dtype=torch.uint8, device=DEV)
    pages = pool[1].transpose(0, 1)[:, :, :size]
    pages.copy_(a["pages"])
    table = torch.full((3, a["table"].shape[1] + 5), 9, dtype=torch.int32, device=DEV)
    table[:, :a["table"].shape[1]] = a["table"]
    kw = dict(cu_q=a["cu_q"], max_length=700)
    got = fcv.paged_attention_fp4(q, pages, table[:, :a["table"].shape[1]], a["lengths"], **kw)
    assert torch.equal(got, want)
    got = fcv.paged_attention_fp4(q, pages, table[:, :a["table"].shape[1]], a["lengths"], out=q, **kw)
    assert torch.equal(got, want) and bool((wide[:, :, :8] == 0).all()) and bool((wide[:, :, 136:] == 0).all())


def test_a_sequence_does_not_depend_on_its_batch(fcv):
    """Other sequences' contents do not change a result's bits; runs are alike."""
    st = make([1, 5, 1], [900, 300, 77], 8, 2, 64, torch.bfloat16)
    want = run(fcv, st, max_q=5, max_length=1000)
    again = run(fcv, st, max_q=5, max_length=1000)
    assert torch.equal(want, again)
    st["q"][1:6] *= 2
    got = run(fcv, st, max_q=5, max_length=1000)
    assert torch.equal(got[0], want[0]) and torch.equal(got[6], want[6])


def test_captured(fcv):
    """Replays with new lengths, pages and queries; two graphs take turns with eager calls."""
    st = {k: v.to(DEV) for k, v in make([1] * 4, [700, 60, 300, 9], 14, 2, 64, torch.bfloat16).items()}

    def call():
        return fcv.paged_attention_fp4(st["q"], st["pages"], st["table"], st["lengths"],
                                       cu_q=st["cu_q"], max_q=1, max_length=2000, return_lse=True)

    call()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for step in range(4):
        st["lengths"].add_(1)
        st["q"].mul_(0.9)
        g, got = graphs[step % 2]
        g.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), step


def test_two_streams(fcv):
    sts = [{k: v.to(DEV) for k, v in make([1] * 3, [1500, 60, 300], 8, 2, 128, torch.bfloat16, seed=s).items()}
           for s in range(2)]

    def call(st):
        return fcv.paged_attention_fp4(st["q"], st["pages"], st["table"], st["lengths"], cu_q=st["cu_q"])

    want = [call(st) for st in sts]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(sts[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_many_sequences(fcv):
    g = torch.Generator().manual_seed(9)
    keys = torch.randint(1, 400, (150,), generator=g).tolist()
    check(fcv, make([1] * 150, keys, 4, 2, 64, torch.float16), "many")


def test_no_rows(fcv):
    st = make([1, 1], [10, 20], 8, 2, 64, torch.bfloat16)
    st["q"], st["cu_q"] = st["q"][:0], torch.zeros(3, dtype=torch.int32)
    out, lse = run(fcv, st, return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


def test_refusals(fcv):
    st = {k: v.to(DEV) for k, v in make([1, 1], [100, 70], 8, 2, 64, torch.bfloat16).items()}

    def call(**kw):
        a = {**st, **{k: v for k, v in kw.items() if k in st}}
        rest = {k: v for k, v in kw.items() if k not in st}
        return fcv.paged_attention_fp4(a["q"], a["pages"], a["table"], a["lengths"], cu_q=a["cu_q"], **rest)

    for bad, match in [
        (dict(q=st["q"][:, :7]), "multiple of 2"), (dict(q=st["q"].float()), "float16 or bfloat16"),
        (dict(q=st["q"][:, :, :32]), "heads, 64"), (dict(pages=st["pages"][..., :100]), "pages must be"),
        (dict(table=st["table"].long()), "int32"), (dict(table=st["table"][:1]), "2 rows"),
        (dict(table=st["table"].t().contiguous().t()), "contiguous"),
        (dict(lengths=st["lengths"].long()), "int32"), (dict(cu_q=st["cu_q"][:2]), "int32"),
        (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(max_q=0), "max_q"),
        (dict(max_length=-1), "max_length"), (dict(out=st["q"][:1]), "out must be"),
        (dict(out=st["q"][:1].expand(2, -1, -1)), "expanded"), (dict(lengths=st["lengths"][:0]), "empty"),
        (dict(max_q=1 << 40), "range"), (dict(pages=st["pages"].cpu()), "pages must be"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**bad)
    buf = torch.zeros(3, 8, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="out overlaps q"):
        call(q=buf[:2], out=buf[1:])


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 1, 9], [700, 300, 600]])
@pytest.mark.parametrize("d", [64, 128])
def test_queries_without_numbers_and_without_pages(fcv, news, d):
    """A padded slot: no page behind its length, and whatever its queries hold."""
    st = make(news, [1000] * 3, 16, 4, d, torch.bfloat16)
    clean = run(fcv, st)
    st["table"][1] = -1
    first, end = st["cu_q"][1:3].tolist()
    st["q"][first:end, 0::2] = math.nan
    st["q"][first:end, 1::2] = math.inf
    out, lse = run(fcv, st, return_lse=True)
    assert bool((out[first:end] == 0).all()) and bool((lse[first:end] == -math.inf).all())
    assert torch.equal(out[:first], clean[:first]) and torch.equal(out[end:], clean[end:])


@pytest.mark.parametrize("batch,heads,n_kv,d", [(300, 4, 1, 64), (70, 16, 4, 64), (1100, 2, 1, 64), (40, 32, 8, 128)])
def test_sequences_of_many_lengths(fcv, batch, heads, n_kv, d):
    """Batches that are taken longest first: equal lengths among them, none, one past the table, and more
    sequences than are ordered together."""
    say(f"[attend fp4] order {batch} {heads}/{n_kv} x {d}")
    g = torch.Generator().manual_seed(batch)
    keys = torch.randint(0, 60, (batch,), generator=g)
    keys[0], keys[batch // 2], keys[-1] = 2300, 2300, 2310
    keys[3:20:3] = 0
    st = make([1] * batch, keys.tolist(), heads, n_kv, d, torch.bfloat16)
    check(fcv, st, "many lengths")
    st["lengths"][batch // 3], st["lengths"][5] = 1 << 30, -7
    check(fcv, st, "bounds", max_length=2310)


def test_ordered_sequences_in_ranges(fcv):
    """Longest first, their pages in ranges: few long sequences among short ones, new tokens of one to five."""
    g = torch.Generator().manual_seed(17)
    news = torch.randint(1, 6, (32,), generator=g).tolist()
    keys = torch.randint(5, 300, (32,), generator=g).tolist()
    keys[7], keys[20], keys[31] = 4500, 4401, 4500
    st = make(news, keys, 16, 8, 64, torch.float16)
    out, lse = check(fcv, st, "ranges", max_q=5)
    again = run(fcv, st, max_q=5, max_length=300)  # a bound that the long ones pass
    compare(again, lse, st, "passed")
