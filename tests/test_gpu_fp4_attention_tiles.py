"""``paged_attention_fp4`` by tiles of 128 rows: enough rows that the launch takes them, against the formula in
64 bits (a matrix product a head) and the other kernel's masks."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4_oracle as F
from tests import fp4_bars, lm_bars
from tests.gpu_helpers import say
from tests.test_gpu_fp4_attention import make, run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def compare(out, lse, st, what=""):
    """All rows of a head at once, in 64 bits."""
    q, d, heads = st["q"].double(), st["q"].shape[2], st["q"].shape[1]
    n_kv, scale = st["pages"].shape[1], st["q"].shape[2] ** -0.5
    cu = st["cu_q"].tolist()
    for b, (k, v, at, length) in enumerate(F.cache(st["pages"], d, st["table"], st["lengths"])):
        n, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        if not len(at):
            assert bool((out[rows] == 0).all()) and bool((lse[rows] == -math.inf).all())
            continue
        hidden = at > (length - n + torch.arange(n))[:, None]
        count = (~hidden).sum(1)
        for h in range(heads):
            g = h // (heads // n_kv)
            s = scale * (q[rows, h] @ k[:, g].t())
            size = (scale * (q[rows, h].abs() @ k[:, g].abs().t())).masked_fill(hidden, 0).amax(1)
            s = s.masked_fill(hidden, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0)
            want, mass = p @ v[:, g], p @ v[:, g].abs()
            if st["q"].dtype == torch.bfloat16:
                tol = fp4_bars.attention_one(want, mass, size, count.double(), d, v[:, g].abs().max(),
                                             (p * v[:, g].abs().amax(1)).amax(1))
            else:
                tol = fp4_bars.attention(want, mass, size, count.double(), d, st["q"].dtype)
            lm_bars.assert_within(out[rows, h], want, tol, f"{what} {b} {h}")
            seen = count > 0
            wl = torch.logsumexp(s, 1)
            lm_bars.assert_within(lse[rows, h][seen.to(DEV)], wl[seen],
                                  lm_bars.lse(size, count.double(), d, wl)[seen], f"{what} {b} {h} lse")
            assert bool((lse[rows, h].cpu()[~seen] == -math.inf).all())


# rows of a key head's tile: whole tiles, a last one of few rows, sequences of few; prompts in front
@pytest.mark.parametrize("news,keys,heads,n_kv,d,dtype", [
    ([129] * 16, [129] * 16, 16, 16, 64, torch.bfloat16), ([64] * 40, [200] * 40, 32, 16, 64, torch.float16),
    ([300, 1, 257, 31] * 3, [300, 1000, 700, 95] * 3, 32, 16, 128, torch.bfloat16),
    ([128] * 11, [191] * 11, 48, 48, 128, torch.float16), ([700, 33], [1400, 2000], 64, 64, 64, torch.bfloat16)])
def test_tiles(fcv, news, keys, heads, n_kv, d, dtype):
    say(f"[attend fp4 tiles] {len(news)} x {max(news)} {heads}/{n_kv} x {d} {dtype}")
    st = make(news, keys, heads, n_kv, d, dtype)
    compare(*run(fcv, st, return_lse=True), st, "tiles")


def test_masks_and_pages(fcv):
    """Fewer keys than queries, no keys, missing pages, hidden garbage, bounds that the batch passes."""
    st = make([130, 200, 64, 300], [130, 200, 64, 300], 64, 64, 64, torch.bfloat16, extra_rows=3)
    st["lengths"] = torch.tensor([20, 0, 64, 100000], dtype=torch.int32)
    n = st["pages"].shape[0]
    st["table"][3, 1], st["table"][3, 3] = -1, n
    out, lse = run(fcv, st, return_lse=True, max_q=300, max_length=300)
    compare(out, lse, st, "short")
    st["lengths"] = torch.tensor([130, 180, 40, 290], dtype=torch.int32)
    clean = run(fcv, st, max_q=300)
    d = 64
    for b, length in enumerate(st["lengths"].tolist()):
        if length % 64 == 0:
            continue
        kv = st["pages"][st["table"][b, length // 64]].view(64, -1)
        kv[:, F.PAGE * d:F.PAGE * d + 128].view(64, 64, 2)[:, length % 64:] = 255
        kv[:, F.PAGE * d + 128:][:, length % 64:] = 255
    rows = int(st["cu_q"][-1])
    assert torch.equal(run(fcv, st, max_q=300)[:rows], clean[:rows])
    for max_q, max_length in ((300, 64), (200, 300), (3000, 7)):
        got, lse = run(fcv, st, return_lse=True, max_q=max_q, max_length=max_length)
        compare(got, lse, st, f"{max_q} {max_length}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_of_many_sizes(fcv, dtype):
    """Values whose scales rise and fall over the pages, the type's largest among them, and all of one size."""
    g = torch.Generator().manual_seed(11)
    st = make([260] * 12, [320] * 12, 16, 16, 64, dtype)
    n = st["pages"].shape[0]
    k = torch.randn(n, 16, F.PAGE, 64, generator=g)
    v = torch.randn(n, 16, F.PAGE, 64, generator=g) * 2.0 ** torch.randint(-9, 8, (n, 1, F.PAGE, 1), generator=g)
    v *= 2.0 ** torch.randint(-3, 4, (n, 1, 1, 1), generator=g)
    st["pages"] = fp4_bars.pack(k, v, dtype)
    compare(*run(fcv, st, return_lse=True), st, "many sizes")
    big = 6.0 * 2.0 ** F.LIMITS[dtype][1]
    st["pages"] = fp4_bars.pack(k, torch.sign(v) * big, dtype)
    out, lse = run(fcv, st, return_lse=True)
    compare(out, lse, st, "largest")
    assert bool(out.isfinite().all())


def test_nan_in_place_and_rows_behind(fcv):
    st = make([200] * 16, [200] * 16, 16, 16, 128, torch.float16, extra_rows=4)
    want = run(fcv, st)
    st["pages"][st["table"][2, 1]][3, F.PAGE * 128 + 30 * 4 + 1] = 255  # key 94 of sequence 2, head 3
    a = {k: v.to(DEV) for k, v in st.items()}
    q = a["q"].clone()
    tail = q[3200:].clone()
    got = fcv.paged_attention_fp4(q, a["pages"], a["table"], a["lengths"], cu_q=a["cu_q"], out=q)
    assert torch.equal(got[3200:], tail)
    nan = got[:3200].isnan()
    assert bool(nan[494:600, 3].all()) and int(nan.sum()) == 106 * 128
    same = ~nan
    assert torch.equal(got[:3200][same], want[:3200][same])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("step", [1.0, 1.5, -1.0])
def test_scores_that_rise_page_by_page(fcv, dtype, d, step):
    """Every page's largest score a little above, or below, that of the one before."""
    g = torch.Generator().manual_seed(3)
    st = make([260] * 12, [320] * 12, 16, 16, d, dtype)
    n = st["pages"].shape[0]
    k = torch.randn(n, 16, F.PAGE, d, generator=g) / 4
    v = torch.randn(n, 16, F.PAGE, d, generator=g)
    for b in range(12):
        for i in range(5):
            k[st["table"][b, i], ..., 0] = step * i
    st["pages"] = fp4_bars.pack(k, v, dtype)
    st["q"][..., 0] = d ** 0.5
    compare(*run(fcv, st, return_lse=True), st, f"rising {step}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_values_without_a_scale(fcv, dtype, d):
    """NaN for the rows that see the key, also where its weight vanishes; nothing for the others."""
    st = make([200] * 16, [200] * 16, 16, 16, d, dtype)
    want = run(fcv, st)
    sees = torch.zeros(3200, 16, dtype=torch.bool)
    for b, head, key in ((0, 0, 0), (1, 3, 63), (2, 5, 64), (2, 7, 94), (2, 7, 129), (15, 15, 199), (9, 2, 190)):
        st["pages"][st["table"][b, key // 64], head].view(-1)[-F.PAGE + key % 64] = 255
        sees[200 * b + key:200 * b + 200, head] = True
    got = run(fcv, st)
    assert torch.equal(got.isnan().all(-1).cpu(), sees) and torch.equal(got.isnan().any(-1).cpu(), sees)
    assert torch.equal(got.cpu()[~sees], want.cpu()[~sees])


def test_huge_values_do_not_touch_others(fcv):
    """Values of 2^100 that a row does not see, or sees with a weight of next to nothing; such ones in front of
    the ones that count, behind them and in one page with them."""
    d = 64
    st = make([200] * 16, [330] * 16, 16, 16, d, torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    n = st["pages"].shape[0]
    k = torch.randn(n, 16, F.PAGE, d, generator=g)
    v = torch.randn(n, 16, F.PAGE, d, generator=g)
    k[..., 0] = 0
    st["q"][..., 0] = d ** 0.5
    for b in range(16):
        for key in ((140,), (329,), (131, 200, 330 - 66), tuple(range(192, 256)))[b % 4]:
            v[st["table"][b, key // 64], :, key % 64] *= 2.0 ** 100
            if b % 8 >= 4:
                k[st["table"][b, key // 64], :, key % 64, 0] = -192.0  # a weight of some 2^-277
        if b >= 12:
            for key in (0, 5, 70):
                v[st["table"][b, key // 64], :, key % 64] *= 2.0 ** 110
                k[st["table"][b, key // 64], :, key % 64, 0] = -160.0
    st["pages"] = fp4_bars.pack(k, v, torch.bfloat16)
    compare(*run(fcv, st, return_lse=True), st, "huge")
