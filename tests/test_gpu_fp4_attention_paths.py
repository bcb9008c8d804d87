"""``paged_attention_fp4`` by every combination of tile, key ranges and order, and with tiles that take turns:
against the formula in 64 bits, with a missing page and values of many sizes, and with a value without a scale."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4_oracle as F
from tests import fp4_bars
from tests.gpu_helpers import say
from tests.test_gpu_fp4_attention import make, run
from tests.test_gpu_fp4_attention_weights import compare

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (rows of a tile, in ranges, longest first): new tokens and keys of every sequence, heads, key heads, head dim,
# max_q, max_length; new tokens or keys past the bounds where tiles take turns and the last range is longer
CASES = {
    (8, False, False): ([1, 2, 1, 1, 2], [300, 64, 65, 1, 200], 8, 4, 64, 2, 320),
    (8, True, False): ([1, 1, 2, 9], [3000, 70, 1500, 2000], 8, 4, 64, 2, 3000),
    (8, False, True): ([1] * 32, [2500, 2400, 2500] + list(range(40, 1780, 60)), 32, 16, 64, 1, 2560),
    (8, True, True): ([1] * 24, [4500, 17, 4400] + list(range(20, 1280, 60)), 16, 8, 128, 1, 4500),
    (16, False, False): ([20, 3, 40, 1], [300, 200, 44, 77], 16, 4, 64, 20, 320),
    (16, True, False): ([20, 33, 7], [3000, 700, 1900], 16, 4, 128, 20, 2500),
    (16, False, True): ([20, 5, 1, 31, 20, 8, 20, 2, 16, 9], [2300, 90, 1200, 200, 2300, 64, 30, 800, 130, 500],
                        32, 8, 64, 20, 2300),
    (16, True, True): ([20, 5, 1, 31, 20, 8, 20, 2, 16, 9, 3, 6],
                       [4200, 90, 1200, 200, 2300, 64, 30, 800, 130, 500, 4190, 7], 16, 4, 64, 20, 4200),
    (128, False, False): ([300, 1, 257, 400], [300, 1000, 700, 450], 32, 8, 128, 300, 1000),
    (128, True, False): ([256, 40, 300, 1], [7000, 100, 1300, 3000], 32, 8, 128, 256, 6800),
    (128, False, True): ([1100, 40, 200, 1, 300, 64, 128, 33], [2100, 2090, 500, 1700, 300, 64, 1200, 100], 16, 4, 128,
                         1100, 2100),
    (128, True, True): ([256, 1, 700, 40, 256, 100, 3, 64, 130], [7000, 2500, 900, 4100, 256, 6990, 40, 64, 1000],
                        16, 4, 128, 256, 7000),
    # heads of 64, whose tiles have to be more
    (128, True, True, 64): ([256, 1, 400] + [5] * 17, [7000, 3500, 5000] + list(range(5, 600, 35)), 16, 4, 64, 256, 7000),
    (128, False, True, 64): ([256, 1, 600] + [5] * 17, [3000, 2500, 2900] + list(range(5, 600, 35)), 16, 4, 64, 256, 3000),
}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("path", CASES, ids=str)
def test_paths(fcv, path, dtype):
    say(f"[attend fp4 paths] {path} {dtype}")
    news, keys, heads, n_kv, d, max_q, max_length = CASES[path]
    group, bounds = heads // n_kv, dict(max_q=max_q, max_length=max_length)
    st = make(news, keys, heads, n_kv, d, dtype)
    g = torch.Generator().manual_seed(13)
    n = st["pages"].shape[0]
    k = torch.randn(n, n_kv, F.PAGE, d, generator=g)
    v = torch.randn(n, n_kv, F.PAGE, d, generator=g) * 2.0 ** torch.randint(-9, 8, (n, n_kv, F.PAGE, 1), generator=g)
    st["pages"] = fp4_bars.pack(k, v, dtype)
    long = max(range(len(keys)), key=lambda b: keys[b] - 65 * (news[b] > 1))
    if keys[long] > 320:
        st["table"][long, 1] = -1  # a page whose keys do not count
    out, lse = run(fcv, st, return_lse=True, **bounds)
    compare(out, lse, st, str(path))
    again, lse2 = run(fcv, st, return_lse=True, **bounds)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # values without a scale: in the first range, in a later one, next to a sequence's last key
    sees = torch.zeros(out.shape[:2], dtype=torch.bool)
    for b, key, h in ((long, 5, 0), (long, keys[long] - 1, n_kv - 1), (len(keys) - 1, keys[-1] // 2, 1)):
        st["pages"][st["table"][b, key // F.PAGE], h].view(-1)[-F.PAGE + key % F.PAGE] = 255
        first = int(st["cu_q"][b]) + max(key - (keys[b] - news[b]), 0)
        sees[first:int(st["cu_q"][b + 1]), h * group:(h + 1) * group] = True
    got = run(fcv, st, **bounds)
    assert torch.equal(got.isnan().all(-1).cpu(), sees) and torch.equal(got.isnan().any(-1).cpu(), sees)
    assert torch.equal(got.cpu()[~sees], out.cpu()[~sees])


@pytest.mark.parametrize("d", [64, 128])
def test_pages_far_apart_by_large_tiles(fcv, d):
    """Pages and heads gigabytes apart, by tiles of 128 rows: as over a dense pool."""
    hk, hq, n, batch, tokens = 2, 8, 6, 33, 300
    g = torch.Generator().manual_seed(d)
    dense = fp4_bars.random_pages(n, hk, d, d).to(DEV)
    size = dense.shape[2]
    flat = torch.empty(5 * 2 ** 30 + 2 ** 29 + size, dtype=torch.uint8, device=DEV)
    far = flat.as_strided((n, hk, size), (2 ** 30, 2 ** 29, 1))
    far.copy_(dense)
    q = torch.randn(batch * tokens, hq, d, generator=g).to(DEV, torch.bfloat16)
    table = torch.stack([torch.randperm(n, generator=g) for _ in range(batch)]).int().to(DEV)
    lengths = (n * F.PAGE - torch.arange(batch)).int().to(DEV)
    got = [fcv.paged_attention_fp4(q, pool, table, lengths, return_lse=True) for pool in (dense, far)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
