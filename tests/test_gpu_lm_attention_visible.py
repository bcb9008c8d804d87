"""``prefix_attention`` of values that are not finite and that a query sees: every visible key has a
weight above zero, so an infinity among the values is what the row gets (NaN for NaN and for both
infinities), wherever its key lies and however small the weight."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_helpers import say
from tests.test_gpu_lm_attention import check, make

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 40, 200])
def test_in_a_tile_that_is_seen_whole(fcv, n, dim, dtype):
    """Several dims each, so that both signs of a weight's rounding error occur."""
    say(f"[visible] full tiles, {n} new tokens x {dim} {dtype}")
    a = make([n, 1], [n + 300, 70], 130, 6, 2, dim, dtype)
    slot = a["slots"].tolist()
    for key in range(0, 96, 7):
        a["v_cache"][slot[0], key, 0, key % dim] = INF if key % 2 else -INF
        a["prefix_v"][key, 1, key % 64] = -INF if key % 2 else INF
    a["v_cache"][slot[1], 3, 0, 9] = NAN
    check(fcv, a, "full tiles", max_q=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [1, 50, 129, 901, 2304])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_in_the_last_key_of_the_prompt(fcv, n, prefix, dim, dtype):
    say(f"[visible] last of {prefix}, {n} new tokens x {dim} {dtype}")
    a = make([n, 1, 1], [n + 5, 9, 0], prefix, 6, 2, dim, dtype)
    a["lengths"][2] = 0
    a["prefix_v"][-1, 0, 5] = INF
    a["prefix_v"][-1, 0, 6] = -INF
    a["prefix_v"][-1, 1, 7] = NAN
    check(fcv, a, "last key", max_q=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_behind_weights_that_vanish(fcv, n, dim, dtype):
    """One own key far above all others (by 2^70, then by 2^250): their weights round to zero in a
    tile, in a wave, and where parts are joined."""
    for prefix in (50, 2304):
        for size in (20.0, 40.0):
            say(f"[visible] behind weights of 0, {prefix} + {n} x {dim} {dtype}")
            a = make([n, 2], [n + 600, 400], prefix, 6, 2, dim, dtype)
            slot = a["slots"].tolist()
            a["q"][:] = 0
            a["q"][..., 0] = size
            for t in ("k_cache", "prefix_k"):
                a[t][..., 0] = 0
            for s, key in zip(slot, (400, 130)):
                a["k_cache"][s, key, :, 0] = size * (dim / 64) ** 0.5
            a["prefix_v"][prefix // 2, 0, 3] = INF
            a["prefix_v"][prefix // 3, 1, 5] = -INF
            a["v_cache"][slot[0], 7, 0, 10] = -INF
            a["v_cache"][slot[0], n + 599, 1, 11] = INF
            a["v_cache"][slot[1], 300, 1, 12] = NAN
            check(fcv, a, "vanishing", max_q=n, max_length=max(n + 600, 400))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [3, 40, 200])
def test_both_infinities_meet_where_a_row_sees_both(fcv, n, dtype):
    """Of the new tokens the first sees +inf alone, the last sees -inf too; then the other dim NaN."""
    for dim in (64, 128):
        say(f"[visible] both, {n} new tokens x {dim} {dtype}")
        a = make([n, 1], [n + 20, 9], 33, 6, 2, dim, dtype)
        slot = int(a["slots"][0])
        a["prefix_v"][4, 0, 2] = INF
        a["v_cache"][slot, n + 19, 0, 2] = -INF
        a["v_cache"][slot, 19 + n // 2, 1, 3] = INF
        a["v_cache"][slot, n + 18, 1, 3] = NAN
        got, _ = check(fcv, a, "both", max_q=n)
        assert (got[:n - 1, :3, 2] == INF).all() and got[n - 1, :3, 2].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_q", [1, 50])
def test_in_tiles_taken_in_turn(fcv, max_q, dim, dtype):
    """Sequences that pass the bound on their new tokens: a workgroup has several row tiles, each of
    which looks for itself."""
    say(f"[visible] several tiles, bound {max_q} x {dim} {dtype}")
    a = make([300, 1, 90], [320, 9, 700], 70, 6, 2, dim, dtype)
    slot = a["slots"].tolist()
    for key in (5, 77, 150, 260, 319):
        a["v_cache"][slot[0], key, 0, key % dim] = INF
        a["v_cache"][slot[0], key, 1, key % 64] = NAN
    a["v_cache"][slot[2], 650, 0, 1] = -INF
    check(fcv, a, "several", max_q=max_q, max_length=700)
    a["prefix_v"][69, 0, 2] = -INF
    check(fcv, a, "and the prompt", max_q=max_q, max_length=60)


@pytest.mark.parametrize("n", [1, 40, 200])
def test_a_query_that_is_not_finite_stays_alone(fcv, n):
    for dim in (64, 128):
        a = make([n, 3], [n + 300, 70], 130, 6, 2, dim, torch.bfloat16)
        want = fcv.prefix_attention(**a, max_q=n)
        a["q"][0, 1, 3] = NAN
        a["v_cache"][int(a["slots"][0]), 2, 0, 4] = INF
        got = fcv.prefix_attention(**a, max_q=n)
        assert got[0, 1].isnan().all()                     # the infinity does not stand over its NaN
        rest = torch.ones_like(got, dtype=torch.bool)
        rest[0, 1] = False
        rest[:n, :3, 4] = False
        assert torch.equal(got[rest], want[rest])
        assert (got[1:n, :3, 4] == INF).all() and got[0, [0, 2], 4].tolist() == [INF, INF]
