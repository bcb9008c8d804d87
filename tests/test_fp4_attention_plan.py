"""How a call of the 4-bit attention is launched: the GPU tests' cases reach every combination of tile, ranges and
order, and tiles that take turns."""

from __future__ import annotations

import ctypes

import pytest

from tests.test_gpu_fp4_attention_paths import CASES

BIG = 1 << 40


def plan(fcv, news, keys, heads, n_kv, d, max_q, max_length, **kw):
    """Rows of a tile, tiles, ranges, whether the longest come first."""
    size = 64 * (d + d // 32 + 1)
    width = max((k + 63) // 64 for k in keys)
    base = dict(q=BIG, pages=BIG, table=BIG, lengths=BIG, cu_q=BIG, out=BIG, q_row=heads * d, q_head=d,
                out_row=heads * d, out_head=d, page_stride=n_kv * size, head_stride=size, table_row=width,
                tokens=sum(news), batch=len(news), n_heads=heads, n_kv_heads=n_kv, head_dim=d, n_pages=1000,
                max_pages=width, max_q=max_q, max_length=max_length, dtype=1, scale=0.125)
    base.update(kw)
    got = [ctypes.c_int32() for _ in range(4)]
    fcv._lib.check(fcv._lib.load().fcv_fp4_attention_plan(fcv._lib.FcvFp4Attention(**base), *got))
    return tuple(v.value for v in got)


@pytest.mark.parametrize("path", CASES, ids=str)
def test_paths(fcv, path):
    rows, _, ranges, ordered = plan(fcv, *CASES[path])
    assert (rows, ranges > 1, ordered == 1) == path[:3]


def test_every_path_is_reached(fcv):
    paths = {(r, c, o) for r in (8, 16, 128) for c in (False, True) for o in (False, True)}
    assert {p[:3] for p in CASES} == paths
    turns = set()
    for path, case in CASES.items():
        rows, tiles, _, _ = plan(fcv, *case)
        if max(case[0]) * (case[2] // case[3]) > rows * tiles:
            turns.add(rows)
    assert turns == {8, 16, 128}


def test_pages_far_apart_take_large_tiles(fcv):
    for d in (64, 128):
        assert plan(fcv, [300] * 33, [384] * 33, 8, 2, d, 300, 384)[0] == 128


def test_refusals(fcv):
    for bad in (dict(head_dim=96), dict(tokens=0), dict(scale=0.0)):
        with pytest.raises(ValueError):
            plan(fcv, *CASES[(8, False, False)], **bad)
    fn = fcv._lib.load().fcv_fp4_attention_plan
    assert fn(None, *[ctypes.c_int32() for _ in range(4)]) != 0
