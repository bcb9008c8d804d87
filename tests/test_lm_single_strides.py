"""Strides of dimensions of one entry are not looked at by the C ABI's checks."""

from __future__ import annotations

import pytest

from tests.test_lm_host import _attention, _refuse, _rope


def test_attention(fcv):
    odd = dict(tokens=0, sessions=1, slots=1 << 40, capacity=1, n_kv_heads=1, n_heads=1, prefix_len=1,
               q_row=3, q_head=3, out_row=3, out_head=3, pk_row=3, pk_head=3, pv_row=1 << 30, pv_head=3,
               k_session=3, k_row=1 << 30, k_head=3, v_session=3, v_row=3, v_head=3)
    assert _attention(fcv, **odd) == 0
    for name, count in (("k_row", "capacity"), ("pv_row", "prefix_len"), ("v_session", "sessions"),
                        ("q_head", "n_heads")):
        bad = dict(odd, **{count: 2})
        bad.update(k_row=8, pv_row=8)
        bad[name] = 12
        if count in ("n_heads",):
            bad["out_head"] = 64
        _refuse(fcv, _attention(fcv, **bad), "multiples of 8")


@pytest.mark.parametrize("bad", [dict(k_row=12), dict(v_head=12), dict(qkv_row=4)])
def test_rope_still_refuses(fcv, bad):
    _refuse(fcv, _rope(fcv, **bad), "multiples of 8")
