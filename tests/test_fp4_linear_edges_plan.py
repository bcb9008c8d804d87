"""The GPU tests' sizes reach every kernel of the 4-bit layer, whole and with K cut, where a row's groups are no
multiple of four, and its large tiles with rows far apart."""

from __future__ import annotations

from tests.test_fp4_linear_plan import plan
from tests.test_gpu_fp4_linear_edges import FAR, SPANS


def test_rows_that_end_inside_a_span(fcv):
    forms = set()
    for m, k, n in SPANS:
        groups = k // 32
        assert k % 32 == 0 and groups % 4
        for dtype in (0, 1):
            form, ranges = plan(fcv, m, k, n, dtype=dtype, bias_dtype=dtype, residual_dtype=dtype, y_dtype=dtype)
            forms.add((dtype, form, ranges > 1))
    assert forms >= {(d, f, False) for d in (0, 1) for f in range(1, 7)}, forms
    assert forms >= {(d, f, True) for d in (0, 1) for f in range(2, 7)}, forms


def test_rows_far_apart_take_tiles_of_256_columns(fcv):
    assert [plan(fcv, m, k, n)[0] for _, m, k, n in FAR] == [form for form, *_ in FAR] == [4, 5, 6]
    assert all(n > 256 for _, _, _, n in FAR)
