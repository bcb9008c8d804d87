"""Which kernels ``fused_linear`` takes: every one that the estimate can pick, with K whole and cut, is
among the sizes that the GPU tests compare with the formula."""

from __future__ import annotations

import ctypes

from tests.test_gpu_lm_linear import SIZES, TILES
from tests.test_gpu_lm_linear_cuts import CUTS, ODD

BIG = 1 << 40  # an address nothing dereferences


def _plan(fcv, m, k, n):
    args = fcv._lib.FcvLmLinear(x=BIG, w=BIG, y=BIG, ldx=k, ldw=k, ldy=n, ldr=0, m=m, n=n, k=k,
                                dtype=1, bias_dtype=1, residual_dtype=1, y_dtype=1, activation=0)
    form, ranges = ctypes.c_int32(), ctypes.c_int32()
    fcv._lib.check(fcv._lib.load().fcv_lm_linear_plan(args, form, ranges))
    return form.value, ranges.value > 1


def test_tested_sizes_reach_every_kernel(fcv):
    steps = [round(1.45 ** i) for i in range(27)]   # 1 .. 16000
    widths = [8 * s for s in steps[:20]] + [71, 3001]
    reached = {_plan(fcv, m, k, n) for m in steps for n in steps for k in widths}
    assert {form for form, _ in reached} == set(range(9))
    tested = {_plan(fcv, *size) for size in SIZES + TILES + CUTS + ODD}
    assert reached <= tested, sorted(reached - tested)


def test_cut_sizes_are_cut(fcv):
    assert all(cut for _, cut in (_plan(fcv, *size) for size in CUTS))


def test_what_the_call_refuses_has_no_plan(fcv):
    args = fcv._lib.FcvLmLinear(x=BIG, w=BIG, y=BIG, ldx=8, ldw=8, ldy=8, m=1, n=8, k=0, dtype=1)
    form, ranges = ctypes.c_int32(), ctypes.c_int32()
    assert fcv._lib.load().fcv_lm_linear_plan(args, form, ranges) != 0
