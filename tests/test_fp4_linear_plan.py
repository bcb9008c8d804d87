"""Which kernel a 4-bit product takes: the sizes of the GPU tests reach every one, whole and with K cut."""

from __future__ import annotations

import ctypes

from tests.test_gpu_fp4_linear import SIZES, TILES

BIG = 1 << 40


def plan(fcv, m, k, n, **kw):
    groups = (k + 31) // 32
    base = dict(x=BIG, codes=BIG, scales=BIG, y=BIG, ldx=k, ld_codes=16 * groups, ld_scales=groups, ldy=n, ldr=n,
                m=m, n=n, k=k, dtype=1, bias_dtype=1, residual_dtype=1, y_dtype=1, activation=0)
    base.update(kw)
    form, ranges = ctypes.c_int32(), ctypes.c_int32()
    fcv._lib.check(fcv._lib.load().fcv_fp4_linear_plan(fcv._lib.FcvFp4Linear(**base), form, ranges))
    return form.value, ranges.value


def test_every_kernel_is_reached(fcv):
    seen = {plan(fcv, *size) for size in SIZES + TILES}
    assert {form for form, ranges in seen if ranges > 1} == set(range(7)), seen
    assert {form for form, ranges in seen if ranges == 1} == set(range(7)), seen


def test_few_rows_keep_to_one_launch_where_weights_are_many(fcv):
    assert plan(fcv, 1, 4096, 4096) == (0, 1) and plan(fcv, 32, 4096, 16384) == (0, 1)
    form, ranges = plan(fcv, 16, 16384, 256)
    assert form == 0 and ranges > 1


def test_workspaces(fcv):
    """Sums of the ranges, and rows of x off their boundaries, which are laid out first; scales lie anywhere."""
    lib = fcv._lib.load()

    def need(m, k, n, **kw):
        groups = (k + 31) // 32
        base = dict(x=BIG, codes=BIG, scales=BIG, y=BIG, ldx=k, ld_codes=16 * groups, ld_scales=groups, ldy=n,
                    ldr=n, m=m, n=n, k=k, dtype=1, bias_dtype=1, residual_dtype=1, y_dtype=1, activation=0)
        base.update(kw)
        return lib.fcv_fp4_linear_workspace_bytes(fcv._lib.FcvFp4Linear(**base))

    def up(n):
        return (n + 255) // 256 * 256

    assert need(1, 4096, 4096) == 0 and need(4096, 4096, 4096) == 0 and need(0, 4096, 4096) == 0
    assert need(4096, 4096, 4096, x=BIG + 2) == up(4096 * 4096 * 2)
    assert need(4096, 4100, 4096) == up(4096 * 4104 * 2)
    assert need(4096, 4128, 4096) == 0 and need(4096, 4096, 4096, scales=BIG + 1) == 0
    form, ranges = plan(fcv, 64, 4096, 4096)
    assert ranges > 1 and need(64, 4096, 4096) == up(ranges * 64 * 4096 * 4)
