"""``fused_linear`` where K is cut over workgroups: every tile shape with a short last range that ends inside
a slice and rows that leave no aligned stores."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say
from tests.test_gpu_lm_linear import check, make

pytestmark = pytest.mark.gpu

# (m, k, n) for each kernel, the first two through registers
CUTS = [(40, 2001, 70), (33, 3003, 129), (8, 4104, 131), (18, 1048, 17), (17, 8728, 2827),
        (150, 9000, 2050), (1000, 9000, 1000), (6744, 3656, 258), (5677, 5272, 135), (3000, 9000, 700),
        (5408, 5456, 385), (6581, 5080, 591), (4431, 6944, 262)]
# and whole, through registers
ODD = [(40, 201, 70), (200, 77, 130), (17, 63, 65)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("m,k,n", CUTS)
def test_cut_products(fcv, m, k, n):
    say(f"[linear] cut {m} x {k} x {n}")
    dtype = torch.bfloat16 if m % 2 else torch.float16
    x, w, b, r = make(m, k, n, dtype, bias=torch.float32, residual=dtype)
    first = fcv.fused_linear(x, w)
    assert torch.equal(first, fcv.fused_linear(x, w))
    y, z, mass = O.linear(x, w, b, "silu", r)
    tol = bars.linear(y, z, mass, r, k, "silu", dtype)
    assert fcv.fused_linear(x, w, b, activation="silu", residual=r, out=r) is r
    bars.assert_within(r, y, tol, "bias, silu, residual in place")


@pytest.mark.parametrize("m,k,n", ODD)
def test_whole_products_through_registers(fcv, m, k, n):
    x, w, b, r = make(m, k, n, torch.bfloat16, bias=torch.bfloat16, residual=torch.float32)
    check(fcv.fused_linear(x, w, b, activation="relu", residual=r), x, w, b, "relu", r, torch.bfloat16,
          "whole")
