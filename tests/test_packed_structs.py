"""The language model's operators pass their arguments as packed bytes: as many as the C struct has, since the
library copies whole structs."""

from __future__ import annotations

import ctypes

import pytest


@pytest.mark.parametrize("module,layout,name", [
    ("lm", "_LINEAR", "FcvLmLinear"), ("lm", "_QK_NORM_ROPE", "FcvLmQkNormRope"), ("lm", "_ATTENTION", "FcvLmAttention"),
    ("lm_fp4", "_QUANTIZE", "FcvFp4Quantize"), ("lm_fp4", "_LINEAR", "FcvFp4Linear"),
    ("lm_fp4", "_APPEND", "FcvFp4Append"), ("lm_fp4", "_READ", "FcvFp4Read"), ("lm_fp4", "_ATTENTION", "FcvFp4Attention")])
def test_sizes(fcv, module, layout, name):
    packed = getattr(__import__(f"faster_cosyvoice_amd.{module}", fromlist=["x"]), layout)
    assert packed.size == ctypes.sizeof(getattr(fcv._lib, name))
