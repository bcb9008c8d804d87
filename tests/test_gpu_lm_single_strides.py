"""A dimension of one entry may have any stride: a row out of a wider buffer, one key head, one session."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_lm_attention as attn
from tests import test_gpu_lm_rope as rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def odd(t, dims):
    """``t`` with odd strides in the given dimensions, which have one entry each."""
    assert all(t.shape[d] == 1 for d in dims)
    return t.as_strided(t.shape, [3 if d in dims else s for d, s in enumerate(t.stride())])


@pytest.mark.parametrize("dim", [64, 128])
def test_rope(fcv, dim):
    qkv, pos, cos, sin, k, v, rows, qw, kw = rope.make(fcv, 1, 2, 1, dim, dim, torch.bfloat16,
                                                       sessions=1)
    buf = torch.zeros(3, qkv.shape[1] + 5, dtype=qkv.dtype, device=DEV)
    buf[0, :qkv.shape[1]] = qkv[0]
    rope.check(fcv, buf[:1, :qkv.shape[1]], pos, cos, sin, odd(k, (0, 2)), odd(v, (0, 2)), rows, 2, qw,
               kw, False, "one of each")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [1, 40])
def test_attention(fcv, prefix, dim):
    a = attn.make([1], [9], prefix, 2, 1, dim, torch.bfloat16, sessions=1)
    a["q"] = odd(a["q"], (0,))
    a["k_cache"], a["v_cache"] = odd(a["k_cache"], (0, 2)), odd(a["v_cache"], (0, 2))
    one = (0, 1) if prefix == 1 else (1,)
    a["prefix_k"], a["prefix_v"] = odd(a["prefix_k"], one), odd(a["prefix_v"], one)
    out = odd(torch.empty(1, 2, dim, dtype=torch.bfloat16, device=DEV), (0,))
    attn.check(fcv, a, "one of each", out=out)
    a = attn.make([1] * 3, [1] * 3, prefix, 1, 1, dim, torch.float16, capacity=1)
    a["q"] = odd(a["q"], (1,))
    a["k_cache"], a["v_cache"] = odd(a["k_cache"], (1, 2)), odd(a["v_cache"], (1, 2))
    attn.check(fcv, a, "one head, one key")
