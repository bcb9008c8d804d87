"""``qk_norm_rope``'s norms over the whole range of the types: heads whose squares pass fp32 or vanish."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say
from tests.test_gpu_lm_rope import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [-120, -62, -40, -30, 40, 50, 62, 64, 100, 125])
def test_norms_of_large_and_small_heads(fcv, power, dim):
    """Token 0 has ordinary heads and must not notice.  Without eps every size has a norm; with it the
    smallest are left small."""
    hq, hk, dtype = 3, 1, torch.bfloat16
    for eps in (0.0, 1e-6):
        say(f"[rope] heads of size 2^{power} x {dim}, eps {eps}")
        qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 4, hq, hk, dim, dim, dtype)
        x = qkv.float().clamp(-3.9, 3.9)
        x[1:] *= 2.0 ** power
        qkv = x.to(dtype)
        got = fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, n_heads=hq, q_weight=qw, k_weight=kw,
                               eps=eps)
        heads = qkv.view(4, hq + 2 * hk, dim)
        at = pos.cpu().long()
        y, size = O.norm_rope(heads[:, :hq], qw, eps, cos.cpu()[at], sin.cpu()[at], False)
        bars.assert_within(got, y, bars.norm_rope(y, size, dim, True, dtype), "q")
        y, size = O.norm_rope(heads[:, hq:hq + hk], kw, eps, cos.cpu()[at], sin.cpu()[at], False)
        kc = k.view(-1, hk, dim)[rows.long()]
        bars.assert_within(kc, y, bars.norm_rope(y, size, dim, True, dtype), "k")
