"""Softmax weights of ``paged_attention_fp4`` by tiles of 128 rows: as exact as the smaller tiles', and values that
a row does not see never touch it, whatever their size."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4_oracle as F
from tests import fp4_bars, lm_bars
from tests.gpu_helpers import say
from tests.test_gpu_fp4_attention import make, run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def compare(out, lse, st, what):
    """Against the formula in 64 bits, a head's rows at once, by the bar that every form of the attention has."""
    q, d, heads = st["q"].double(), st["q"].shape[2], st["q"].shape[1]
    group, scale = heads // st["pages"].shape[1], st["q"].shape[2] ** -0.5
    cu = st["cu_q"].tolist()
    for b, (k, v, at, length) in enumerate(F.cache(st["pages"], d, st["table"], st["lengths"])):
        n, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        hidden = at > (length - n + torch.arange(n))[:, None]
        count = (~hidden).sum(1).double()
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            s = scale * (q[rows, h] @ kh.t())
            size = (scale * (q[rows, h].abs() @ kh.abs().t())).masked_fill(hidden, 0).amax(1)
            s = s.masked_fill(hidden, -math.inf)
            p, wl = torch.softmax(s, 1), torch.logsumexp(s, 1)
            want = p @ vh
            tol = fp4_bars.attention(want, p @ vh.abs(), size, count, d, st["q"].dtype)
            lm_bars.assert_within(out[rows, h], want, tol, f"{what} {b} {h}")
            lm_bars.assert_within(lse[rows, h], wl, lm_bars.lse(size, count, d, wl), f"{what} {b} {h} lse")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_cancel(fcv, d, dtype):
    """Keys' values of 1 and -1 in turn and nearly equal weights: a result far below the weights, whose own
    rounding hides none of theirs."""
    say(f"[attend fp4 weights] cancel {d} {dtype}")
    st = make([200] * 20, [200] * 20, 16, 16, d, dtype, q_scale=0.004)
    n = st["pages"].shape[0]
    k = torch.randn(n, 16, F.PAGE, d, generator=torch.Generator().manual_seed(d))
    v = (1.0 - 2.0 * (torch.arange(F.PAGE) % 2))[:, None].expand(n, 16, F.PAGE, d)
    st["pages"] = fp4_bars.pack(k, v, dtype)
    compare(*run(fcv, st, max_q=200, return_lse=True), st, "cancel")


@pytest.mark.parametrize("d", [64, 128])
def test_hidden_values_of_any_size(fcv, d):
    """Values of 2^-42 that count, and of 2^100 that a row does not see, or sees with a weight that vanishes."""
    say(f"[attend fp4 weights] hidden {d}")
    st = make([200] * 20, [330] * 20, 16, 16, d, torch.bfloat16)
    g = torch.Generator().manual_seed(7)
    n = st["pages"].shape[0]
    k = torch.randn(n, 16, F.PAGE, d, generator=g)
    v = torch.randn(n, 16, F.PAGE, d, generator=g).double() * 2.0 ** -42  # 2^142 passes fp32
    k[..., 0] = 0
    st["q"][..., 0] = d ** 0.5
    for b in range(20):
        for key in ((329,), (325, 329), tuple(range(321, 330)))[b % 3]:
            v[st["table"][b, key // 64], :, key % 64] *= 2.0 ** 142
        if b % 2:  # first keys of vanishing weight: a score 192 below the others'
            for key in (0, 5, 70):
                v[st["table"][b, key // 64], :, key % 64] *= 2.0 ** 142
                k[st["table"][b, key // 64], :, key % 64, 0] = -192.0
    st["pages"] = fp4_bars.pack(k, v, torch.bfloat16)
    out, lse = run(fcv, st, max_q=200, return_lse=True)
    compare(out, lse, st, "hidden")
    assert bool((out.float().abs().amax(-1) > 0).all())
