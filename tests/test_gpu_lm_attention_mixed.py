"""``prefix_attention`` of batches whose sequences append very different numbers of tokens."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_helpers import say
from tests.test_gpu_lm_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("prefix", [3, 65, 1100])
def test_a_text_among_tokens(fcv, prefix, hq, hk, dim, dtype):
    say(f"[attn] mixed, behind {prefix}, {hq}/{hk} x {dim} {dtype}")
    news = [1] * 5 + [150] + [1] * 6 + [0, 33, 2]
    lengths = [1 + 17 * i for i in range(12)] + [9, 33, 90]
    lengths[5] = 170
    a = make(news, lengths, prefix, hq, hk, dim, dtype)
    check(fcv, a, "mixed", parts=2, max_q=150, max_length=187)
    check(fcv, a, "default bounds", parts=2)


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_with_cu_q_alone_are_a_decode_step(fcv, dim):
    """Without a bound on the new tokens, as many rows as sequences are taken as one each: the same
    launch as with the bound, and the same bits."""
    a = make([1] * 12, [1 + 30 * i for i in range(12)], 700, 8, 2, dim, torch.bfloat16)
    want = fcv.prefix_attention(**a, max_q=1)
    assert torch.equal(fcv.prefix_attention(**a), want)
    check(fcv, a, "decode", parts=2)
