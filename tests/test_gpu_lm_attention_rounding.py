"""``prefix_attention``'s error is that of rounding the result: its softmax weights lose nothing that counts,
whichever tiles a call takes and whatever else is in its batch."""

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
@pytest.mark.parametrize("news,lengths,prefix", [
    ([1] * 4, [100, 1, 333, 40], 0), ([1] * 4, [100, 1, 333, 40], 2304),   # tokens
    ([40, 9, 33], [45, 200, 33], 300),                                     # a few tokens each
    ([200, 130], [300, 130], 0), ([200, 130], [300, 130], 500),            # texts
])
def test_the_results_rounding_alone(fcv, news, lengths, prefix, hq, hk, dim, dtype):
    for sharp in (0.5, 2.0, 8.0):
        say(f"[attn] rounding, {news} behind {prefix}, {hq}/{hk} x {dim} {dtype}, sharp {sharp}")
        a = make(news, lengths, prefix, hq, hk, dim, dtype, sharp=sharp)
        check(fcv, a, "rounding", parts=2, max_q=max(news), max_length=max(lengths))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,hq,hk,dim", [(66, 64, 8, 128), (129, 128, 8, 128), (65, 512, 16, 64)])
def test_a_large_batch_keeps_a_tokens_precision(fcv, batch, hq, hk, dim, dtype):
    """Stacked rows on both sides of 2^21 elements, where the prompt's tiles change."""
    say(f"[attn] rounding, {batch} tokens x {hq} heads x {dim} {dtype}")
    lengths = [1 + 13 * i % 70 for i in range(batch)]
    a = make([1] * batch, lengths, 900, hq, hk, dim, dtype)
    check(fcv, a, "stacked", parts=2, max_q=1, max_length=max(lengths))
