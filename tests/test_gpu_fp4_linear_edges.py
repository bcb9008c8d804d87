"""``fused_linear_fp4`` where a row of weights ends inside a group, in every kernel."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_helpers import say
from tests.test_fp4_linear_plan import plan
from tests.test_gpu_fp4_linear import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype,scale", [(torch.float16, 14), (torch.bfloat16, 126)])
@pytest.mark.parametrize("form,m,k,n", [(0, 1, 100, 70), (0, 20, 1001, 300), (0, 2, 4101, 130), (1, 40, 31, 70),
                                        (1, 40, 1000, 70), (2, 600, 1000, 4096), (3, 2048, 127, 4096),
                                        (4, 4096, 1000, 2048), (5, 6144, 200, 2048), (6, 4096, 1001, 4096)])
def test_codes_past_k(fcv, form, m, k, n, dtype, scale):
    """Codes behind a row's end count for nothing, also where the last group's scale makes an infinity of them
    (6 times 2^14 in fp16, 2^126 in bf16) and numbers of those below K (at most 3/2 times it)."""
    say(f"[linear fp4] codes past K {m} x {k} x {n} {dtype}")
    assert plan(fcv, m, k, n)[0] == form
    g = torch.Generator().manual_seed(k + n)
    groups = (k + 31) // 32
    codes = torch.randint(0, 4, (n, 32 * groups), generator=g) + 8 * torch.randint(0, 2, (n, 32 * groups), generator=g)
    codes[:, k:] = 0
    full = codes.clone()
    full[:, k:] = 7 + 8 * torch.randint(0, 2, (n, 32 * groups - k), generator=g)
    clean, full = ((c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8).to(DEV) for c in (codes, full))
    scales = torch.full((n, groups), 127 - 5, dtype=torch.uint8, device=DEV)
    scales[:, -1] = 127 + scale
    x = (torch.randn(m, k, generator=g) * 2.0 ** -10).to(dtype).to(DEV)
    want = fcv.fused_linear_fp4(x, clean, scales, out_dtype=torch.float32)
    assert torch.equal(fcv.fused_linear_fp4(x, full, scales, out_dtype=torch.float32), want)
    if m <= 40:
        check(want, x, clean, scales, None, None, None, torch.float32, "codes")
