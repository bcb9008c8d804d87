"""``fused_linear_fp4`` in every kernel and both types: rows of weights that end inside a group or a span of four,
scales on any byte, rows far apart."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4_oracle as F
from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say
from tests.test_fp4_linear_plan import plan
from tests.test_gpu_fp4_linear import TILES, check, make

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


@pytest.mark.parametrize("m,k,n", TILES)
def test_large_in_fp16(fcv, m, k, n):
    say(f"[linear fp4] tiles in fp16 {m} x {k} x {n}")
    dtype = torch.float16
    x, c, s, b, r = make(m, k, n, dtype, bias=dtype, residual=torch.float32)
    check(fcv.fused_linear_fp4(x, c, s, b, activation="gelu_tanh", residual=r), x, c, s, b, "gelu_tanh", r, dtype,
          "tiles")


# a last span of one to three groups, whole and with K cut into ranges: every tile
SPANS = [(40, 96, 70), (709, 4192, 67), (2100, 1184, 1030), (2740, 352, 200), (19000, 224, 381), (2717, 3232, 787),
         (2048, 416, 4096), (2740, 7840, 149), (9184, 224, 1024), (2708, 3296, 1455), (4096, 160, 4096),
         (3069, 4192, 1301)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SPANS)
def test_scales_on_any_byte(fcv, m, k, n, dtype):
    """From every byte of a word, at odd strides; NaN around them."""
    say(f"[linear fp4] scales {m} x {k} x {n} {dtype}")
    x, c, s, b, _ = make(m, k, n, dtype, bias=dtype)
    want = fcv.fused_linear_fp4(x, c, s, b)
    check(want, x, c, s, b, None, None, dtype, "dense")
    for start in range(4):
        for pad in (0, 5, 7):
            wide = torch.full((n * (s.shape[1] + pad) + 16,), 255, dtype=torch.uint8, device=DEV)
            view = wide[4 + start:4 + start + n * (s.shape[1] + pad)].view(n, -1)[:, :s.shape[1]]
            view.copy_(s)
            assert torch.equal(fcv.fused_linear_fp4(x, c, view, b), want), (start, pad)


# tiles of 256 columns, whose last row lies 255 strides behind the first
FAR = [(4, 16000, 512, 300), (5, 24000, 512, 257), (6, 30000, 512, 300)]


@pytest.mark.parametrize("form,m,k,n", FAR)
def test_rows_of_weights_far_apart(fcv, form, m, k, n):
    """The largest row strides: a tile's offsets pass 2^31 (255 strides of nearly 2^24 bytes).  In front of the
    rows lie 4 GiB more, where a signed offset would point."""
    say(f"[linear fp4] far rows {m} x {k} x {n}")
    assert plan(fcv, m, k, n) == (form, 1)
    x, c, s, b, _ = make(m, k, n, torch.bfloat16, bias=torch.bfloat16)
    buf = torch.empty(2 ** 32 + n * 2 ** 24, dtype=torch.uint8, device=DEV)
    far = buf[2 ** 32:]
    codes = far.as_strided((n, k // 2), (2 ** 24 - 16, 1), far.storage_offset())
    codes.copy_(c)
    want = fcv.fused_linear_fp4(x, c, s, b)
    assert torch.equal(fcv.fused_linear_fp4(x, codes, s, b), want)
    scales = far.as_strided((n, k // 32), (2 ** 24 - 3, 1), far.storage_offset() + 1)
    scales.copy_(s)
    assert torch.equal(fcv.fused_linear_fp4(x, c, scales, b), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantized_weights(fcv, dtype):
    """``quantize_fp4`` and the layer together: the product with the numbers that the definition makes of the
    weights."""
    g = torch.Generator().manual_seed(8)
    w = (torch.randn(96, 200, generator=g) * 0.07).to(dtype)
    x = torch.randn(5, 200, generator=g).to(dtype)
    got = fcv.fused_linear_fp4(x.to(DEV), *fcv.quantize_fp4(w.to(DEV)))
    numbers = F.quantized(torch.nn.functional.pad(w, (0, 24)), dtype, 32)[:, :200]
    want, z, mass = O.linear(x, numbers.to(dtype), None, None, None)
    bars.assert_within(got, want, bars.linear(want, z, mass, None, 200, None, dtype), "quantized")
