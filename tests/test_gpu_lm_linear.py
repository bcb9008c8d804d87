"""``fused_linear`` against its formula in 64 bits, at the sizes, strides and types where it can go
wrong; refusals that need GPU tensors."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def make(m, k, n, dtype, seed=0, bias=None, residual=None):
    g = torch.Generator().manual_seed(seed + 7919 * m + 31 * k + n)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype)
    b = None if bias is None else torch.randn(n, generator=g).to(bias)
    r = None if residual is None else torch.randn(m, n, generator=g).to(residual)
    return [None if t is None else t.to(DEV) for t in (x, w, b, r)]


def check(got, x, w, b, act, r, dtype, what):
    y, z, mass = O.linear(x, w, b, act, r)
    assert got.dtype == dtype
    bars.assert_within(got, y, bars.linear(y, z, mass, r, w.shape[1], act, dtype), what)


SIZES = [(1, 8, 1), (1, 64, 5), (1, 1024, 2048), (2, 72, 33), (3, 200, 100), (7, 896, 130),
         (16, 1000, 64), (17, 512, 96), (31, 4104, 48), (32, 256, 4096), (33, 2048, 257),
         (48, 640, 1000), (64, 1024, 640), (65, 320, 513), (96, 4096, 128), (127, 136, 300),
         (128, 1024, 512), (200, 96, 700), (256, 512, 256), (257, 1032, 263), (511, 64, 129),
         (600, 2048, 1024), (1000, 448, 1100), (1500, 128, 1537)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(fcv, m, k, n, dtype):
    say(f"[linear] {m} x {k} x {n} {dtype}")
    x, w, b, r = make(m, k, n, dtype, bias=dtype, residual=dtype)
    check(fcv.fused_linear(x, w), x, w, None, None, None, dtype, "plain")
    check(fcv.fused_linear(x, w, b, activation="silu", residual=r), x, w, b, "silu", r, dtype,
          "bias, silu, residual")


# one size for each tile shape and ring that the estimate picks, K ending inside a slice, rows and
# columns inside a tile, with and without four aligned columns a store
TILES = [(77, 904, 601), (600, 1000, 4096), (2000, 4104, 2000), (19000, 200, 381), (2048, 1032, 4096),
         (4600, 1000, 2000), (4096, 1000, 4090), (4090, 1000, 4100), (8, 4104, 130), (300, 4104, 70)]


@pytest.mark.parametrize("m,k,n", TILES)
def test_every_tile_shape(fcv, m, k, n):
    say(f"[linear] tiles {m} x {k} x {n}")
    dtype = torch.bfloat16
    x, w, b, r = make(m, k, n, dtype, bias=torch.float32, residual=dtype)
    check(fcv.fused_linear(x, w, b, activation="gelu", residual=r), x, w, b, "gelu", r, dtype, "tiles")


@pytest.mark.parametrize("act", [None, "none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(1, 512, 64), (40, 256, 72), (300, 128, 260)])
def test_activations_and_fp32_sides(fcv, m, k, n, act):
    say(f"[linear] {act} {m} x {k} x {n}")
    for dtype in (torch.bfloat16, torch.float16):
        for side in (dtype, torch.float32):
            x, w, b, r = make(m, k, n, dtype, seed=3, bias=side, residual=side)
            w = (w.float() * 4).to(dtype)  # arguments from -20 to 20: both tails
            for out in (dtype, torch.float32):
                got = fcv.fused_linear(x, w, b, activation=act, residual=r, out_dtype=out)
                check(got, x, w, b, act, r, out, f"{side} {out}")


@pytest.mark.parametrize("k", [1, 3, 7, 9, 15, 63, 65, 129, 1001])
@pytest.mark.parametrize("m,n", [(1, 70), (20, 33), (150, 140)])
def test_widths_that_are_no_multiple_of_eight(fcv, m, k, n):
    say(f"[linear] odd K {m} x {k} x {n}")
    x, w, b, _ = make(m, k, n, torch.float16, bias=torch.float16)
    check(fcv.fused_linear(x, w, b), x, w, b, None, None, torch.float16, "packed rows")
    # rows of a wider buffer whose tail holds NaN: 16-byte aligned, only the tail is masked
    pad = (k + 7) // 8 * 8 + 8
    xw = torch.full((m, pad), float("nan"), dtype=x.dtype, device=DEV)
    ww = torch.full((n, pad), float("nan"), dtype=x.dtype, device=DEV)
    xw[:, :k], ww[:, :k] = x, w
    check(fcv.fused_linear(xw[:, :k], ww[:, :k], b), x, w, b, None, None, torch.float16, "padded")


@pytest.mark.parametrize("m", [1, 9, 40, 130, 520])
def test_strides_and_outputs_in_place(fcv, m):
    k, n, dtype = 320, 200, torch.bfloat16
    say(f"[linear] strides {m}")
    x, w, b, r = make(m, k, n, dtype, bias=dtype, residual=dtype)
    wide = torch.full((m, k + 24), float("nan"), dtype=dtype, device=DEV)
    for off in (8, 3):  # rows on 16-byte boundaries, and off them
        wide[:, off:off + k] = x
        check(fcv.fused_linear(wide[:, off:off + k], w, b), x, w, b, None, None, dtype, f"x + {off}")
    ww = torch.full((n, k + 1), float("nan"), dtype=dtype, device=DEV)
    ww[:, 1:] = w
    check(fcv.fused_linear(x, ww[:, 1:], b), x, w, b, None, None, dtype, "w off by one")
    # an output inside a wider buffer: only its columns change
    for out_type, off in ((dtype, 8), (dtype, 1), (torch.float32, 4), (torch.float32, 3)):
        buf = torch.full((m, n + 13), 7.0, dtype=out_type, device=DEV)
        got = fcv.fused_linear(x, w, b, activation="relu", residual=r, out=buf[:, off:off + n])
        assert got.data_ptr() == buf[:, off:].data_ptr()
        check(got, x, w, b, "relu", r, out_type, f"out + {off}")
        assert (buf[:, :off] == 7).all() and (buf[:, off + n:] == 7).all()
    # the residual updated in place, in both types
    for t in (dtype, torch.float32):
        h = r.to(t).clone()
        want = O.linear(x, w, b, "gelu_tanh", h)
        before = h.clone()
        assert fcv.fused_linear(x, w, b, activation="gelu_tanh", residual=h, out=h) is h
        check(h, x, w, b, "gelu_tanh", before, t, "in place")
        del want
    # leading dimensions, one broadcast row, no rows
    x3 = x.view(1, m, k)
    assert fcv.fused_linear(x3, w).shape == (1, m, n)
    check(fcv.fused_linear(x[:1].expand(m, k), w), x[:1].expand(m, k), w, None, None, None, dtype,
          "broadcast rows")
    assert fcv.fused_linear(x[:0], w).shape == (0, n)


def test_one_dimensional_input(fcv):
    x, w, b, _ = make(1, 256, 48, torch.float16, bias=torch.float16)
    got = fcv.fused_linear(x[0], w, b)
    assert got.shape == (48,)
    check(got[None], x, w, b, None, None, torch.float16, "vector")


@pytest.mark.parametrize("m", [1, 33, 300])
def test_infinities_and_nan_stay_in_their_rows(fcv, m):
    say(f"[linear] not finite {m}")
    x, w, b, _ = make(m, 136, 72, torch.bfloat16, bias=torch.bfloat16)
    x[0, 5] = float("nan")
    if m > 1:
        x[m - 1, 135] = float("inf")
    got = fcv.fused_linear(x, w, b, activation="relu")
    assert got[0].isnan().all()
    clean = slice(1, m - 1)
    check(got[clean], x[clean], w, b, "relu", None, torch.bfloat16, "rows between")
    if m > 1:
        y = O.linear(x[m - 1:], w, b, "relu")[0]
        assert torch.equal(got[m - 1:].double().cpu().isinf(), y.isinf())


def test_repeats_are_bit_identical(fcv):
    for m, k, n in ((1, 2048, 512), (40, 4096, 256), (700, 512, 384)):
        x, w, b, r = make(m, k, n, torch.bfloat16, bias=torch.bfloat16, residual=torch.bfloat16)
        first = fcv.fused_linear(x, w, b, residual=r)
        for _ in range(3):
            assert torch.equal(first, fcv.fused_linear(x, w, b, residual=r))


def test_refusals(fcv):
    x, w, b, r = make(4, 64, 32, torch.bfloat16, bias=torch.bfloat16, residual=torch.bfloat16)
    for call, match in [
            (lambda: fcv.fused_linear(x, w.half()), "weight must be"),
            (lambda: fcv.fused_linear(x.float(), w.float()), "float16 or bfloat16"),
            (lambda: fcv.fused_linear(x, w.cpu()), "weight must be"),
            (lambda: fcv.fused_linear(x[:, :60], w), "64 columns"),
            (lambda: fcv.fused_linear(x, w, b[:31]), "vector of 32"),
            (lambda: fcv.fused_linear(x, w, b.half()), "bias must be"),
            (lambda: fcv.fused_linear(x, w, b.cpu()), "bias is on"),
            (lambda: fcv.fused_linear(x, w, residual=r[:3]), "residual must have"),
            (lambda: fcv.fused_linear(x, w, residual=r.t().contiguous().t()), "contiguous"),
            (lambda: fcv.fused_linear(x, w, activation="tanh"), "activation"),
            (lambda: fcv.fused_linear(x, w, out=r[:, :31]), "out must have"),
            (lambda: fcv.fused_linear(x, w, out=r[:1].expand(4, 32)), "overlap"),
            (lambda: fcv.fused_linear(x, w, out_dtype=torch.float64), "out must be"),
            (lambda: fcv.fused_linear(x, w, out=r, out_dtype=torch.float32), "out is"),
            (lambda: fcv.fused_linear(x.t().contiguous().t(), w), "contiguous"),
            (lambda: fcv.fused_linear(x[:0], w[:0]), "empty")]:
        with pytest.raises(ValueError, match=match):
            call()
