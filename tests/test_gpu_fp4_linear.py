"""``quantize_fp4`` and ``fused_linear_fp4`` against their formulas in 64 bits, at the sizes, strides and types
where they can go wrong; refusals that need GPU tensors."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4_oracle as F
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
    """x, codes, scales, bias and residual; scales vary from group to group, what lies past K in a row's
    last group is random."""
    g = torch.Generator().manual_seed(seed + 7919 * m + 31 * k + n)
    groups = (k + 31) // 32
    x = torch.randn(m, k, generator=g).to(dtype)
    codes = torch.randint(0, 256, (n, 16 * groups), generator=g, dtype=torch.uint8)
    e = torch.randint(-3, 2, (n, groups), generator=g) - round(math.log2(4 * k ** 0.5))
    b = None if bias is None else torch.randn(n, generator=g).to(bias)
    r = None if residual is None else torch.randn(m, n, generator=g).to(residual)
    return [None if t is None else t.to(DEV) for t in (x, codes, (e + 127).to(torch.uint8), b, r)]


def check(got, x, codes, scales, b, act, r, dtype, what):
    w = F.weights(codes, scales, x.shape[-1], x.dtype)
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
    say(f"[linear fp4] {m} x {k} x {n} {dtype}")
    x, c, s, b, r = make(m, k, n, dtype, bias=dtype, residual=dtype)
    check(fcv.fused_linear_fp4(x, c, s), x, c, s, None, None, None, dtype, "plain")
    check(fcv.fused_linear_fp4(x, c, s, b, activation="silu", residual=r), x, c, s, b, "silu", r,
          dtype, "bias, silu, residual")


# tiles of every shape, K ending inside a slice, rows and columns inside a tile
TILES = [(77, 904, 601), (600, 1000, 4096), (2000, 4104, 2000), (19000, 200, 381), (2048, 1032, 4096),
         (4600, 1000, 2000), (4096, 1000, 4090), (4090, 1000, 4100), (8, 4104, 130), (300, 4104, 70),
         (709, 4101, 67), (2717, 3277, 787), (2740, 7883, 149), (2708, 3426, 1455), (3069, 4194, 1301)]


@pytest.mark.parametrize("m,k,n", TILES)
def test_large(fcv, m, k, n):
    say(f"[linear fp4] tiles {m} x {k} x {n}")
    dtype = torch.bfloat16
    x, c, s, b, r = make(m, k, n, dtype, bias=torch.float32, residual=dtype)
    check(fcv.fused_linear_fp4(x, c, s, b, activation="gelu", residual=r), x, c, s, b, "gelu", r,
          dtype, "tiles")


@pytest.mark.parametrize("act", [None, "none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(1, 512, 64), (40, 256, 72), (300, 128, 260)])
def test_activations_and_fp32_sides(fcv, m, k, n, act):
    say(f"[linear fp4] {act} {m} x {k} x {n}")
    for dtype in (torch.bfloat16, torch.float16):
        for side in (dtype, torch.float32):
            x, c, s, b, r = make(m, k, n, dtype, seed=3, bias=side, residual=side)
            s += 2  # arguments in both tails
            for out in (dtype, torch.float32):
                got = fcv.fused_linear_fp4(x, c, s, b, activation=act, residual=r, out_dtype=out)
                check(got, x, c, s, b, act, r, out, f"{side} {out}")


@pytest.mark.parametrize("k", [1, 3, 7, 9, 31, 33, 63, 65, 129, 1001])
@pytest.mark.parametrize("m,n", [(1, 70), (20, 33), (150, 140)])
def test_widths_that_end_inside_a_group(fcv, m, k, n):
    say(f"[linear fp4] odd K {m} x {k} x {n}")
    x, c, s, b, _ = make(m, k, n, torch.float16, bias=torch.float16)
    check(fcv.fused_linear_fp4(x, c, s, b), x, c, s, b, None, None, torch.float16, "packed rows")
    # rows of a wider buffer whose tail holds NaN
    pad = (k + 7) // 8 * 8 + 8
    xw = torch.full((m, pad), float("nan"), dtype=x.dtype, device=DEV)
    xw[:, :k] = x
    check(fcv.fused_linear_fp4(xw[:, :k], c, s, b), x, c, s, b, None, None, torch.float16, "wide rows")


@pytest.mark.parametrize("m,k,n", [(1, 160, 40), (13, 104, 70), (70, 256, 90), (300, 520, 130)])
def test_strides_and_starts(fcv, m, k, n):
    """Rows of x, codes, scales and y inside wider buffers, and x off 16-byte boundaries."""
    say(f"[linear fp4] strides {m} x {k} x {n}")
    dtype = torch.bfloat16
    x, c, s, b, r = make(m, k, n, dtype, bias=dtype, residual=dtype)
    wide = [torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=DEV)
            for t, pad in ((x, 11), (c, 48), (s, 3), (r, 5))]
    starts = (3, 16, 1, 1)
    views = []
    for t, buf, at in zip((x, c, s, r), wide, starts):
        views.append(buf[:, at:at + t.shape[1]])
        views[-1].copy_(t)
    out = torch.full((m, n + 9), 7.0, dtype=dtype, device=DEV)
    got = fcv.fused_linear_fp4(views[0], views[1], views[2], b, residual=views[3], out=out[:, 2:2 + n])
    check(got, x, c, s, b, None, r, dtype, "views")
    assert bool((out[:, :2] == 7).all()) and bool((out[:, 2 + n:] == 7).all())
    got = fcv.fused_linear_fp4(x, c, s, b, residual=r, out=r)  # in place over the residual
    assert got.data_ptr() == r.data_ptr()
    one = fcv.fused_linear_fp4(x[:1].expand(m, k), c, s)  # one row told m times
    assert bool((one == one[:1]).all())


def test_leading_dimensions_and_no_rows(fcv):
    x, c, s, b, _ = make(12, 96, 40, torch.float16, bias=torch.float16)
    y = fcv.fused_linear_fp4(x.view(3, 4, 96), c, s, b)
    assert y.shape == (3, 4, 40)
    assert torch.equal(y.view(12, 40), fcv.fused_linear_fp4(x, c, s, b))
    assert fcv.fused_linear_fp4(x[:0], c, s).shape == (0, 40)
    assert fcv.fused_linear_fp4(x[0], c, s).shape == (40,)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_values_that_are_not_finite(fcv, m):
    """A group whose scale is NaN makes its output column NaN, an infinity in x its row (0 times it), and
    nothing else."""
    say(f"[linear fp4] not finite, {m} rows")
    x, c, s, _, _ = make(m, 320, 100, torch.bfloat16)
    clean = fcv.fused_linear_fp4(x, c, s)
    s2, x2 = s.clone(), x.clone()
    s2[37, 4] = 255
    x2[m - 1, 99] = math.inf
    got = fcv.fused_linear_fp4(x, c, s2)
    assert bool(got[:, 37].isnan().all())
    keep = [j for j in range(100) if j != 37]
    assert torch.equal(got[:, keep], clean[:, keep])
    got = fcv.fused_linear_fp4(x2, c, s)
    assert not bool(got[m - 1].isfinite().any())
    assert torch.equal(got[:m - 1], clean[:m - 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_at_the_ends(fcv, dtype):
    """Weights of the largest and smallest exponents are the type's numbers."""
    lo, hi = F.LIMITS[dtype]
    codes = torch.arange(16, dtype=torch.uint8).repeat(4, 1)  # codes 0 .. 15 in the low half, 0 in the high
    codes = codes.to(DEV)
    scales = torch.tensor([[lo], [-10], [5], [hi]], dtype=torch.int64).add(127).to(torch.uint8).to(DEV)
    x = torch.zeros(16, 32, dtype=dtype, device=DEV)
    x[torch.arange(16), 2 * torch.arange(16)] = 1
    got = fcv.fused_linear_fp4(x, codes, scales, out_dtype=torch.float32)
    want = F.weights(codes, scales, 32, torch.float64)[:, 0::2].t()
    # products of fp32's smallest normal numbers may flush
    small = want.abs() < 2.0 ** -126
    assert bool((got.double().cpu() == want)[~small].all())


def test_quantize(fcv):
    """Codes and scales equal the definition's: ties, borders, limits, zeros, infinities, every type."""
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        lo, hi = F.LIMITS[dtype]
        rows = [torch.randn(40, 200, generator=g) * 2.0 ** e for e in (-6, 0, 3)]
        grid = torch.arange(0, 200) / 32.0 - 3.0
        rows.append(torch.stack([grid * 2.0 ** e for e in (-4, 0, 5)]))
        edge = torch.zeros(9, 200)
        edge[0, :5] = torch.tensor([7.0, 6.99, 5.0, 2.5, -0.25])
        edge[1, :5] = torch.tensor([6.96875, 5.0, 3.5, 1.25, -0.75])
        edge[2, 3], edge[3, 70], edge[4, 199] = math.inf, math.nan, -math.inf
        edge[5, :3] = torch.tensor([7.9 * 2.0 ** hi, 6.5 * 2.0 ** hi, -3 * 2.0 ** hi]).clamp(
            -torch.finfo(dtype).max, torch.finfo(dtype).max)
        edge[6, :4] = torch.tensor([1.0, 0.5, 0.75, -0.25]) * 2.0 ** lo
        edge[7, 40:44] = torch.tensor([1e-3, -1e-3, 1e-6, 0.0])
        w = torch.cat(rows + [edge]).to(dtype)
        codes, scales = fcv.quantize_fp4(w.to(DEV))
        padded = torch.zeros(w.shape[0], 224, dtype=dtype)
        padded[:, :200] = w
        c, s = F.quantize(padded.view(-1, 7, 32), dtype)
        assert torch.equal(scales.cpu(), s)
        values = F.numbers(F.unpack(codes)) * F.scales(s).repeat_interleave(32, 1)
        want = (F.numbers(c) * F.scales(s)[..., None]).flatten(1)
        assert bool(((values == want) | (values.isnan() & want.isnan())).all()), dtype
    view = torch.randn(9, 70, generator=g, device="cpu").to(DEV)[:, 3:68]
    a, b = fcv.quantize_fp4(view), fcv.quantize_fp4(view.contiguous())
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert fcv.quantize_fp4(view[:0])[0].shape == (0, 48)


def test_quantized_weights_through_the_layer(fcv):
    g = torch.Generator().manual_seed(8)
    w = (torch.randn(96, 200, generator=g) * 0.07).to(torch.float16).to(DEV)
    x = torch.randn(5, 200, generator=g).to(torch.float16).to(DEV)
    codes, scales = fcv.quantize_fp4(w)
    check(fcv.fused_linear_fp4(x, codes, scales), x, codes, scales, None, None, None, torch.float16,
          "quantized")
    ref = x.double() @ w.double().t()
    off = (fcv.fused_linear_fp4(x, codes, scales).double() - ref).norm() / ref.norm()
    # a value is off by a quarter of itself at most, or by a quarter of its scale: 3.5 of it are in a group
    assert float(off) < 0.25


def test_runs_are_alike_and_captured(fcv):
    """Results do not change from run to run; a captured call replays with new inputs."""
    for m, k, n in ((1, 2048, 512), (24, 4096, 300), (130, 1024, 256)):
        x, c, s, b, r = make(m, k, n, torch.bfloat16, bias=torch.bfloat16, residual=torch.bfloat16)
        want = fcv.fused_linear_fp4(x, c, s, b, activation="silu", residual=r)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fcv.fused_linear_fp4(x, c, s, b, activation="silu", residual=r)
        for seed in range(3):
            x.copy_(make(m, k, n, torch.bfloat16, seed=seed)[0])
            graph.replay()
            want = fcv.fused_linear_fp4(x, c, s, b, activation="silu", residual=r)
            assert torch.equal(got, want), (m, seed)


def test_two_streams(fcv):
    x, c, s, b, _ = make(48, 4096, 512, torch.bfloat16, bias=torch.bfloat16)
    want = fcv.fused_linear_fp4(x, c, s, b)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(fcv.fused_linear_fp4(x, c, s, b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(fcv):
    x, c, s, b, r = make(4, 96, 40, torch.float16, bias=torch.float16, residual=torch.float16)
    f = fcv.fused_linear_fp4
    for bad, match in [
        (lambda: f(x.float(), c, s), "float16 or bfloat16"), (lambda: f(x, c[:, :32], s), "codes"),
        (lambda: f(x, c, s[:, :2]), "scales"), (lambda: f(x, c.int(), s), "codes"),
        (lambda: f(x, c, s[:39]), "scales"), (lambda: f(x, c, s, activation="tanh"), "unknown"),
        (lambda: f(x, c, s, b[:39]), "bias"), (lambda: f(x, c, s, residual=r[:3]), "residual"),
        (lambda: f(x, c, s, out_dtype=torch.bfloat16), "out must be"), (lambda: f(x, c.t(), s), "codes"),
        (lambda: f(x, c, s, out=x[:, :40]), "out overlaps x"),
        (lambda: f(x, torch.zeros(40, 64, dtype=torch.uint8, device=DEV)[:, 8:56], s), "16-byte"),
        (lambda: f(x, c, s, out=torch.empty(4, 41, dtype=x.dtype, device=DEV)), "shape"),
        (lambda: f(x.t(), c, s), "matrix|columns|contiguous"), (lambda: f(x, c.cpu(), s), "codes"),
        (lambda: fcv.quantize_fp4(x.double()), "float32"), (lambda: fcv.quantize_fp4(x[0]), "matrix"),
        (lambda: fcv.quantize_fp4(x.t()), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()
    flat = torch.zeros(4 * 48 + 4 * 40, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="out overlaps codes"):
        f(x, flat[:4 * 48].view(4, 48), s[:4],
          out=flat[16:16 + 32].view(torch.float16).view(4, 4))


@pytest.mark.parametrize("m", [3, 40, 300, 1100])
def test_rows_of_weights_far_apart(fcv, m):
    """The largest row strides: a tile's offsets pass 2^31."""
    n, k = 300, 256
    x, c, s, b, _ = make(m, k, n, torch.bfloat16, bias=torch.bfloat16)
    far = torch.empty(300 * 2 ** 24, dtype=torch.uint8, device=DEV)
    codes = far.as_strided((n, 128), (2 ** 24 - 16, 1))
    codes.copy_(c)
    want = fcv.fused_linear_fp4(x, c, s, b)
    assert torch.equal(fcv.fused_linear_fp4(x, codes, s, b), want)
    scales = far.as_strided((n, 8), (2 ** 24 - 4, 1))
    scales.copy_(s)
    assert torch.equal(fcv.fused_linear_fp4(x, c, scales, b), want)


@pytest.mark.parametrize("m,k,n", [(40, 96, 70), (100, 2112, 200), (300, 416, 300), (700, 160, 600), (2100, 1184, 1030)])
@pytest.mark.parametrize("start", [0, 1, 2, 3])
def test_scales_on_any_byte(fcv, m, k, n, start):
    """Rows of 3, 13, 66, 5 and 37 scales from every byte of a word, at odd strides; NaN around them."""
    x, c, s, b, _ = make(m, k, n, torch.bfloat16)
    want = fcv.fused_linear_fp4(x, c, s)
    check(want, x, c, s, None, None, None, torch.bfloat16, "dense")
    for pad in (0, 5, 7):
        wide = torch.full((n * (s.shape[1] + pad) + 16,), 255, dtype=torch.uint8, device=DEV)
        view = wide[4 + start:4 + start + n * (s.shape[1] + pad)].view(n, -1)[:, :s.shape[1]]
        view.copy_(s)
        assert torch.equal(fcv.fused_linear_fp4(x, c, view), want), pad
