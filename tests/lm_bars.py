"""Tolerances of the language model operators' tests, counted in roundings (never fitted to a run).

U = 2^-24 is half a step of fp32.  A sum of n products in any order is off by at most n U sum|x y|
(products of 16-bit numbers are exact in fp32).  A result rounded to a type T is off by half a step
of T, eps(T) / 2 relative, or by half of T's smallest number.  Hardware exp2, reciprocal, square
root and division are within 2 U each.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24
# half of the smallest positive number; fp32 results below 2^-126 may flush to 0
FLOOR = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}


def rounding(y, dtype):
    return (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2) * y.abs() + FLOOR[dtype]


def linear(y, z, mass, residual, k, activation, dtype):
    """z = K products and the bias: (K + 1) U mass.  Every activation's slope is below 1.2.
    Its own error: relu none; the others end in z times a factor whose exponential has an argument
    of size g (silu: 1.5 |z|; gelu_tanh: |z| (2.31 + 0.104 z^2)) with 4 U relative, so at most
    (4 g + 10) U |act|; gelu: 0.5 z (1 + erf), erf within 8 U, so 8 U |z|.  The sum with the
    residual adds U |y|."""
    act = y if residual is None else y - residual.double().cpu()
    err = 1.2 * (k + 2) * U * mass + 2 * U * y.abs()
    if activation == "silu":
        err = err + (6 * z.abs() + 10) * U * act.abs()
    elif activation == "gelu_tanh":
        err = err + (4 * z.abs() * (2.31 + 0.104 * z * z) + 10) * U * act.abs()
    elif activation == "gelu":
        err = err + 8 * U * z.abs()
    return (err + rounding(y.abs() + err, dtype)) * (1 + 2 ** -10)


def norm_rope(y, size, dim, normed, dtype):
    """The mean of dim squares is off by (dim + 2) U relative, its root by half of that, the root,
    division and two products by 2 U each; the rotation's two products and sum by 3 U size."""
    err = ((dim / 2 + 12 if normed else 0) + 4) * U * size
    return (err + rounding(y.abs() + err, dtype)) * (1 + 2 ** -10)


def attention(out, mass, score, keys, dim, dtype, v_max, parts=1):
    """Scores are off by (dim + 4) U score; twice that relative in a weight (numerator and
    denominator).  A weight is rounded to T: eps(T) / 2 relative, and with `parts` 2 its rest
    is rounded again.  fp16 weights are held at 2^11 times their size, so one below fp16's normal
    numbers (2^-14) is below 2^-25 of the row's largest and off by at most that, read as zero or not.  Sums of `keys` weights and of the parts:
    (keys + 64) U."""
    score, keys = score[..., None], keys[..., None]
    eps = (torch.finfo(dtype).eps / 2) ** parts
    rel = eps + 2 * ((dim + 4) * score + 8 + keys + 64) * U
    err = rel * mass
    if dtype == torch.float16:
        err = err + keys * 2.0 ** -25 * v_max
    return (err + rounding(out.abs() + err, dtype)) * (1 + 2 ** -8)


def lse(score, keys, dim, value):
    """d(lse) is at most the largest score's error plus the relative error of the sum and of the
    logarithm, (keys + 64 + 8) U, and the final products' 4 U |lse|."""
    return ((dim + 4) * score + keys + 72 + 4 * value.abs().nan_to_num(0, 0, 0)) * U * (1 + 2 ** -8)


def assert_within(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() / tol)
    off = torch.where(off.isnan(), torch.full_like(off, float("inf")), off)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance at {int(off.argmax())}"
