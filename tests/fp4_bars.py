"""Tolerances and inputs of the 4-bit operators' tests; roundings are counted as in ``lm_bars``."""

from __future__ import annotations

import torch

from oracle import fp4_oracle as F
from tests import lm_bars as bars
from tests.lm_bars import U

DEV = "cuda:0"


def attention(out, mass, score, keys, dim, dtype):
    """Scores are off by (dim + 4) U score, twice that relative in a weight (numerator and denominator).
    A weight goes in as two bf16 numbers: its rounding is off by 2^-8 of it at most, and that rest's by 2^-8
    of the rest.  Sums of `keys` weights and of the parts, exponentials and the factors between parts:
    (keys + 72) U.  The values' scales are powers of two."""
    score, keys = score[..., None], keys[..., None]
    err = (2.0 ** -16 + 2 * ((dim + 4) * score + 8 + keys + 72) * U) * mass
    return (err + bars.rounding(out.abs() + err, dtype)) * (1 + 2 ** -8)


def attention_one(out, mass, score, keys, dim, v_max, reach):
    """bf16 by tiles of 128 rows: a weight times its value's scale goes in as one fp16 number, off by 2^-11 of
    it at most.  They are held at 2^14 over a scale 2^u, so one that fp16's normal numbers do not reach is off
    by 2^-25 / 2^14 = 2^-39 of 2^u, times a number of 6 at most.  2^u is at most the largest scale of the keys
    and, with `reach` the largest product of a weight and a value among those that the row sees, 2^17 of the
    largest weight times scale; a scale's group holds a value of 3.5 of it.  So for each key
    it is 2^-39 6 / 3.5 < 2^-38 of the largest value, and 2^-21 of `reach`."""
    score, keys = score[..., None], keys[..., None]
    least = torch.minimum(2.0 ** -38 * v_max, 2.0 ** -21 * reach[..., None])
    err = (2.0 ** -11 + 2 * ((dim + 4) * score + 8 + keys + 72) * U) * mass + keys * least
    return (err + bars.rounding(out.abs() + err, torch.bfloat16)) * (1 + 2 ** -8)


def random_pages(n, heads, d, seed=0, dtype=torch.bfloat16, scale=1.0):
    """A pool whose bytes are those of normal keys and values, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n, heads, F.PAGE, d, generator=g) * scale
    v = torch.randn(n, heads, F.PAGE, d, generator=g) * scale
    return pack(k, v, dtype)


def pack(k, v, dtype):
    """Bytes of pages [n, heads, 64, D] of keys and values."""
    kc, ks = F.quantize(k.unflatten(-1, (-1, F.GROUP)), dtype)
    vc, vs = F.quantize(v, dtype)
    kc = kc.flatten(-2)
    kb = kc[..., 0::2] | kc[..., 1::2] << 4
    vb = (vc[..., 0::2] | vc[..., 1::2] << 4).transpose(-1, -2)
    return torch.cat((kb.flatten(-2), vb.flatten(-2), ks.flatten(-2), vs), -1)
