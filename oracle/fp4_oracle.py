"""64-bit CPU restatement of the 4-bit operators (include/fcv_fp4.h).

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  Codes, scales and pages are taken apart bit by bit
here; products and attention are those of ``lm_oracle`` on the numbers that come out.
"""

from __future__ import annotations

import math

import torch

from oracle import lm_oracle as O

Tensor = torch.Tensor
NUMBERS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
PAGE, GROUP = 64, 32
LIMITS = {torch.float16: (-23, 13), torch.bfloat16: (-125, 125), torch.float32: (-125, 125)}


def numbers(codes: Tensor) -> Tensor:
    """Codes 0 .. 15 -> their numbers."""
    table = torch.tensor(NUMBERS + tuple(-v for v in NUMBERS), dtype=torch.float64)
    return table[codes.long().cpu()]


def scales(b: Tensor) -> Tensor:
    b = b.cpu()
    s = torch.ldexp(torch.ones(b.shape, dtype=torch.float64), b.double() - 127)
    return torch.where(b == 255, torch.full_like(s, math.nan), s)


def unpack(codes: Tensor) -> Tensor:
    """Bytes [..., n] -> codes [..., 2 n]."""
    codes = codes.cpu()
    return torch.stack((codes % 16, codes // 16), -1).flatten(-2)


def weights(codes: Tensor, scale_bytes: Tensor, k: int, dtype) -> Tensor:
    """The weights [N, K] that codes and scales stand for, in the type of the call."""
    w = numbers(unpack(codes)) * scales(scale_bytes).repeat_interleave(GROUP, 1)
    return w[:, :k].to(dtype)


def quantize(x: Tensor, dtype) -> tuple[Tensor, Tensor]:
    """Groups along the last dimension -> (codes 0 .. 15, scale bytes), by the definition: the smallest
    exponent with every magnitude below 7 2^e, the nearest number, ties to the even code."""
    x = x.double().cpu()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    lo, hi = LIMITS[dtype]
    e = torch.full(amax.shape, lo, dtype=torch.int64)
    for i in range(lo, hi):
        e = torch.where(amax >= 7.0 * 2.0 ** i, torch.full_like(e, i + 1), e)
    y = (x.abs() / torch.ldexp(torch.ones_like(amax), e.double())[..., None]).nan_to_num(0, 0, 0)
    table = torch.tensor(NUMBERS, dtype=torch.float64)
    off = (y[..., None].clamp_max(6) - table).abs()
    odd = torch.tensor([i % 2 for i in range(8)])
    code = torch.where(off == off.amin(-1, keepdim=True), odd, 2).argmin(-1)  # a tie: the even code
    code = code + 8 * (x < 0)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.to(torch.uint8), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def quantized(x: Tensor, dtype, group: int | None = None) -> Tensor:
    """The numbers that groups along the last dimension become (all of it without ``group``)."""
    shape = x.shape
    if group:
        x = x.unflatten(-1, (-1, group))
    c, s = quantize(x, dtype)
    return (numbers(c) * scales(s)[..., None]).reshape(shape)


def split(pages: Tensor, d: int):
    """(keys [.., 64, D], values [.., 64, D]) of pages' bytes [.., page bytes], in 64 bits."""
    p = pages.cpu()
    kb = p[..., :PAGE * d // 2].unflatten(-1, (PAGE, d // 2))
    vb = p[..., PAGE * d // 2:PAGE * d].unflatten(-1, (d // 2, PAGE)).transpose(-1, -2)
    ks = p[..., PAGE * d:PAGE * d + PAGE * (d // 32)].unflatten(-1, (PAGE, d // 32))
    vs = p[..., PAGE * d + PAGE * (d // 32):]
    return (numbers(unpack(kb)) * scales(ks).repeat_interleave(GROUP, -1),
            numbers(unpack(vb)) * scales(vs)[..., None])


def cache(pages: Tensor, d: int, table: Tensor, lengths):
    """Keys and values of every sequence ``[keys, heads, D]`` (keys of missing pages left out), and which of
    its positions they are."""
    k, v = split(pages, d)
    out = []
    for row, length in zip(table.tolist(), lengths.tolist()):
        length = min(max(length, 0), PAGE * len(row))
        at = [j for j in range(length) if 0 <= row[j // PAGE] < pages.shape[0]]
        ids = torch.tensor([row[j // PAGE] for j in at], dtype=torch.long)
        place = torch.tensor([j % PAGE for j in at], dtype=torch.long)
        out.append((k[ids, :, place], v[ids, :, place], torch.tensor(at, dtype=torch.long), length))
    return out


def attention(q: Tensor, pages: Tensor, table: Tensor, lengths: Tensor, cu_q=None, scale=None):
    """``(out, lse, mass, score_mass, keys)`` of a batch, as ``lm_oracle.prefix_attention``."""
    tokens, heads, d = q.shape
    n_kv, batch = pages.shape[1], len(lengths)
    scale = d ** -0.5 if scale is None else scale
    cu = [tokens // batch * b for b in range(batch + 1)] if cu_q is None else [int(c) for c in cu_q]
    out = torch.zeros(tokens, heads, d, dtype=torch.float64)
    mass, lse = torch.zeros_like(out), torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    score, keys = torch.zeros(tokens, heads, dtype=torch.float64), torch.zeros(tokens, heads)
    for b, (k, v, at, length) in enumerate(cache(pages, d, table, lengths)):
        n = cu[b + 1] - cu[b]
        visible = at <= (length - n + torch.arange(n))[:, None]
        rows = slice(cu[b], cu[b + 1])
        for h in range(heads):
            g = h // (heads // n_kv)
            out[rows, h], lse[rows, h], mass[rows, h], score[rows, h] = O.attention(
                q[rows, h], k[:, g], v[:, g], visible, scale)
            keys[rows, h] = visible.sum(1).float()
    return out, lse, mass, score, keys
