"""64-bit CPU restatement of the speech language model's operators (include/fcv_lm.h).

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  Each function returns the exact result of its
formula on the given (already rounded) inputs, and the magnitudes that the rounding errors of a
fp32 computation scale with, so that a test's tolerance can be counted in roundings.
"""

from __future__ import annotations

import math

import torch

Tensor = torch.Tensor


def activate(z: Tensor, kind: str | None) -> Tensor:
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def linear(x: Tensor, w: Tensor, bias=None, activation=None, residual=None):
    """``(y, z, mass)``: the result, the activation's argument and ``sum |x w| + |bias|``."""
    x, w = x.double().cpu(), w.double().cpu()
    z, mass = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, mass = z + bias.double().cpu(), mass + bias.double().cpu().abs()
    y = activate(z, activation)
    if residual is not None:
        y = y + residual.double().cpu()
    return y, z, mass


def norm_rope(x: Tensor, weight, eps: float, cos: Tensor, sin: Tensor, interleaved: bool):
    """``(y, size)`` for heads ``x`` ``[T, H, D]`` and table rows ``cos``/``sin`` ``[T, R / 2]``;
    ``size`` is ``|a| + |b|`` of the rotated pair (``|y|`` where nothing is rotated)."""
    x, c, s = x.double().cpu(), cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double().cpu()
    y, size, r = x.clone(), x.abs(), 2 * c.shape[-1]
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2),
                                                                  slice(r // 2, r))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo] = size[..., hi] = a.abs() + b.abs()
    return y, size


def attention(q: Tensor, k: Tensor, v: Tensor, visible: Tensor, scale: float):
    """One head of one sequence: ``q`` ``[n, D]``, ``k``/``v`` ``[keys, D]``, ``visible``
    ``[n, keys]``.  ``(out, lse, mass, score_mass)``: ``mass`` is the softmax-weighted ``|v|``,
    ``score_mass`` the largest ``scale * sum |q k|`` of a row's visible keys.  Hidden keys and
    values are left out, whatever they hold."""
    q, k, v, visible = q.double().cpu(), k.double().cpu(), v.double().cpu(), visible.cpu()
    out, mass = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64), None
    mass = torch.zeros_like(out)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    score = torch.zeros(q.shape[0], dtype=torch.float64)
    for i in range(q.shape[0]):
        kk, vv = k[visible[i]], v[visible[i]]
        if not len(kk):
            continue
        s = scale * (kk @ q[i])
        p = torch.softmax(s, 0)
        out[i], lse[i] = p @ vv, torch.logsumexp(s, 0)
        mass[i], score[i] = p @ vv.abs(), scale * (kk.abs() @ q[i].abs()).max()
    return out, lse, mass, score


def prefix_attention(q, k_cache, v_cache, lengths, prefix_k=None, prefix_v=None, cu_q=None,
                     slots=None, scale=None):
    """``(out, lse, mass, score_mass, keys)`` of a batch, rows past the last sequence zero; ``keys``
    counts a row's visible ones."""
    tokens, heads, dim = q.shape
    n_kv, batch = k_cache.shape[2], len(lengths)
    scale = dim ** -0.5 if scale is None else scale
    cu = [tokens // batch * b for b in range(batch + 1)] if cu_q is None else [int(c) for c in cu_q]
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    mass, lse = torch.zeros_like(out), torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    score, keys = torch.zeros(tokens, heads, dtype=torch.float64), torch.zeros(tokens, heads)
    for b in range(batch):
        n = cu[b + 1] - cu[b]
        slot = b if slots is None else int(slots[b])
        length = min(max(int(lengths[b]), 0), k_cache.shape[1])
        length = length if 0 <= slot < k_cache.shape[0] else 0
        for h in range(heads):
            g = h // (heads // n_kv)
            k, v = k_cache[slot if length else 0, :length, g], v_cache[slot if length else 0, :length, g]
            p = 0
            if prefix_k is not None:
                p = prefix_k.shape[0]
                k, v = torch.cat((prefix_k[:, g], k)), torch.cat((prefix_v[:, g], v))
            last = p + length - n + torch.arange(n)
            at = torch.arange(p + length)
            visible = (at <= last[:, None]) | (at < p)
            rows = slice(cu[b], cu[b + 1])
            out[rows, h], lse[rows, h], mass[rows, h], score[rows, h] = attention(
                q[rows, h], k, v, visible, scale)
            keys[rows, h] = visible.sum(1).float()
    return out, lse, mass, score, keys
