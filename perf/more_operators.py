"""Cases of the speech language model's operators in 4 bits: the linear layer over 4-bit weights, the
rotation with the append to a cache of 4-bit pages, attention over such pages, and copies of pages.

A 4-bit number is one sign bit and a magnitude out of 0, 1/2, 1, 3/2, 2, 3, 4, 6; a group of them has a
scale of 2^(b - 127), one byte b.  The group's exponent e is the smallest with every magnitude below
7 2^e, within what the 16-bit type of the call represents; values go to the nearest number, ties to the
even code, 6 at most.  Weights and keys have groups of 32 along a row, a head's value has one group.

A page holds 64 tokens' keys and values of every key head.  Its bytes per head are: keys [64][D / 2], values
[D / 2][64] (byte j of a token has elements 2 j, 2 j + 1, the first in the low half), the keys' scales
[64][D / 32], the values' scales [64].

A case is one call of a server that speaks with many voices: a decoder layer's product, append or
attention, or a fork or a compaction of the cache.  Lengths of a ragged case come from its ``layout``
number, tensors from the seed.
"""

from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

REPO = Path(__file__).resolve().parent.parent
PKG = "faster_cosyvoice_amd"
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EXPONENTS = {"bf16": (-125, 125), "fp16": (-23, 13)}  # every number times 2^e is one of the type's
EPS = 1e-6
PAGE = 64


def _fcv():
    if PKG not in sys.modules:
        d = REPO / "faster-cosyvoice_amd"
        spec = importlib.util.spec_from_file_location(PKG, d / "__init__.py",
                                                      submodule_search_locations=[str(d)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[PKG] = mod
        spec.loader.exec_module(mod)
    return sys.modules[PKG]


# ---- the cases ---------------------------------------------------------------------------------


def _linear(m, k, n, act, bias, residual, dtype, out="same"):
    return {"op": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual, "dtype": dtype, "out": out}


def _append(tokens, sessions, heads, kv_heads, dim, rope_dim, norm, interleaved, dtype):
    return {"op": "append", "tokens": tokens, "sessions": sessions, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rope_dim": rope_dim, "norm": norm,
            "interleaved": interleaved, "dtype": dtype}


def _attend(batch, shared, own_lo, own_hi, q_lo, q_hi, heads, kv_heads, dim, dtype, lse=False,
            layout=0):
    return {"op": "attend", "batch": batch, "shared": shared, "own_lo": own_lo, "own_hi": own_hi,
            "q_lo": q_lo, "q_hi": q_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "lse": lse, "layout": layout}


def _pages(layers, pages, kv_heads, dim, moves, kind):
    return {"op": "pages", "layers": layers, "pages": pages, "kv_heads": kv_heads, "dim": dim,
            "moves": moves, "kind": kind}


def listed() -> list[dict]:
    cases = {
        # one token of one request through a feed-forward's first layer: latency alone
        "linear4_token": _linear(1, 1024, 2048, "gelu_tanh", True, False, "fp16"),
        # a decode step of 32 requests through an output projection, added to the residual
        "linear4_decode32": _linear(32, 4096, 4096, "none", False, True, "bf16"),
        # logits of 77 rows over the 6561 speech tokens, kept in fp32 for the sampler
        "linear4_logits": _linear(77, 896, 6561, "none", True, False, "bf16", "fp32"),
        # a large prefill: compute-bound
        "linear4_prefill": _linear(8192, 4096, 8192, "silu", True, False, "bf16"),
        # one request's next token, keys without a norm
        "append4_token": _append(1, 1, 14, 2, 64, 64, False, False, "bf16"),
        # a decode step of 64 requests
        "append4_decode64": _append(64, 64, 32, 8, 128, 128, True, False, "bf16"),
        # a long prompt prefilled at once, half of each head rotated
        "append4_prefill": _append(8191, 1, 32, 8, 128, 64, True, True, "fp16"),
        # one request's next token after a short prompt
        "attend4_token": _attend(1, 512, 100, 100, 1, 1, 14, 2, 64, "bf16"),
        # a decode step of 64 long requests, a quarter of whose keys is a voice's prompt that all share
        "attend4_decode64": _attend(64, 1024, 1000, 7000, 1, 1, 32, 8, 128, "bf16", False, 1),
        # four requests' texts (300 to 1024 tokens) appended behind a prompt: compute-bound
        "attend4_extend": _attend(4, 4096, 300, 1024, 300, 1024, 32, 8, 128, "bf16", True, 2),
        # a voice's last, partly filled page copied for 8 new requests, in all layers
        "pages_fork": _pages(24, 64, 2, 64, 8, "fork"),
        # a cache after many requests have ended: 256 pages moved to the front, in all layers
        "pages_compact": _pages(16, 600, 8, 128, 256, "compact"),
    }
    return [{"name": n, **c} for n, c in cases.items()]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2, 64), (16, 16, 64), (16, 4, 64), (32, 8, 128), (16, 2, 128), (12, 12, 128))
MAX_LINEAR_FLOPS = 2 * 8192 * 4096 * 8192
MAX_ATTEND = {"flops": 1.2e11, "bytes": 2.5e8}
MAX_PAGES_BYTES = 5.0e8


def draw(rng: random.Random) -> dict:
    op = rng.choice(("linear", "append", "attend", "pages"))
    dtype = rng.choice(("bf16", "fp16"))
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "linear":
        while True:
            m, n = _spread(rng, 1, 9000), _spread(rng, 64, 9000)
            k = _spread(rng, 64, 9000)
            if rng.random() < 0.85:
                k = (k + 31) // 32 * 32
            if 2 * m * n * k <= MAX_LINEAR_FLOPS:
                return _linear(m, k, n, rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                               rng.random() < 0.5, rng.random() < 0.5, dtype,
                               rng.choice(("same", "same", "fp32")))
    if op == "append":
        tokens = _spread(rng, 1, 8191)
        return _append(tokens, tokens if tokens <= 128 else 1, heads, kv_heads, dim,
                       rng.choice((dim, dim // 2)), rng.random() < 0.7, rng.random() < 0.5, dtype)
    while op == "attend":
        q_hi = rng.choice((1, 1, 1, rng.randint(2, 9), _spread(rng, 10, 1024)))
        q_lo = max(1, q_hi // 3)
        own_hi = max(q_hi, _spread(rng, 1, 7000))
        case = _attend(_spread(rng, 1, 64), rng.choice((0, PAGE * _spread(rng, 1, 64))),
                       max(q_hi, own_hi // 4), own_hi, q_lo, q_hi, heads, kv_heads, dim, dtype,
                       rng.random() < 0.3, rng.randint(0, 10 ** 6))
        cost = work(case)
        if cost["flops"] <= MAX_ATTEND["flops"] and cost["bytes"] <= MAX_ATTEND["bytes"]:
            return case
    while True:
        kind, moves = rng.choice(("fork", "compact")), _spread(rng, 1, 500)
        case = _pages(_spread(rng, 1, 32), 2 * moves + _spread(rng, 1, 100), kv_heads, dim, moves,
                      kind)
        if work(case)["bytes"] <= MAX_PAGES_BYTES:
            return case


def _layout(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and keys behind the shared ones (the new ones among them) of every sequence."""
    rng = random.Random(case["layout"])
    news, keys = [], []
    for _ in range(case["batch"]):
        news.append(rng.randint(case["q_lo"], case["q_hi"]))
        keys.append(max(news[-1], rng.randint(case["own_lo"], case["own_hi"])))
    return news, keys


def _page_bytes(d: int) -> int:
    return PAGE * (d + d // 32 + 1)


def work(case: dict) -> dict:
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = (k + 31) // 32
        size = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * (m * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0))
                + 17 * n * groups + size * m * n, "flops": 2 * m * n * k}
    d = case["dim"]
    token = case["kv_heads"] * _page_bytes(d) // PAGE  # bytes of a token's keys and values in a page
    if case["op"] == "append":  # its values are returned, too
        row = (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": case["tokens"] * (2 * 2 * row + 4 * case["rope_dim"] + 8 + token),
                "flops": 8 * case["tokens"] * row}
    if case["op"] == "pages":
        moved = case["moves"] * case["layers"] * case["kv_heads"] * _page_bytes(d)
        return {"bytes": moved + (moved if case["kind"] == "compact" else moved // case["moves"]),
                "flops": 0}
    news, keys = _layout(case)
    pairs = sum(n * (case["shared"] + k - n) + n * (n + 1) // 2 for n, k in zip(news, keys))
    rows = 2 * case["heads"] * d * sum(news)
    return {"bytes": 2 * rows + token * (case["shared"] + sum(keys)),
            "flops": 4 * d * case["heads"] * pairs}


# ---- 4-bit numbers and pages, in elementary operations -------------------------------------------


def _quantize(x, limits):
    """Codes 0 .. 15 and scale bytes of groups that lie along the last dimension."""
    amax = x.abs().amax(-1, keepdim=True)
    f, e = torch.frexp(amax)
    e = torch.where(f < 0.875, e - 3, e - 2).clamp(*limits)  # amax < 7 2^e
    y = torch.ldexp(x.abs(), -e)
    code = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (y >= border) if i % 2 else (y > border)
    return code + 8 * (x < 0).to(torch.uint8), (e[..., 0] + 127).to(torch.uint8)


def _numbers(codes):
    table = torch.tensor((0, 0.5, 1, 1.5, 2, 3, 4, 6), device=codes.device)
    return torch.cat((table, -table))[codes.long()]


def _halves(b):
    """The two codes of every byte, along the last dimension."""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _scales(b):
    return torch.exp2(b.float() - 127)


def _split(pages, d):
    """Views of a page's parts: keys [.., 64, D / 2], values [.., D / 2, 64], their scales."""
    k, v, ks, vs = pages.split((PAGE * d // 2, PAGE * d // 2, PAGE * d // 32, PAGE), -1)
    return (k.unflatten(-1, (PAGE, d // 2)), v.unflatten(-1, (d // 2, PAGE)),
            ks.unflatten(-1, (PAGE, d // 32)), vs)


def _page_values(pages, d):
    """Keys and values [.., 64, D] of pages, in 32 bits."""
    k, v, ks, vs = _split(pages, d)
    k = (_numbers(_halves(k)).unflatten(-1, (d // 32, 32)) * _scales(ks)[..., None]).flatten(-2)
    return k, _numbers(_halves(v.transpose(-1, -2))) * _scales(vs)[..., None]


# ---- what a program has in hand before the call ------------------------------------------------


def _tables(rows: int, rope_dim: int):
    half = rope_dim // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / rope_dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(DEV), angle.sin().float().to(DEV)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _random_pages(n, hk, d, g, limits):
    """A pool whose pages hold normal keys and values."""
    pages = torch.empty(n, hk, _page_bytes(d), dtype=torch.uint8, device=DEV)
    for at in range(0, n, 512):
        part = pages[at:at + 512]
        k, v, ks, vs = _split(part, d)
        x = torch.randn(2, *part.shape[:2], PAGE, d, generator=g, device=DEV)
        c, s = _quantize(x[0].unflatten(-1, (d // 32, 32)), limits)
        c = c.flatten(-2)
        k.copy_(c[..., 0::2] | c[..., 1::2] << 4)
        ks.copy_(s)
        c, s = _quantize(x[1], limits)
        v.copy_((c[..., 0::2] | c[..., 1::2] << 4).transpose(-1, -2))
        vs.copy_(s)
    return pages


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": case}
    if case["op"] == "pages":
        n, moves = case["pages"], case["moves"]
        order = list(range(n))
        rng.shuffle(order)
        if case["kind"] == "fork":
            src, dst = [order[0]] * moves, order[1:moves + 1]
        else:  # the last pages in use move to the first free ones
            free, used = sorted(order[:n - moves]), sorted(order[n - moves:])
            src, dst = used[::-1], free[:moves]
        st |= {"src": src, "dst": dst,
               "pages": torch.randint(0, 256, (case["layers"], n, case["kv_heads"],
                                               _page_bytes(case["dim"])), generator=g, device=DEV,
                                      dtype=torch.uint8)}
        return st
    dt, limits = DTYPES[case["dtype"]], EXPONENTS[case["dtype"]]

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = (k + 31) // 32
        w = torch.zeros(n, 32 * groups, device=DEV)
        w[:, :k] = rand(n, k, scale=k ** -0.5)
        codes, scales = _quantize(w.view(n, groups, 32), limits)
        codes = codes.flatten(1)
        st |= {"x": rand(m, k), "codes": codes[:, 0::2] | codes[:, 1::2] << 4, "scales": scales,
               "b": rand(n, scale=0.5) if case["bias"] else None,
               "r": rand(m, n) if case["residual"] else None}
        return st
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        t, s = case["tokens"], case["sessions"]
        cos, sin = _tables(t + 2000, case["rope_dim"])
        if s > 1:  # every session's next position, in a page of its own
            n, at = s + 3, [rng.randrange(1000) for _ in range(s)]
            ids = rng.sample(range(n), s)
            rows = [i * PAGE + p % PAGE for i, p in zip(ids, at)]
        else:      # one session's next positions
            first = rng.randrange(500)
            at = list(range(first, first + t))
            n = at[-1] // PAGE + 4
            ids = rng.sample(range(n), at[-1] // PAGE + 1)
            rows = [ids[p // PAGE] * PAGE + p % PAGE for p in at]
        st |= {"qkv": rand(t, (hq + 2 * hk) * d), "cos": cos, "sin": sin,
               "qw": 1 + rand(d, scale=0.2) if case["norm"] else None,
               "kw": 1 + rand(d, scale=0.2) if case["norm"] else None,
               "positions": _ints(at) + 700, "rows": _ints(rows),
               "pages": torch.zeros(n, hk, _page_bytes(d), dtype=torch.uint8, device=DEV)}
        return st
    news, keys = _layout(case)
    first = case["shared"] // PAGE  # the shared pages are the first of every sequence
    counts = [(k + PAGE - 1) // PAGE for k in keys]
    n = first + sum(counts) + 2
    ids = rng.sample(range(n), n)   # pages sit anywhere
    table, used = [], first
    for c in counts:
        row = ids[:first] + ids[used:used + c]
        table.append(row + [-1] * (first + max(counts) - len(row)))
        used += c
    starts = [0]
    for q in news:
        starts.append(starts[-1] + q)
    st |= {"q": rand(starts[-1], hq, d, scale=1.5), "pages": _random_pages(n, hk, d, g, limits),
           "table": _ints(table), "lengths": _ints([case["shared"] + k for k in keys]),
           "cu": _ints(starts), "max_q": max(news), "max_length": case["shared"] + max(keys)}
    return st


# ---- one pass ----------------------------------------------------------------------------------


def run(st: dict):
    return {"linear": run_linear, "append": run_append, "attend": run_attend,
            "pages": run_pages}[st["case"]["op"]](st)


def run_linear(st: dict):
    case = st["case"]
    kind = torch.float32 if case["out"] == "fp32" else st["x"].dtype
    if own:
        return _fcv().fused_linear_fp4(st["x"], st["codes"], st["scales"], st["b"],
                                       activation=case["act"], residual=st["r"], out_dtype=kind)
    w = _numbers(_halves(st["codes"])).unflatten(-1, (-1, 32)) * _scales(st["scales"])[..., None]
    y = st["x"].float() @ w.flatten(1)[:, :case["k"]].t()
    if st["b"] is not None:
        y = y + st["b"].float()
    if case["act"] == "relu":
        y = y.clamp_min(0)
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))
    elif case["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if st["r"] is not None:
        y = y + st["r"].float()
    return y.to(kind)


def _norm_rotate(x, w, cos, sin, interleaved):
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    r = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., r:]), -1)


def run_append(st: dict):
    """The queries, and the appended keys and values as the cache holds them."""
    case = st["case"]
    if own:
        q = _fcv().qk_norm_rope_fp4(st["qkv"], st["positions"], st["cos"], st["sin"], st["pages"],
                                    st["rows"], n_heads=case["heads"], q_weight=st["qw"],
                                    k_weight=st["kw"], eps=EPS, interleaved=case["interleaved"])
        k, v = _fcv().read_fp4_pages(st["pages"], st["rows"], dtype=st["qkv"].dtype)
        return q, k, v
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    # a value next to a border of two 4-bit numbers: in 64 bits
    q, k, v = st["qkv"].double().view(-1, hq + 2 * hk, d).split((hq, hk, hk), 1)
    at, dt = st["positions"].long(), st["qkv"].dtype
    cos, sin = st["cos"][at].double(), st["sin"][at].double()
    weights = (None, None) if st["qw"] is None else (st["qw"].double(), st["kw"].double())
    q = _norm_rotate(q, weights[0], cos, sin, case["interleaved"]).to(dt)
    k = _norm_rotate(k, weights[1], cos, sin, case["interleaved"])
    limits = EXPONENTS[case["dtype"]]
    kc, ke = _quantize(k.unflatten(-1, (d // 32, 32)), limits)
    kc = kc.flatten(-2)
    vc, ve = _quantize(v, limits)
    page, key = st["rows"].long() // PAGE, st["rows"].long() % PAGE
    pk, pv, pks, pvs = _split(st["pages"], d)
    pk[page, :, key] = kc[..., 0::2] | kc[..., 1::2] << 4
    pv[page, :, :, key] = vc[..., 0::2] | vc[..., 1::2] << 4
    pks[page, :, key] = ke
    pvs[page, :, key] = ve
    k = (_numbers(_halves(pk[page, :, key])).unflatten(-1, (d // 32, 32))
         * _scales(pks[page, :, key])[..., None]).flatten(-2)
    v = _numbers(_halves(pv[page, :, :, key])) * _scales(pvs[page, :, key])[..., None]
    return q, k.to(dt), v.to(dt)


def run_attend(st: dict):
    case = st["case"]
    if own:
        return _fcv().paged_attention_fp4(st["q"], st["pages"], st["table"], st["lengths"],
                                          cu_q=st["cu"], max_q=st["max_q"],
                                          max_length=st["max_length"], return_lse=case["lse"])
    hk, d = case["kv_heads"], case["dim"]
    group, b, mq = case["heads"] // hk, case["batch"], st["max_q"]
    cu, lengths = st["cu"].long(), st["lengths"].long()
    news = cu[1:] - cu[:-1]
    k, v = _page_values(st["pages"][st["table"].clamp_min(0).long()], d)  # [b, pages, hk, 64, d]
    k = k.transpose(1, 2).flatten(2, 3).transpose(-1, -2).contiguous()    # [b, hk, d, keys]
    v = v.transpose(1, 2).flatten(2, 3)
    i, j = torch.arange(mq, device=DEV), torch.arange(k.shape[-1], device=DEV)
    at = (cu[:-1, None] + i).clamp_max(st["q"].shape[0] - 1)              # [b, mq] rows of q
    q = st["q"][at].float() * d ** -0.5
    q = q.view(b, mq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * mq, d)
    seen = j <= (lengths - news)[:, None, None] + i[:, None]              # [b, mq, keys]
    s = (q @ k).view(b, hk, group, mq, -1).masked_fill(~seen[:, None, None], -math.inf).flatten(2, 3)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - m)
    l = s.sum(-1, keepdim=True)
    o = (s @ v / l).view(b, hk, group, mq, d).permute(0, 3, 1, 2, 4).flatten(2, 3)
    row = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu, row, right=True) - 1                     # sequence of each row
    o = o[seq, row - cu[seq]].to(st["q"].dtype)
    if not case["lse"]:
        return o
    lse = (m + torch.log(l)).view(b, hk, group, mq).permute(0, 3, 1, 2).flatten(2, 3)
    return o, lse[seq, row - cu[seq]]


def run_pages(st: dict):
    if own:
        _fcv().copy_pages(st["pages"], st["src"], st["dst"])
        return st["pages"]
    src = torch.tensor(st["src"], device=DEV)
    dst = torch.tensor(st["dst"], device=DEV)
    st["pages"].index_copy_(1, dst, st["pages"].index_select(1, src))
    return st["pages"]


# ---- the definition in 64 bits -----------------------------------------------------------------


def exact(case: dict, seed: int):
    if case["op"] == "pages":
        return None  # bytes: the plain form has them
    st = prepare(case, seed)
    return {"linear": exact_linear, "append": exact_append, "attend": exact_attend}[case["op"]](
        case, st)


def _value(code):
    """A code's number in 64 bits, from its bits: exponent 2, mantissa 1, as the format has them."""
    sign, e, m = code >> 3 & 1, code >> 1 & 3, code & 1
    big = torch.ldexp(1 + 0.5 * m.double(), e.double() - 1)
    return torch.where(e == 0, 0.5 * m.double(), big) * (1 - 2 * sign.double())


def _power(b):
    return torch.ldexp(torch.ones(b.shape, dtype=torch.float64, device=b.device), b.double() - 127)


def exact_linear(case, st):
    n, k = case["n"], case["k"]
    c = st["codes"].long()
    w = torch.empty(n, 2 * c.shape[1], dtype=torch.float64, device=DEV)
    w[:, 0::2], w[:, 1::2] = _value(c % 16), _value(c // 16)
    w *= _power(st["scales"]).repeat_interleave(32, 1)
    y = torch.mm(st["x"].double(), w[:, :k].t().contiguous())
    if case["bias"]:
        y += st["b"].double()
    if case["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = torch.nn.functional.gelu(y)
    elif case["act"] == "gelu_tanh":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    if case["residual"]:
        y += st["r"].double()
    return y


def _nearest(x, lo, hi):
    """The 4-bit numbers nearest to groups along the last dimension, times their scale."""
    _, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 7)  # amax < 7 2^e, and not 7 2^(e - 1)
    scale = torch.ldexp(torch.ones_like(x[..., :1]), e.double().clamp(lo, hi))
    y = x / scale
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    return (torch.round(y / step) * step).clamp(-6, 6) * scale  # round: ties to even


def exact_append(case, st):
    hq, hk, d, r = case["heads"], case["kv_heads"], case["dim"], case["rope_dim"]
    x = st["qkv"].double().view(case["tokens"], hq + 2 * hk, d)
    q, k, v = x[:, :hq].clone(), x[:, hq:hq + hk].clone(), x[:, hq + hk:]
    at = st["positions"].long()
    turn = torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, None]  # [t, 1, r/2]
    out = []
    for t, w in ((q, st["qw"]), (k, st["kw"])):
        if case["norm"]:
            rms = ((t * t).sum(-1, keepdim=True) / d + EPS).sqrt()
            t = t / rms * w.double()
        if case["interleaved"]:
            z = torch.view_as_complex(t[..., :r].reshape(*t.shape[:2], r // 2, 2).contiguous())
            t[..., :r] = torch.view_as_real(z * turn).flatten(-2)
        else:
            z = torch.complex(t[..., :r // 2].contiguous(), t[..., r // 2:r].contiguous()) * turn
            t[..., :r // 2], t[..., r // 2:r] = z.real, z.imag
        out.append(t)
    lo, hi = EXPONENTS[case["dtype"]]
    k = _nearest(out[1].view(-1, hk, d // 32, 32), lo, hi).flatten(-2)
    return out[0], k, _nearest(v, lo, hi)


def exact_attend(case, st):
    news, keys = _layout(case)
    hq, hk, d, shared = case["heads"], case["kv_heads"], case["dim"], case["shared"]
    group = hq // hk
    o = torch.empty(sum(news), hq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(sum(news), hq, dtype=torch.float64, device=DEV)
    first = 0
    for b, (n, length) in enumerate(zip(news, keys)):
        length += shared
        count = (length + PAGE - 1) // PAGE
        p = st["pages"][st["table"][b, :count].long()].long()  # [pages, hk, bytes]
        ends = (PAGE * d // 2, PAGE * d, PAGE * (d + d // 32))
        kb = p[..., :ends[0]].view(count, hk, PAGE, d // 2)
        vb = p[..., ends[0]:ends[1]].view(count, hk, d // 2, PAGE).permute(0, 1, 3, 2)
        ks = p[..., ends[1]:ends[2]].view(count, hk, PAGE, d // 32)
        k = torch.empty(count, hk, PAGE, d, dtype=torch.float64, device=DEV)
        v = torch.empty_like(k)
        k[..., 0::2], k[..., 1::2] = _value(kb % 16), _value(kb // 16)
        v[..., 0::2], v[..., 1::2] = _value(vb % 16), _value(vb // 16)
        k *= _power(ks).repeat_interleave(32, -1)
        v *= _power(p[..., ends[2]:])[..., None]
        k = k.transpose(0, 1).reshape(hk, -1, d)[:, :length]
        v = v.transpose(0, 1).reshape(hk, -1, d)[:, :length]
        last = torch.arange(n, device=DEV).repeat_interleave(group) + length - n
        hidden = torch.arange(length, device=DEV) > last[:, None]
        for h in range(hk):
            q = st["q"][first:first + n, h * group:(h + 1) * group].double().reshape(-1, d)
            s = q @ k[h].t().contiguous() / math.sqrt(d)
            s[hidden] = -math.inf
            o[first:first + n, h * group:(h + 1) * group] = (s.softmax(-1) @ v[h]).view(n, group, d)
            lse[first:first + n, h * group:(h + 1) * group] = s.logsumexp(-1).view(n, group)
        first += n
    return (o, lse) if case["lse"] else o
