"""Cases of the speech language model's operators: the linear layer with its epilogue, per-head
norms with the rotation and the cache append, and attention over a prompt that a batch shares.

A case is one call that a decoder layer of the model that writes the speech tokens makes: a voice's
prompt (its reference text and speech tokens) is prefilled once, every request of that voice appends
to a cache of its own.  Lengths of a ragged case come from its ``layout`` number, tensors from the
seed.  Weights have the scale that keeps activations near one; the rotation's tables are the usual
base-10000 ones.
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
EPS = 1e-6


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


def _rope(tokens, sessions, capacity, heads, kv_heads, dim, rope_dim, norm, interleaved, dtype):
    return {"op": "rope", "tokens": tokens, "sessions": sessions, "capacity": capacity,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "rope_dim": rope_dim, "norm": norm,
            "interleaved": interleaved, "dtype": dtype}


def _attn(batch, prefix, own_lo, own_hi, q_lo, q_hi, heads, kv_heads, dim, dtype, lse=False,
          layout=0):
    return {"op": "attn", "batch": batch, "prefix": prefix, "own_lo": own_lo, "own_hi": own_hi,
            "q_lo": q_lo, "q_hi": q_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "lse": lse, "layout": layout}


def listed() -> list[dict]:
    cases = {
        # one token of one request through a feed-forward's first layer: latency alone
        "linear_token": _linear(1, 1024, 2048, "gelu_tanh", True, False, "fp16"),
        # a decode step of 32 requests through an output projection, added to the residual
        "linear_decode32": _linear(32, 4096, 4096, "none", False, True, "bf16"),
        # logits of 77 rows over the 6561 speech tokens, kept in fp32 for the sampler
        "linear_logits": _linear(77, 896, 6561, "none", True, False, "bf16", "fp32"),
        # the benchmark's 9184 packed rows through a feed-forward's first layer
        "linear_rows": _linear(9184, 1024, 2048, "gelu_tanh", True, False, "fp16"),
        # a large prefill: compute-bound
        "linear_prefill": _linear(8192, 4096, 8192, "silu", True, False, "bf16"),
        # one request's next token, keys without a norm
        "rope_token": _rope(1, 1, 512, 14, 2, 64, 64, False, False, "bf16"),
        # a decode step of 64 requests
        "rope_decode64": _rope(64, 64, 512, 32, 8, 128, 128, True, False, "bf16"),
        # a long prompt prefilled at once, half of each head rotated
        "rope_prefill": _rope(8191, 1, 8192, 32, 8, 128, 64, True, True, "fp16"),
        # one request's next token after a short prompt
        "attn_token": _attn(1, 512, 100, 100, 1, 1, 14, 2, 64, "bf16"),
        # a decode step of 32 requests of one voice, 2 to 24 s of speech each
        "attn_decode32": _attn(32, 1500, 50, 600, 1, 1, 14, 2, 64, "fp16", True, 1),
        # a decode step of 64 long requests behind a long prompt
        "attn_decode64": _attn(64, 8192, 200, 2000, 1, 1, 32, 8, 128, "bf16", False, 2),
        # four requests' texts (300 to 1024 tokens) appended behind a prompt: compute-bound
        "attn_extend": _attn(4, 4096, 300, 1024, 300, 1024, 32, 8, 128, "bf16", False, 3),
    }
    return [{"name": n, **c} for n, c in cases.items()]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2, 64), (16, 16, 64), (16, 4, 64), (32, 8, 128), (16, 2, 128), (12, 12, 128))
MAX_LINEAR_FLOPS = 2 * 8192 * 4096 * 8192
MAX_ROPE_TOKENS = 8191
MAX_ATTN = {"flops": 4.0e11, "bytes": 3.0e8}


def draw(rng: random.Random) -> dict:
    op = rng.choice(("linear", "rope", "attn"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "linear":
        while True:
            m, n = _spread(rng, 1, 9000), _spread(rng, 64, 9000)
            k = _spread(rng, 64, 9000)
            if rng.random() < 0.85:
                k = (k + 7) // 8 * 8
            if 2 * m * n * k <= MAX_LINEAR_FLOPS:
                return _linear(m, k, n, rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                               rng.random() < 0.5, rng.random() < 0.5, dtype,
                               rng.choice(("same", "same", "fp32")))
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "rope":
        tokens = _spread(rng, 1, MAX_ROPE_TOKENS)
        sessions = tokens if tokens <= 128 else 1
        return _rope(tokens, sessions, rng.randint(300, 600) if sessions > 1 else tokens + 100,
                     heads, kv_heads, dim, rng.choice((dim, dim // 2)), rng.random() < 0.7,
                     rng.random() < 0.5, dtype)
    while True:
        q_hi = rng.choice((1, 1, 1, rng.randint(2, 9), _spread(rng, 10, 1024)))
        q_lo = max(1, q_hi // 3)
        own_hi = max(q_hi, _spread(rng, 1, 2000))
        case = _attn(_spread(rng, 1, 64), _spread(rng, 1, 8192), max(q_hi, own_hi // 4), own_hi,
                     q_lo, q_hi, heads, kv_heads, dim, dtype, rng.random() < 0.3,
                     rng.randint(0, 10 ** 6))
        cost = work(case)
        if cost["flops"] <= MAX_ATTN["flops"] and cost["bytes"] <= MAX_ATTN["bytes"]:
            return case


def _layout(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and cached keys (the new ones among them) of every sequence of a batch."""
    rng = random.Random(case["layout"])
    news, keys = [], []
    for _ in range(case["batch"]):
        news.append(rng.randint(case["q_lo"], case["q_hi"]))
        keys.append(max(news[-1], rng.randint(case["own_lo"], case["own_hi"])))
    return news, keys


def work(case: dict) -> dict:
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * (m * k + n * k + (n if case["bias"] else 0)
                              + (m * n if case["residual"] else 0)) + size * m * n,
                "flops": 2 * m * n * k}
    d = case["dim"]
    if case["op"] == "rope":
        row = (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": case["tokens"] * (2 * 2 * row + 4 * case["rope_dim"] + 8),
                "flops": 8 * case["tokens"] * row}
    news, keys = _layout(case)
    pairs = sum(n * (case["prefix"] + k - n) + n * (n + 1) // 2 for n, k in zip(news, keys))
    rows = 2 * case["heads"] * d * sum(news)
    return {"bytes": 2 * rows + 2 * 2 * case["kv_heads"] * d * (case["prefix"] + sum(keys)),
            "flops": 4 * d * case["heads"] * pairs}


# ---- what a program has in hand before the call ------------------------------------------------


def _tables(rows: int, rope_dim: int):
    half = rope_dim // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / rope_dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(DEV), angle.sin().float().to(DEV)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)

    st = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st |= {"x": rand(m, k), "w": rand(n, k, scale=k ** -0.5),
               "b": rand(n, scale=0.5) if case["bias"] else None,
               "r": rand(m, n) if case["residual"] else None}
        return st
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        t, s, c = case["tokens"], case["sessions"], case["capacity"]
        cos, sin = _tables(c + 1000, case["rope_dim"])
        rng = random.Random(seed)
        if s > 1:  # every session's next position
            at = [rng.randrange(c) for _ in range(s)]
            rows = [i * c + p for i, p in enumerate(at)]
        else:      # one session's next positions
            first = rng.randint(0, c - t)
            at = list(range(first, first + t))
            rows = at
        st |= {"qkv": rand(t, (hq + 2 * hk) * d), "cos": cos, "sin": sin,
               "qw": 1 + rand(d, scale=0.2) if case["norm"] else None,
               "kw": 1 + rand(d, scale=0.2) if case["norm"] else None,
               "positions": torch.tensor(at, dtype=torch.int32, device=DEV) + 700,
               "rows": torch.tensor(rows, dtype=torch.int32, device=DEV),
               "k": rand(s, c, hk, d), "v": rand(s, c, hk, d)}
        return st
    news, keys = _layout(case)
    b, cap = case["batch"], (max(keys) + 63) // 64 * 64
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    slots = list(range(b))
    random.Random(seed).shuffle(slots)  # sessions sit anywhere in the cache

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    st |= {"q": rand(starts[-1], hq, d, scale=1.5), "pk": rand(case["prefix"], hk, d),
           "pv": rand(case["prefix"], hk, d), "k": rand(b, cap, hk, d), "v": rand(b, cap, hk, d),
           "lengths": ints(keys), "cu": ints(starts), "slots": ints(slots),
           "max_q": max(news), "max_length": max(keys)}
    return st


# ---- one pass ----------------------------------------------------------------------------------


def run(st: dict):
    return {"linear": run_linear, "rope": run_rope, "attn": run_attn}[st["case"]["op"]](st)


def run_linear(st: dict):
    case = st["case"]
    kind = torch.float32 if case["out"] == "fp32" else st["x"].dtype
    if own:
        return _fcv().fused_linear(st["x"], st["w"], st["b"], activation=case["act"],
                                   residual=st["r"], out_dtype=kind)
    y = st["x"].float() @ st["w"].float().t()
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
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    r = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., r:]), -1)


def run_rope(st: dict):
    case = st["case"]
    if own:
        q = _fcv().qk_norm_rope(st["qkv"], st["positions"], st["cos"], st["sin"], st["k"], st["v"],
                                st["rows"], n_heads=case["heads"], q_weight=st["qw"],
                                k_weight=st["kw"], eps=EPS, interleaved=case["interleaved"])
        return q, st["k"], st["v"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = st["qkv"].view(-1, hq + 2 * hk, d).split((hq, hk, hk), 1)
    at = st["positions"].long()
    cos, sin = st["cos"][at], st["sin"][at]
    q = _norm_rotate(q.float(), st["qw"], cos, sin, case["interleaved"]).to(st["qkv"].dtype)
    k = _norm_rotate(k.float(), st["kw"], cos, sin, case["interleaved"]).to(st["qkv"].dtype)
    rows = st["rows"].long()
    st["k"].view(-1, hk, d).index_copy_(0, rows, k)
    st["v"].view(-1, hk, d).index_copy_(0, rows, v)
    return q, st["k"], st["v"]


def run_attn(st: dict):
    case = st["case"]
    if own:
        return _fcv().prefix_attention(
            st["q"], st["k"], st["v"], st["lengths"], prefix_k=st["pk"], prefix_v=st["pv"],
            cu_q=st["cu"], max_q=st["max_q"], slots=st["slots"], max_length=st["max_length"],
            return_lse=case["lse"])
    hk, d = case["kv_heads"], case["dim"]
    group, b, mq, ml = case["heads"] // hk, case["batch"], st["max_q"], st["max_length"]
    cu, lengths = st["cu"].long(), st["lengths"].long()
    news = cu[1:] - cu[:-1]
    i, j = torch.arange(mq, device=DEV), torch.arange(ml, device=DEV)
    at = (cu[:-1, None] + i).clamp_max(st["q"].shape[0] - 1)          # [b, mq] rows of q
    q = st["q"][at].float() * d ** -0.5                                # [b, mq, hq, d]
    q = q.view(b, mq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * mq, d)
    k = st["k"][st["slots"].long(), :ml].float().permute(0, 2, 3, 1).contiguous()
    v = st["v"][st["slots"].long(), :ml].float().permute(0, 2, 1, 3).contiguous()
    seen = j <= (lengths - news)[:, None, None] + i[:, None]           # [b, mq, ml]
    s = (q @ k).view(b, hk, group, mq, ml)
    s = s.masked_fill(~seen[:, None, None], -math.inf).view(b, hk, group * mq, ml)
    flat = q.transpose(0, 1).reshape(hk, b * group * mq, d)            # one product for the batch
    pre = flat @ st["pk"].float().permute(1, 2, 0).contiguous()
    m = pre.amax(-1).view(hk, b, -1).transpose(0, 1)                   # [b, hk, rows]
    m = torch.maximum(m, s.amax(-1))[..., None]
    s = torch.exp(s - m)
    pre = torch.exp(pre - m.transpose(0, 1).reshape(hk, -1, 1))
    o = pre @ st["pv"].float().transpose(0, 1).contiguous()
    o = o.view(hk, b, -1, d).transpose(0, 1) + s @ v
    l = s.sum(-1) + pre.sum(-1).view(hk, b, -1).transpose(0, 1)
    o = (o / l[..., None]).view(b, hk, group, mq, d).permute(0, 3, 1, 2, 4).flatten(2, 3)
    row = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu, row, right=True) - 1                  # sequence of each row
    o = o[seq, row - cu[seq]].to(st["q"].dtype)
    if not case["lse"]:
        return o
    lse = (m[..., 0] + torch.log(l)).view(b, hk, group, mq).permute(0, 3, 1, 2).flatten(2, 3)
    return o, lse[seq, row - cu[seq]]


# ---- the definition in 64 bits -----------------------------------------------------------------


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"linear": exact_linear, "rope": exact_rope, "attn": exact_attn}[case["op"]](case, st)


def exact_linear(case, st):
    y = torch.mm(st["x"].double(), st["w"].double().t().contiguous())
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


def exact_rope(case, st):
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
    k_cache, v_cache = st["k"].double(), st["v"].double()
    rows = st["rows"].long()
    k_cache.view(-1, hk, d)[rows] = out[1]
    v_cache.view(-1, hk, d)[rows] = v
    return out[0], k_cache, v_cache


def exact_attn(case, st):
    news, keys = _layout(case)
    hq, hk, d, p = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    group = hq // hk
    slots = st["slots"].tolist()
    o = torch.empty(sum(news), hq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(sum(news), hq, dtype=torch.float64, device=DEV)
    for h in range(hk):
        first = 0
        pk, pv = st["pk"][:, h].double(), st["pv"][:, h].double()
        for n, length, slot in zip(news, keys, slots):
            q = st["q"][first:first + n, h * group:(h + 1) * group].double().reshape(-1, d)
            k = torch.cat((pk, st["k"][slot, :length, h].double()))
            v = torch.cat((pv, st["v"][slot, :length, h].double()))
            s = q @ k.t().contiguous() / math.sqrt(d)
            last = torch.arange(n, device=DEV).repeat_interleave(group) + p + length - n
            s[torch.arange(p + length, device=DEV) > last[:, None]] = -math.inf
            o[first:first + n, h * group:(h + 1) * group] = (s.softmax(-1) @ v).view(n, group, d)
            lse[first:first + n, h * group:(h + 1) * group] = s.logsumexp(-1).view(n, group)
            first += n
    return (o, lse) if case["lse"] else o
