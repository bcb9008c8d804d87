"""``qk_norm_rope`` against its formula in 64 bits: both rotations, partial ones, caches at other
strides, padding rows, positions past the tables."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def make(fcv, tokens, hq, hk, dim, rope_dim, dtype, seed=0, sessions=3, capacity=50, max_pos=400):
    g = torch.Generator().manual_seed(seed + tokens)
    qkv = torch.randn(tokens, (hq + 2 * hk) * dim, generator=g).to(dtype).to(DEV)
    cos, sin = fcv.rope_tables(max_pos, rope_dim, rope_dim)
    pos = torch.randint(0, max_pos, (tokens,), generator=g, dtype=torch.int32)
    rows = torch.randperm(sessions * capacity, generator=g)[:tokens].to(torch.int32)
    k, v = (torch.randn(sessions, capacity, hk, dim, generator=g).to(dtype).to(DEV)
            for _ in range(2))
    qw, kw = (1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2))
    return qkv, pos.to(DEV), cos.to(DEV), sin.to(DEV), k, v, rows.to(DEV), qw.to(DEV), kw.to(DEV)


def check(fcv, qkv, pos, cos, sin, k, v, rows, hq, qw, kw, interleaved, what, **kw_args):
    s, c, hk, dim = k.shape
    dtype, tokens = qkv.dtype, qkv.shape[0]
    k0, v0 = k.clone(), v.clone()
    got = fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, n_heads=hq, q_weight=qw, k_weight=kw,
                           eps=EPS, interleaved=interleaved, **kw_args)
    heads = qkv.reshape(tokens, hq + 2 * hk, dim).cpu()
    at = pos.cpu().long().clamp(0, cos.shape[0] - 1)
    y, size = O.norm_rope(heads[:, :hq], qw, EPS, cos.cpu()[at], sin.cpu()[at], interleaved)
    bars.assert_within(got, y, bars.norm_rope(y, size, dim, qw is not None, dtype), what + " q")
    y, size = O.norm_rope(heads[:, hq:hq + hk], kw, EPS, cos.cpu()[at], sin.cpu()[at], interleaved)
    tol = bars.norm_rope(y, size, dim, qw is not None, dtype)
    named = [(t, int(r)) for t, r in enumerate(rows.cpu()) if 0 <= int(r) < s * c]
    where = torch.tensor([r for _, r in named], dtype=torch.long)
    which = torch.tensor([t for t, _ in named], dtype=torch.long)
    kc, vc = k.cpu().reshape(s * c, hk, dim), v.cpu().reshape(s * c, hk, dim)
    bars.assert_within(kc[where], y[which], tol[which], what + " k")
    assert torch.equal(vc[where], heads[:, hq + hk:][which]), what + " v"
    rest = torch.ones(s * c, dtype=torch.bool)
    rest[where] = False
    assert torch.equal(kc[rest], k0.cpu().reshape(s * c, hk, dim)[rest])
    assert torch.equal(vc[rest], v0.cpu().reshape(s * c, hk, dim)[rest])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim,rope_dim", [(14, 2, 64, 64), (1, 1, 64, 16), (16, 4, 64, 32),
                                                (32, 8, 128, 128), (5, 5, 128, 48), (8, 1, 128, 16),
                                                (3, 1, 64, 48), (12, 4, 128, 112)])
@pytest.mark.parametrize("tokens", [1, 3, 77])
def test_heads_and_rotations(fcv, tokens, hq, hk, dim, rope_dim, dtype):
    say(f"[rope] {tokens} tokens {hq}/{hk} x {dim}, {rope_dim} rotated, {dtype}")
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, tokens, hq, hk, dim, rope_dim, dtype)
    for interleaved in (False, True):
        check(fcv, qkv, pos, cos, sin, k, v, rows, hq, None, None, interleaved, "no norm")
        check(fcv, qkv, pos, cos, sin, k, v, rows, hq, qw, kw, interleaved, "fp32 weights")
        check(fcv, qkv, pos, cos, sin, k, v, rows, hq, qw.to(dtype), kw.to(dtype), interleaved,
              "16-bit weights")


def test_padding_rows_and_positions_past_the_tables(fcv):
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 9, 4, 2, 64, 64, torch.bfloat16)
    rows[2], rows[5], rows[8] = -1, 150, 2 ** 31 - 1   # before, one past, far past
    rows[0], rows[1] = 0, 149                          # the first and the last
    pos[3], pos[4] = -5, 100000
    check(fcv, qkv, pos, cos, sin, k, v, rows, 4, qw, kw, False, "padding")
    zero = torch.zeros_like(qkv)                        # rows of zeros: eps alone under the root
    check(fcv, zero, pos, cos, sin, k, v, rows, 4, qw, kw, True, "zeros")


def test_the_same_row_twice_holds_one_of_its_tokens(fcv):
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 2, 4, 2, 64, 64, torch.bfloat16)
    apart = [t.clone() for t in (k, v)]
    fcv.qk_norm_rope(qkv, pos, cos, sin, *apart, rows, n_heads=4, q_weight=qw, k_weight=kw)
    rows2 = rows[:1].repeat(2)
    fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows2, n_heads=4, q_weight=qw, k_weight=kw)
    for got, both in zip((k, v), apart):
        flat, other = got.view(-1, 2, 64), both.view(-1, 2, 64)
        here = flat[int(rows[0])]
        assert ((here == other[int(rows[0])]) | (here == other[int(rows[1])])).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_strides(fcv, dim):
    """qkv and out inside wider buffers, caches with heads before positions, a prompt's own buffer."""
    hq, hk, dtype = 6, 2, torch.float16
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 20, hq, hk, dim, dim, dtype)
    width = (hq + 2 * hk) * dim
    wide = torch.full((20, width + 16), float("nan"), dtype=dtype, device=DEV)
    wide[:, 8:8 + width] = qkv
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    out = torch.full((20, hq + 1, dim), 7.0, dtype=dtype, device=DEV)
    got = check(fcv, wide[:, 8:8 + width], pos, cos, sin, kt, vt, rows, hq, qw, kw, False, "strided",
                out=out[:, :hq])
    assert got.data_ptr() == out.data_ptr() and (out[:, hq] == 7).all()
    both = torch.zeros(150, 2, hk, dim, dtype=dtype, device=DEV)  # keys and values side by side
    check(fcv, qkv, pos, cos, sin, both[None, :, 0], both[None, :, 1], rows, hq, qw, kw, False,
          "one session")
    empty = fcv.qk_norm_rope(qkv[:0], pos[:0], cos, sin, k, v, rows[:0], n_heads=hq)
    assert empty.shape == (0, hq, dim)


def test_not_finite_values_stay_in_their_head(fcv):
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 4, 4, 2, 64, 64, torch.bfloat16)
    qkv[1, 64 + 3] = float("nan")      # token 1, query head 1
    qkv[2, 4 * 64 + 5] = float("inf")  # token 2, key head 0
    got = fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, n_heads=4, q_weight=qw, k_weight=kw)
    bad = ~got.isfinite().all(-1)
    assert bad.nonzero().tolist() == [[1, 1]]
    at = rows.cpu().long()
    keys = k.reshape(150, 2, 64)[at.to(DEV)]
    assert (~keys.isfinite().all(-1)).nonzero().tolist() == [[2, 0]]


def test_long_cache_offsets_pass_32_bits(fcv):
    """A cache of 2^31 + elements: the last rows' offsets do not fit 32 bits."""
    hk, dim, cap = 8, 128, (1 << 21) + 7
    qkv, pos, cos, sin, _, _, _, qw, kw = make(fcv, 3, 8, hk, dim, dim, torch.bfloat16)
    k = torch.zeros(1, cap, hk, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(1, cap, hk, dim, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([cap - 1, 0, cap - 3], dtype=torch.int32, device=DEV)
    say("[rope] a cache of 4 GiB")
    fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, n_heads=8, q_weight=qw, k_weight=kw)
    small = torch.zeros(1, 3, hk, dim, dtype=torch.bfloat16, device=DEV)
    small_v = small.clone()
    fcv.qk_norm_rope(qkv, pos, cos, sin, small, small_v, torch.arange(3, dtype=torch.int32,
                                                                      device=DEV), n_heads=8,
                     q_weight=qw, k_weight=kw)
    assert torch.equal(k[0, rows.long()], small[0]) and torch.equal(v[0, rows.long()], small_v[0])
    assert not k[0, 1:cap - 3].any() and not k[0, cap - 2].any()


def test_refusals(fcv):
    qkv, pos, cos, sin, k, v, rows, qw, kw = make(fcv, 4, 4, 2, 64, 64, torch.bfloat16)

    def call(**kw_args):
        a = dict(qkv=qkv, positions=pos, cos=cos, sin=sin, k_cache=k, v_cache=v, cache_rows=rows,
                 n_heads=4)
        a.update(kw_args)
        return fcv.qk_norm_rope(**a)

    for args, match in [
            (dict(qkv=qkv.float()), "float16 or bfloat16"), (dict(qkv=qkv.half()), "k_cache must"),
            (dict(n_heads=5), "qkv must be"), (dict(positions=pos.long()), "positions must"),
            (dict(positions=pos[:3]), "positions must"), (dict(cache_rows=rows[::2]), "cache_rows"),
            (dict(cos=cos.half()), "cos must"), (dict(sin=sin[:5]), "equal tables"),
            (dict(cos=cos[:, :4], sin=sin[:, :4]), "cos must"),
            (dict(cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous()), "rope_dim"),
            (dict(k_cache=k[:2]), "differ"), (dict(k_cache=k[0], v_cache=v[0]), "k_cache must"),
            (dict(k_cache=k[:1].expand(3, 50, 2, 64)), "expanded"),
            (dict(q_weight=qw), "together"), (dict(q_weight=qw[:32], k_weight=kw[:32]), "vector"),
            (dict(q_weight=qw, k_weight=kw.bfloat16()), "one type"),
            (dict(out=torch.empty(4, 4, 64, device=DEV)), "out must"),
            (dict(k_cache=k[..., :32], v_cache=v[..., :32]), "head dim")]:
        with pytest.raises(ValueError, match=match):
            call(**args)
