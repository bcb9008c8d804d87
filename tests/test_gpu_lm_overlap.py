"""Outputs that share memory with inputs: in place where that is offered, refused elsewhere."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_lm_attention as attn
from tests import test_gpu_lm_linear as linear
from tests import test_gpu_lm_rope as rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_rope_in_its_own_columns(fcv, dim, tokens):
    qkv, pos, cos, sin, k, v, rows, qw, kw = rope.make(fcv, tokens, 6, 2, dim, dim, torch.bfloat16)
    want_k, want_v = k.clone(), v.clone()
    call = dict(n_heads=6, q_weight=qw, k_weight=kw)
    want = fcv.qk_norm_rope(qkv, pos, cos, sin, want_k, want_v, rows, **call)
    own = qkv[:, :6 * dim].unflatten(1, (6, dim))
    got = fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, out=own, **call)
    assert got is own and torch.equal(got, want) and torch.equal(k, want_k) and torch.equal(v, want_v)
    if tokens > 1:
        shifted = qkv[:, dim:7 * dim].unflatten(1, (6, dim))
        with pytest.raises(ValueError, match="overlaps qkv"):
            fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, out=shifted, **call)
    with pytest.raises(ValueError, match="overlaps k_cache"):
        fcv.qk_norm_rope(qkv, pos, cos, sin, k, v, rows, out=k.view(-1, 2, dim)[:3 * tokens].view(
            tokens, 6, dim), **call)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news,prefix", [([1, 1, 1], 20), ([1, 1, 1], 2000), ([40, 3], 50),
                                         ([200, 150], 300)])
def test_attention_over_its_queries(fcv, news, prefix, dim):
    a = attn.make(news, [n + 30 for n in news], prefix, 6, 2, dim, torch.bfloat16)
    want = fcv.prefix_attention(**a, max_q=max(news))
    packed = torch.zeros(sum(news), 10, dim, dtype=torch.bfloat16, device=DEV)
    packed[:, :6] = a["q"]
    b = dict(a, q=packed[:, :6])
    beside = torch.zeros(sum(news), 12, dim, dtype=torch.bfloat16, device=DEV)
    beside[:, :6] = a["q"]
    assert torch.equal(fcv.prefix_attention(**dict(a, q=beside[:, :6]), max_q=max(news),
                                            out=beside[:, 6:]), want)
    with pytest.raises(ValueError, match="overlaps q"):
        fcv.prefix_attention(**b, max_q=max(news), out=packed[:, 1:7])
    with pytest.raises(ValueError, match="overlaps prefix_v"):
        fcv.prefix_attention(**dict(a, prefix_v=beside[:prefix, :2], prefix_k=a["prefix_k"][:len(
            beside[:prefix])]), max_q=max(news), out=beside[:, :6])
    got = fcv.prefix_attention(**b, max_q=max(news), out=packed[:, :6])
    assert torch.equal(got, want) and (packed[:, 6:] == 0).all()


def test_linear_refuses_what_overlaps(fcv):
    x, w, b, r = linear.make(8, 64, 64, torch.bfloat16, bias=torch.bfloat16, residual=torch.bfloat16)
    buf = torch.zeros(9, 64, dtype=torch.bfloat16, device=DEV)
    for call, match in [
            (lambda: fcv.fused_linear(x, w, out=x), "overlaps x"),
            (lambda: fcv.fused_linear(x, w, out=w[:8]), "overlaps weight"),
            (lambda: fcv.fused_linear(x, w, residual=buf[:8], out=buf[1:]), "overlaps residual"),
            (lambda: fcv.fused_linear(x[:1], w, b, out=b[None]), "overlaps bias")]:
        with pytest.raises(ValueError, match=match):
            call()
    h = torch.zeros(8, 128, dtype=torch.bfloat16, device=DEV)
    h[:, :64] = x
    want = fcv.fused_linear(x, w, b)
    assert torch.equal(fcv.fused_linear(h[:, :64], w, b, out=h[:, 64:]), want)


def test_views_that_lie_apart_or_are_the_same(fcv):
    x, w, b, r = linear.make(12, 64, 64, torch.bfloat16, bias=torch.bfloat16, residual=torch.bfloat16)
    want = fcv.fused_linear(x, w, b, residual=r)
    buf = torch.zeros(3, 4, 192, dtype=torch.bfloat16, device=DEV)   # leading dimensions
    buf[..., :64], buf[..., 64:128] = x.view(3, 4, 64), r.view(3, 4, 64)
    got = fcv.fused_linear(buf[..., :64], w, b, residual=buf[..., 64:128], out=buf[..., 128:])
    assert torch.equal(got.reshape(12, 64), want)
    got = fcv.fused_linear(buf[..., :64], w, b, residual=buf[..., 64:128], out=buf[..., 64:128])
    assert torch.equal(got.reshape(12, 64), want)
    wide = torch.zeros(2, 80, dtype=torch.bfloat16, device=DEV)      # one row, told at two strides
    wide[0, :64] = r[0]
    got = fcv.fused_linear(x[:1], w, b, residual=wide[:1, :64], out=wide[0][None, :64])
    assert torch.equal(got[0], fcv.fused_linear(x[:1], w, b, residual=r[:1])[0])
    a = attn.make([1], [20], 30, 6, 2, 64, torch.bfloat16)
    want = fcv.prefix_attention(**a)
    rows = torch.zeros(2, 8, 64, dtype=torch.bfloat16, device=DEV)
    rows[0, :6] = a["q"][0]
    got = fcv.prefix_attention(**dict(a, q=rows[:1, :6]), out=rows[0][None, :6])
    assert torch.equal(got, want)
    heads = torch.zeros(1, 6, 2, 64, dtype=torch.bfloat16, device=DEV)  # outputs between the queries
    heads[:, :, 0] = a["q"]
    assert torch.equal(fcv.prefix_attention(**dict(a, q=heads[:, :, 0]), out=heads[:, :, 1]), want)
