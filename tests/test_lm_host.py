"""Argument checks of the language model operators, on the CPU: the C ABI refuses what the kernels do
not take before anything is launched, and the Python entry points say why."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parent.parent / "include" / "fcv_lm.h"
BIG = 1 << 40  # an address nothing dereferences


def _refuse(fcv, rc, match):
    with pytest.raises(ValueError, match=match):
        fcv._lib.check(rc)


@pytest.mark.parametrize("name", ["FcvLmLinear", "FcvLmQkNormRope", "FcvLmAttention"])
def test_struct_fields_match_the_header(fcv, name):
    text = HEADER.read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    kinds = {"int64_t": 8, "int32_t": 4, "float": 4}
    want = []
    for line in (ln.strip() for ln in body.split(";")):
        if line:
            kind, field = re.match(r"(?:const )?(\w+ ?\*?) ?(\w+)$", line).groups()
            want.append((field, 8 if "*" in kind else kinds[kind.strip()]))
    got = [(f, ctypes.sizeof(t)) for f, t in getattr(fcv._lib, name)._fields_]
    assert got == want


def _linear(fcv, **kw):
    base = dict(x=BIG, w=BIG, y=BIG, ldx=64, ldw=64, ldy=32, ldr=0, m=4, n=32, k=64, dtype=1,
                bias_dtype=1, residual_dtype=1, y_dtype=1, activation=0)
    base.update(kw)
    return fcv._lib.load().fcv_lm_linear(fcv._lib.FcvLmLinear(**base), None, 0, None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(bias_dtype=0), "FCV_LM_F32"), (dict(y_dtype=0), "FCV_LM_F32"),
    (dict(activation=5), "activation"), (dict(m=-1), "m >= 0"), (dict(n=0), "n >= 1"),
    (dict(k=0), "k >= 1"), (dict(ldx=-64), "negative"), (dict(ldw=-64), "negative"),
    (dict(ldy=31), "shorter"), (dict(ldr=-8), "negative"), (dict(x=None), "null"),
    (dict(w=BIG + 1), "boundary"), (dict(y=BIG + 2, y_dtype=2), "boundary"),
    (dict(m=1 << 23), "limited"), (dict(k=1 << 29), "2\\^28"), (dict(m=1 << 20, n=1 << 20, ldy=1 << 20), "limited"),
])
def test_linear_refuses(fcv, bad, match):
    _refuse(fcv, _linear(fcv, **bad), match)


def test_linear_of_no_rows_launches_nothing(fcv):
    assert _linear(fcv, m=0, x=None, y=None) == 0


def _rope(fcv, **kw):
    base = dict(qkv=BIG, positions=BIG, cache_rows=BIG, rope_cos=BIG, rope_sin=BIG, q_out=BIG,
                k_cache=BIG, v_cache=BIG, qkv_row=8 * 64, q_row=4 * 64, k_session=10 * 128,
                k_row=128, k_head=64, v_session=10 * 128, v_row=128, v_head=64, tokens=3,
                n_heads=4, n_kv_heads=2, head_dim=64, rope_dim=64, max_pos=100, sessions=5,
                capacity=10, dtype=1, weight_dtype=1, interleaved=0, eps=1e-6)
    base.update(kw)
    return fcv._lib.load().fcv_lm_qk_norm_rope(fcv._lib.FcvLmQkNormRope(**base), None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"), (dict(tokens=-1), "tokens"),
    (dict(n_heads=0), "heads"), (dict(rope_dim=8), "rope_dim"), (dict(rope_dim=72), "rope_dim"),
    (dict(rope_dim=80), "rope_dim"), (dict(max_pos=0), "tables"), (dict(sessions=0), "sessions"),
    (dict(sessions=1 << 20, capacity=1 << 20), "2\\^31"), (dict(q_weight=BIG), "together"),
    (dict(weight_dtype=0), "weight_dtype"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(k_cache=None), "null"), (dict(qkv=BIG + 8), "16-byte"),
    (dict(v_cache=BIG + 2), "16-byte"), (dict(k_row=130), "multiples of 8"),
    (dict(q_row=8), "overlap"), (dict(v_head=-64), "negative"), (dict(tokens=1 << 28), "too many"),
])
def test_norm_rope_refuses(fcv, bad, match):
    _refuse(fcv, _rope(fcv, **bad), match)


def _attention(fcv, ws=BIG, ws_bytes=1 << 40, **kw):
    base = dict(q=BIG, prefix_k=BIG, prefix_v=BIG, k_cache=BIG, v_cache=BIG, lengths=BIG, out=BIG,
                q_row=256, q_head=64, out_row=256, out_head=64, pk_row=128, pk_head=64, pv_row=128,
                pv_head=64, k_session=1280, k_row=128, k_head=64, v_session=1280, v_row=128,
                v_head=64, tokens=4, batch=4, n_heads=4, n_kv_heads=2, head_dim=64, prefix_len=7,
                sessions=5, capacity=10, max_q=1, max_length=10, dtype=1, scale=0.125)
    base.update(kw)
    args = fcv._lib.FcvLmAttention(**base)
    return fcv._lib.load().fcv_lm_prefix_attention(args, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=80), "head_dim"), (dict(n_heads=5), "multiple"),
    (dict(n_kv_heads=0), "multiple"), (dict(batch=0), "batch"), (dict(tokens=-4), "batch"),
    (dict(tokens=5), "whole number"), (dict(prefix_len=-1), "prefix_len"),
    (dict(prefix_len=(1 << 29) + 1), "prefix_len"), (dict(capacity=1 << 30), "capacity"),
    (dict(sessions=0), "session"), (dict(sessions=3), "slots"), (dict(max_q=0), "max_q"),
    (dict(max_length=-1), "max_length"), (dict(scale=0.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q_head=60), "multiples of 8"), (dict(pv_row=-8), "multiples of 8"),
    (dict(k_row=1 << 24), "2\\^24"), (dict(out_head=0), "overlap"), (dict(out_row=0), "overlap"), (dict(lengths=None), "null"), (dict(prefix_v=None), "prefix"),
    (dict(out=BIG + 8), "16-byte"), (dict(prefix_k=BIG + 4), "16-byte"),
    (dict(tokens=1 << 26), "2\\^26"), (dict(ws=None, prefix_len=4000), "null workspace"),
    (dict(ws_bytes=16, prefix_len=4000), "too small"),
    (dict(ws=BIG + 16, prefix_len=4000), "256-byte"),
])
def test_attention_refuses(fcv, bad, match):
    _refuse(fcv, _attention(fcv, **bad), match)


def test_workspace_sizes(fcv):
    """None where one launch does it all; it grows with the rows and holds a part a range."""
    lib = fcv._lib.load()

    def need(**kw):
        base = dict(q=BIG, prefix_k=BIG, prefix_v=BIG, k_cache=BIG, v_cache=BIG, lengths=BIG,
                    out=BIG, q_row=256, q_head=64, out_row=256, out_head=64, pk_row=128, pk_head=64,
                    pv_row=128, pv_head=64, k_session=1 << 20, k_row=128, k_head=64,
                    v_session=1 << 20, v_row=128, v_head=64, tokens=4, batch=4, n_heads=4,
                    n_kv_heads=2, head_dim=64, prefix_len=7, sessions=64, capacity=5000, max_q=1,
                    max_length=10, dtype=1, scale=0.125)
        base.update(kw)
        return lib.fcv_lm_prefix_attention_workspace_bytes(fcv._lib.FcvLmAttention(**base))

    assert need() == 0 and need(tokens=0, q=None, out=None) == 0
    few = need(prefix_len=5000)
    assert few >= 2 * 4 * 4 * 64 * 4
    assert need(prefix_len=5000, tokens=8, batch=8) > few
    assert need(head_dim=65) == 0  # what the call refuses needs none


def test_cpu_tensors_are_refused(fcv):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on the GPU"):
        fcv.fused_linear(x, torch.zeros(8, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="on the GPU"):
        fcv.qk_norm_rope(x, x, x, x, x, x, x, n_heads=1)
    with pytest.raises(ValueError, match="on the GPU"):
        fcv.prefix_attention(x, x, x, x)
