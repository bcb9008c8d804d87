"""Argument checks of the 4-bit operators, on the CPU: the C ABI refuses what the kernels do not take before
anything is launched."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parent.parent / "include" / "fcv_fp4.h"
BIG = 1 << 40  # an address nothing dereferences


def _refuse(fcv, rc, match):
    with pytest.raises(ValueError, match=match):
        fcv._lib.check(rc)


@pytest.mark.parametrize("name", ["FcvFp4Quantize", "FcvFp4Linear", "FcvFp4Append", "FcvFp4Read",
                                  "FcvFp4Attention"])
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
    layout = {"FcvFp4Quantize": "_QUANTIZE", "FcvFp4Linear": "_LINEAR", "FcvFp4Append": "_APPEND",
              "FcvFp4Read": "_READ", "FcvFp4Attention": "_ATTENTION"}[name]
    packed = getattr(__import__("faster_cosyvoice_amd.lm_fp4", fromlist=["x"]), layout)
    assert ctypes.sizeof(getattr(fcv._lib, name)) - packed.size in (0, 4)  # the struct's own tail


def test_page_bytes(fcv):
    f = fcv._lib.load().fcv_fp4_page_bytes
    assert [f(d) for d in (64, 128, 96, 0, -1)] == [4288, 8512, 0, 0, 0]


def _quantize(fcv, **kw):
    base = dict(w=BIG, codes=BIG, scales=BIG, ldw=70, ld_codes=48, ld_scales=3, n=4, k=70, dtype=1)
    base.update(kw)
    return fcv._lib.load().fcv_fp4_quantize(fcv._lib.FcvFp4Quantize(**base), None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=3), "dtype"), (dict(n=-1), "n <= 2"), (dict(k=0), "1 <= k"), (dict(k=1 << 27), "k <= 2"),
    (dict(w=None), "null"), (dict(w=BIG + 1), "boundary"), (dict(codes=BIG + 8), "16-byte"),
    (dict(ld_codes=56), "16-byte"), (dict(ld_codes=32), "overlap"), (dict(ld_scales=2), "overlap"),
    (dict(n=1 << 22, k=1 << 20, ld_codes=1 << 20, ld_scales=1 << 20), "2\\^31 groups")])
def test_quantize_refuses(fcv, bad, match):
    _refuse(fcv, _quantize(fcv, **bad), match)


def _linear(fcv, **kw):
    base = dict(x=BIG, codes=BIG, scales=BIG, y=BIG, ldx=64, ld_codes=32, ld_scales=2, ldy=32, ldr=0, m=4,
                n=32, k=64, dtype=1, bias_dtype=1, residual_dtype=1, y_dtype=1, activation=0)
    base.update(kw)
    return fcv._lib.load().fcv_fp4_linear(fcv._lib.FcvFp4Linear(**base), None, 0, None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(bias_dtype=0), "FCV_LM_F32"), (dict(y_dtype=0), "FCV_LM_F32"),
    (dict(activation=5), "activation"), (dict(m=-1), "m >= 0"), (dict(n=0), "n >= 1"),
    (dict(k=0), "k >= 1"), (dict(ldx=-64), "negative"), (dict(ld_codes=-64), "negative"),
    (dict(ld_scales=-2), "negative"), (dict(ldy=31), "shorter"), (dict(ldr=-8), "negative"),
    (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"),
    (dict(codes=BIG + 8), "16-byte"), (dict(ld_codes=40), "16-byte"), (dict(x=BIG + 1), "boundary"),
    (dict(y=BIG + 2, y_dtype=2), "boundary"), (dict(m=1 << 23), "limited"), (dict(k=1 << 22), "2\\^21"),
    (dict(ld_codes=1 << 24), "2\\^24"), (dict(ld_scales=1 << 24), "2\\^24"),
    (dict(m=1 << 20, n=1 << 20, ldy=1 << 20), "limited")])
def test_linear_refuses(fcv, bad, match):
    _refuse(fcv, _linear(fcv, **bad), match)


def test_linear_of_no_rows_launches_nothing(fcv):
    assert _linear(fcv, m=0, x=None, y=None) == 0


def _append(fcv, **kw):
    base = dict(qkv=BIG, positions=BIG, cache_rows=BIG, rope_cos=BIG, rope_sin=BIG, q_out=BIG, pages=BIG,
                qkv_row=8 * 64, q_row=4 * 64, page_stride=2 * 4288, head_stride=4288, tokens=3, n_heads=4,
                n_kv_heads=2, head_dim=64, rope_dim=64, max_pos=100, n_pages=5, dtype=1, weight_dtype=1,
                interleaved=0, eps=1e-6)
    base.update(kw)
    return fcv._lib.load().fcv_fp4_append(fcv._lib.FcvFp4Append(**base), None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"), (dict(tokens=-1), "tokens"),
    (dict(n_heads=0), "heads"), (dict(rope_dim=8), "rope_dim"), (dict(rope_dim=72), "rope_dim"),
    (dict(rope_dim=80), "rope_dim"), (dict(max_pos=0), "tables"), (dict(n_pages=0), "n_pages"),
    (dict(n_pages=(1 << 24) + 1), "n_pages"), (dict(q_weight=BIG), "together"),
    (dict(weight_dtype=0), "weight_dtype"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(pages=None), "null"), (dict(qkv=BIG + 8), "16-byte"), (dict(pages=BIG + 8), "16-byte"),
    (dict(qkv_row=516), "multiples of 8"), (dict(q_row=8), "overlap"), (dict(page_stride=4288), "over another"),
    (dict(head_stride=4280), "over another"), (dict(page_stride=-8576), "over another"),
    (dict(tokens=1 << 28), "too many")])
def test_append_refuses(fcv, bad, match):
    _refuse(fcv, _append(fcv, **bad), match)


def _read(fcv, **kw):
    base = dict(pages=BIG, rows=BIG, k=BIG, v=BIG, page_stride=2 * 4288, head_stride=4288, k_row=128,
                v_row=128, tokens=3, n_kv_heads=2, head_dim=64, n_pages=5, dtype=1)
    base.update(kw)
    return fcv._lib.load().fcv_fp4_read(fcv._lib.FcvFp4Read(**base), None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=32), "head_dim"), (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 27), "2\\^27"), (dict(n_pages=0), "n_pages"), (dict(rows=None), "null"),
    (dict(k=BIG + 8), "16-byte"), (dict(v_row=132), "16-byte"), (dict(k_row=64), "overlap"),
    (dict(page_stride=4288), "over another")])
def test_read_refuses(fcv, bad, match):
    _refuse(fcv, _read(fcv, **bad), match)


def _attention(fcv, ws=BIG, ws_bytes=1 << 40, **kw):
    base = dict(q=BIG, pages=BIG, table=BIG, lengths=BIG, out=BIG, q_row=256, q_head=64, out_row=256,
                out_head=64, page_stride=2 * 4288, head_stride=4288, table_row=100, tokens=4, batch=4,
                n_heads=4, n_kv_heads=2, head_dim=64, n_pages=500, max_pages=100, max_q=1, max_length=6400,
                dtype=1, scale=0.125)
    base.update(kw)
    args = fcv._lib.FcvFp4Attention(**base)
    return fcv._lib.load().fcv_fp4_attention(args, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"), (dict(batch=0), "batch"),
    (dict(n_heads=3), "multiple"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 25), "2\\^24"),
    (dict(tokens=5), "divide"), (dict(n_pages=0), "n_pages"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 25), "max_pages"), (dict(max_q=0), "max_q"), (dict(max_length=-1), "max_length"),
    (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "null"),
    (dict(table=None), "null"), (dict(out=BIG + 8), "16-byte"), (dict(q_head=68), "multiples of 8"),
    (dict(out_row=-256), "multiples of 8"), (dict(head_stride=4200), "over another"),
    (dict(table_row=-1), "negative"), (dict(ws=None), "null workspace"), (dict(ws_bytes=64), "too small"),
    (dict(ws=BIG + 16), "256-byte")])
def test_attention_refuses(fcv, bad, match):
    _refuse(fcv, _attention(fcv, **bad), match)


def test_workspaces_grow_with_the_call(fcv):
    lib = fcv._lib.load()

    def attention(**kw):
        base = dict(q=BIG, pages=BIG, table=BIG, lengths=BIG, out=BIG, q_row=256, q_head=64, out_row=256,
                    out_head=64, page_stride=2 * 4288, head_stride=4288, table_row=100, tokens=4, batch=4,
                    n_heads=4, n_kv_heads=2, head_dim=64, n_pages=500, max_pages=100, max_q=1,
                    max_length=6400, dtype=1, scale=0.125)
        base.update(kw)
        return lib.fcv_fp4_attention_workspace_bytes(fcv._lib.FcvFp4Attention(**base))

    assert attention() > 0 and attention(max_length=64) == 0 and attention(tokens=0) == 0
    assert attention(head_dim=96) == 0  # refused by the call itself
    assert attention(tokens=4096, batch=4096) == 0


def _copy(fcv, src=(0, 1), dst=(2, 3), pages=BIG, layers=2, layer_stride=6400, n_pages=10, page_stride=640,
          page_bytes=640, count=None):
    a = (ctypes.c_int32 * len(src))(*src) if src is not None else None
    b = (ctypes.c_int32 * len(dst))(*dst) if dst is not None else None
    return fcv._lib.load().fcv_copy_pages(pages, layers, layer_stride, n_pages, page_stride, page_bytes, a, b,
                                          len(src or dst) if count is None else count, None)


@pytest.mark.parametrize("bad,match", [
    (dict(src=(0, 10)), "outside"), (dict(dst=(-1, 3)), "outside"), (dict(dst=(2, 2)), "page 2 is a destination twice"),
    (dict(src=(0, 2)), "page 2 is both"), (dict(src=(5, 5), dst=(5, 6)), "both"), (dict(pages=None), "null pages"),
    (dict(src=None), "null page lists"), (dict(dst=None), "null page lists"), (dict(count=-1), "negative"),
    (dict(layers=-1), "negative"), (dict(layers=1 << 17), "65535"), (dict(page_stride=639), "pages overlap"),
    (dict(layer_stride=639), "layers overlap"), (dict(layer_stride=1280), "layers overlap"),
    (dict(page_bytes=1 << 40), "page_bytes"), (dict(page_stride=1 << 50), "too far"), (dict(n_pages=0), "outside")])
def test_copy_pages_refuses(fcv, bad, match):
    _refuse(fcv, _copy(fcv, **bad), match)


def test_copies_of_nothing_launch_nothing(fcv):
    assert _copy(fcv, src=(), dst=(), count=0, pages=None) == 0
    assert _copy(fcv, layers=0, pages=None) == 0
    assert _copy(fcv, page_bytes=0, pages=None) == 0


def test_cpu_tensors_are_refused(fcv):
    x = torch.zeros(2, 64, dtype=torch.float16)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    pages = fcv.new_fp4_pages(3, 1, 64, device="cpu")
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(4, 32)
    for call in (lambda: fcv.fused_linear_fp4(x, codes, scales), lambda: fcv.quantize_fp4(x),
                 lambda: fcv.qk_norm_rope_fp4(x.repeat(1, 3), ints, table, table, pages, ints, n_heads=1),
                 lambda: fcv.read_fp4_pages(pages, ints, dtype=torch.float16),
                 lambda: fcv.paged_attention_fp4(x.view(2, 1, 64), pages, table.int(), ints)):
        with pytest.raises(ValueError, match="GPU"):
            call()
