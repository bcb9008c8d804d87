"""The speech language model's operators in 4 bits, on libfcvdit.so (include/fcv_fp4.h): linear layers over
4-bit weights, and a key/value cache of 4-bit pages.

They stand beside those of ``lm.py``: a token's step reads every weight and every cached key once, so a
quarter of the bytes is what a step of few requests takes, and four times the requests fit a card.

    codes, scales = quantize_fp4(w_qkv)                      # once
    pages = new_fp4_pages(4096, n_kv_heads, head_dim, layers=n_layers, device="cuda")
    qkv = fused_linear_fp4(x, codes, scales, b_qkv)          # every step, of every layer i
    q = qk_norm_rope_fp4(qkv, positions, cos, sin, pages[i], cache_rows, n_heads=32)
    o = paged_attention_fp4(q, pages[i], table, lengths)

Numbers are those of the microscaling format (OCP MXFP4): 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives,
times a power of two for each group of 32 elements of a weight row or a key, and for each head's value.
``CachePages`` (pages.py) keeps the book: which pages a session has, forks and compactions.

Calls are asynchronous on the current stream of the tensors' device, compute no gradients, and may be
captured into a graph.  Wrong shapes, types and layouts raise ``ValueError`` before anything is launched;
values inside device tensors are not looked at on the host (include/fcv_fp4.h says what the kernels make
of each).
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from .lm import (_F32, ACTIVATIONS, _check_apart, _dtype, _entry, _indices, _launch, _out_of_range,
                 _rows, _side, _size)

PAGE = 64    # FCV_FP4_PAGE, tokens of a page
GROUP = 32   # FCV_FP4_GROUP, elements of a weight row or a key that share a scale
_HEAD_DIMS = {PAGE * (d + d // 32 + 1): d for d in (64, 128)}  # by the bytes of a page's head

# 4x: the struct's own tail, which the library copies with the rest
_QUANTIZE = struct.Struct("@3Q3q3i4x")
_LINEAR = struct.Struct("@6Q5q8i")
_APPEND = struct.Struct("@9Q4q10if4x")
_READ = struct.Struct("@4Q4q5i4x")
_ATTENTION = struct.Struct("@7Q7q10if4x")


def _pack(layout: struct.Struct, *args) -> bytes:
    try:
        return layout.pack(*args)
    except struct.error as e:
        raise _out_of_range(e) from e


def _bytes_matrix(t: torch.Tensor, name: str, rows: int, columns: int, like: torch.Tensor):
    """Address and row stride of a matrix of bytes."""
    if t.dtype is not torch.uint8 or t.shape != (rows, columns) or t.get_device() != like.get_device() \
            or (columns > 1 and t.stride()[1] != 1):
        raise ValueError(f"{name} must be a uint8 matrix {(rows, columns)} on {like.device} whose rows "
                         f"are contiguous, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr(), t.stride()[0] if rows > 1 else columns


def quantize_fp4(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights ``[N, K]`` (fp16, bf16 or fp32) as ``(codes, scales)``: uint8 ``[N, 16 G]`` and ``[N, G]``
    with ``G = ceil(K / 32)`` groups a row.  Byte ``j`` of a row has codes ``2 j`` (low half) and
    ``2 j + 1``; scale ``b`` stands for ``2 ** (b - 127)``.  The largest magnitude of a group comes out
    between 3.5 and 7 times its scale, values go to the nearest number (ties to the even code, 6 at
    most); a group that holds an infinity or NaN is NaN."""
    if weight.dtype not in (torch.float16, torch.bfloat16, torch.float32) or not weight.is_cuda \
            or weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError("weight must be a float16, bfloat16 or float32 matrix on the GPU, got "
                         f"{weight.dtype} {tuple(weight.shape)} on {weight.device}")
    n, k = weight.shape
    _, ldw = _rows(weight, "weight", k)
    groups = (k + GROUP - 1) // GROUP
    codes = weight.new_empty((n, 16 * groups), dtype=torch.uint8)
    scales = weight.new_empty((n, groups), dtype=torch.uint8)
    if n:
        code = {torch.float16: 0, torch.bfloat16: 1, torch.float32: _F32}[weight.dtype]
        args = _pack(_QUANTIZE, weight.data_ptr(), codes.data_ptr(), scales.data_ptr(), ldw,
                     16 * groups, groups, n, k, code)
        _launch(_entry("fcv_fp4_quantize", 1), weight.device.index, args)
    return codes, scales


def fused_linear_fp4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                     bias: torch.Tensor | None = None, *, activation: str | None = None,
                     residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``act(x @ W.T + bias) + residual`` as ``fused_linear``, over the 4-bit weights ``codes``
    ``[N, 16 G]`` and ``scales`` ``[N, G]`` of ``quantize_fp4``, ``G = ceil(K / 32)``.

    Weights are the numbers that the codes stand for, in ``x``'s type, products and sums those of the
    16-bit layer.  ``x``, ``bias``, ``residual``, ``out``, ``out_dtype`` and ``activation`` are
    ``fused_linear``'s.  Rows of codes start on 16-byte boundaries; those of ``x`` may lie at any stride
    (many rows go faster where they start on 16-byte boundaries and K is a multiple of 8)."""
    code = _dtype(x, "x")
    size = x.shape
    if not size or size[-1] < 1:
        raise ValueError(f"x must be rows of at least one element, got {tuple(size)}")
    k = size[-1]
    groups = (k + GROUP - 1) // GROUP
    if codes.dim() != 2 or codes.shape[0] < 1:
        raise ValueError(f"codes must be a matrix of bytes, got {tuple(codes.shape)}")
    n = codes.shape[0]
    codes_ptr, ld_codes = _bytes_matrix(codes, "codes", n, 16 * groups, x)
    scales_ptr, ld_scales = _bytes_matrix(scales, "scales", n, groups, x)
    m, ldx = _rows(x, "x", k)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    shape = (m, n) if len(size) == 2 else (*size[:-1], n)
    given = out is not None
    if not given:
        if out_dtype is None or out_dtype is x.dtype:
            out_code = code
        elif out_dtype == torch.float32:
            out_code = _F32
        else:
            raise ValueError(f"out must be {x.dtype} or float32, not {out_dtype}")
        out = x.new_empty(shape) if out_code == code else x.new_empty(shape, dtype=out_dtype)
        ldy = n
    else:
        if out.shape != shape:
            raise ValueError(f"out must have shape {shape}, got {tuple(out.shape)}")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"out is {out.dtype}, not {out_dtype}")
        out_code = _side(out, "out", x, code)
        _, ldy = _rows(out, "out", n)
        if m > 1 and ldy < n:
            raise ValueError("out's rows overlap")
    bias_ptr, bias_code = 0, code
    if bias is not None:
        bias_code = _side(bias, "bias", x, code)
        if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            raise ValueError(f"bias must be a contiguous vector of {n}")
        bias_ptr = bias.data_ptr()
    res_ptr, res_code, ldr = 0, code, 0
    if residual is not None:
        res_code = _side(residual, "residual", x, code)
        if residual.shape != shape:
            raise ValueError(f"residual must have shape {shape}, got {tuple(residual.shape)}")
        _, ldr = _rows(residual, "residual", n)
        res_ptr = residual.data_ptr()
    if m == 0:
        return out
    x_ptr, out_ptr = x.data_ptr(), out.data_ptr()
    if given:
        inputs = [("x", x, x_ptr, 2 * ((m - 1) * ldx + k)),
                  ("codes", codes, codes_ptr, (n - 1) * ld_codes + 16 * groups),
                  ("scales", scales, scales_ptr, (n - 1) * ld_scales + groups)]
        if bias is not None:
            inputs.append(("bias", bias, bias_ptr, _size(bias_code) * n))
        if residual is not None and (res_ptr != out_ptr or (m > 1 and ldr != ldy)
                                     or res_code != out_code):
            inputs.append(("residual", residual, res_ptr, _size(res_code) * ((m - 1) * ldr + n)))
        _check_apart(out, out_ptr, _size(out_code) * ((m - 1) * ldy + n), inputs, rows=True)
    args = _pack(_LINEAR, x_ptr, codes_ptr, scales_ptr, bias_ptr, res_ptr, out_ptr, ldx, ld_codes,
                 ld_scales, ldr, ldy, m, n, k, code, bias_code, res_code, out_code, act)
    need = _entry("fcv_fp4_linear_workspace_bytes", 0)(args)
    fn = _entry("fcv_fp4_linear", 3)
    if need:
        ws = x.new_empty(need, dtype=torch.uint8)
        _launch(fn, x.get_device(), args, ws.data_ptr(), need)
    else:
        _launch(fn, x.get_device(), args, None, 0)
    return out


def new_fp4_pages(n_pages: int, n_kv_heads: int, head_dim: int, *, layers: int | None = None,
                  device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty pool of 4-bit pages, uint8 ``[n_pages, n_kv_heads, page bytes]`` (behind ``[layers]``
    where given).  A page holds 64 tokens' keys and values, ``head_dim`` 64 or 128, in 67 or 133 bytes a
    token and head (include/fcv_fp4.h has the layout)."""
    if head_dim not in _HEAD_DIMS.values():
        raise ValueError(f"head dim must be 64 or 128, got {head_dim}")
    if n_pages < 1 or n_kv_heads < 1 or (layers is not None and layers < 1):
        raise ValueError("a pool has at least one page, head and layer")
    shape = (n_pages, n_kv_heads, PAGE * (head_dim + head_dim // 32 + 1))
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8,
                       device=device)


def _pool(pages: torch.Tensor, device: torch.device):
    """Pages, key heads, head dim and strides of a layer's pool."""
    if pages.dtype is not torch.uint8 or pages.device != device or pages.dim() != 3 \
            or pages.shape[2] not in _HEAD_DIMS or pages.numel() == 0 or pages.stride()[2] != 1:
        raise ValueError("pages must be a uint8 tensor [pages, kv heads, page bytes] of new_fp4_pages on "
                         f"{device}, got {pages.dtype} {tuple(pages.shape)} on {pages.device}")
    n_pages, n_kv, size = pages.shape
    page_stride, head_stride, _ = pages.stride()
    return n_pages, n_kv, _HEAD_DIMS[size], page_stride, head_stride


def _reach(pages: torch.Tensor) -> int:
    n_pages, n_kv, size = pages.shape
    return (n_pages - 1) * pages.stride(0) + (n_kv - 1) * pages.stride(1) + size


def qk_norm_rope_fp4(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor,
                     sin: torch.Tensor, pages: torch.Tensor, cache_rows: torch.Tensor, *,
                     n_heads: int, q_weight: torch.Tensor | None = None,
                     k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                     interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``qk_norm_rope`` with a cache of 4-bit pages: RMS norms of queries and keys per head, the position
    rotation and the append, in one pass over ``qkv`` ``[T, (n_heads + 2 kv heads) * head dim]``.

    Token ``t``'s key and value go to place ``cache_rows[t] % 64`` of page ``cache_rows[t] // 64`` of
    ``pages`` (a layer of ``new_fp4_pages``); a negative row or one past the pool goes nowhere.  Keys
    are quantized after norm and rotation, computed in 64 bits, in groups of 32, values in one group a
    head (``quantize_fp4`` has the rule).  Of tokens that name the same row any one's bytes may remain.
    Everything else is ``qk_norm_rope``'s.  Returns the queries ``[T, n_heads, head dim]``, in ``out`` if
    given, which may be their own columns of ``qkv`` and overlaps nothing else."""
    code = _dtype(qkv, "qkv")
    n_pages, n_kv, dim, page_stride, head_stride = _pool(pages, qkv.device)
    width = (n_heads + 2 * n_kv) * dim
    if qkv.dim() != 2 or n_heads < 1 or qkv.shape[1] != width:
        raise ValueError(f"qkv must be [tokens, {width}], got {tuple(qkv.shape)}")
    tokens, qkv_row = _rows(qkv, "qkv", width)
    pos_ptr = _indices(positions, "positions", tokens, qkv)
    row_ptr = _indices(cache_rows, "cache_rows", tokens, qkv)
    index, table = qkv.get_device(), cos.shape
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype is not torch.float32 or t.get_device() != index or t.dim() != 2 \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 table on {qkv.device}")
    if table != sin.shape or table[0] < 1:
        raise ValueError(f"cos {tuple(table)} and sin {tuple(sin.shape)} must be equal tables")
    w_code, qw_ptr, kw_ptr = code, 0, 0
    if q_weight is not None and k_weight is not None:
        w_code = _side(q_weight, "q_weight", qkv, code)
        if _side(k_weight, "k_weight", qkv, code) != w_code:
            raise ValueError("q_weight and k_weight must have one type")
        for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if t.shape != (dim,) or t.stride(0) != 1:
                raise ValueError(f"{name} must be a contiguous vector of {dim}")
        qw_ptr, kw_ptr = q_weight.data_ptr(), k_weight.data_ptr()
    elif q_weight is not k_weight:
        raise ValueError("q_weight and k_weight come together")
    given = out is not None
    if not given:
        out = qkv.new_empty((tokens, n_heads, dim))
    elif out.dtype != qkv.dtype or out.device != qkv.device or out.shape != (tokens, n_heads, dim) \
            or out.stride(2) != 1 or (n_heads > 1 and out.stride(1) != dim):
        raise ValueError(f"out must be a {qkv.dtype} tensor {(tokens, n_heads, dim)} on "
                         f"{qkv.device} whose heads are contiguous")
    if tokens == 0:
        return out
    qkv_ptr, out_ptr, pages_ptr = qkv.data_ptr(), out.data_ptr(), pages.data_ptr()
    q_row = n_heads * dim if not given or tokens == 1 else out.stride(0)
    if given:
        inputs = [("pages", pages, pages_ptr, _reach(pages))]
        if out_ptr != qkv_ptr or (tokens > 1 and q_row != qkv_row):
            inputs.append(("qkv", qkv, qkv_ptr, 2 * ((tokens - 1) * qkv_row + width)))
        _check_apart(out, out_ptr, 2 * ((tokens - 1) * q_row + n_heads * dim), inputs)
    args = _pack(_APPEND, qkv_ptr, pos_ptr, row_ptr, cos.data_ptr(), sin.data_ptr(), qw_ptr, kw_ptr,
                 out_ptr, pages_ptr, qkv_row, q_row, page_stride, head_stride, tokens, n_heads,
                 n_kv, dim, 2 * table[1], table[0], n_pages, code, w_code, bool(interleaved), eps)
    _launch(_entry("fcv_fp4_append", 1), index, args)
    return out


def read_fp4_pages(pages: torch.Tensor, rows: torch.Tensor, *,
                   dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at ``rows`` (int32 ``[T]``, page * 64 + place) of a layer's pages, as
    ``[T, kv heads, head dim]`` of ``dtype`` (fp16 or bf16): what attention over the pages sees, or a
    voice's prompt for ``prefix_attention``.  A row outside the pool gives zeros."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"dtype must be float16 or bfloat16, not {dtype}")
    if not pages.is_cuda:
        raise ValueError(f"pages must be on the GPU, got {pages.device}")
    n_pages, n_kv, dim, page_stride, head_stride = _pool(pages, pages.device)
    tokens = rows.numel()
    row_ptr = _indices(rows, "rows", tokens, pages)
    k = pages.new_empty((tokens, n_kv, dim), dtype=dtype)
    v = torch.empty_like(k)
    if tokens:
        args = _pack(_READ, pages.data_ptr(), row_ptr, k.data_ptr(), v.data_ptr(), page_stride,
                     head_stride, n_kv * dim, n_kv * dim, tokens, n_kv, dim, n_pages,
                     0 if dtype == torch.float16 else 1)
        _launch(_entry("fcv_fp4_read", 1), pages.device.index, args)
    return k, v


def paged_attention_fp4(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor,
                        lengths: torch.Tensor, *, cu_q: torch.Tensor | None = None,
                        max_q: int | None = None, max_length: int | None = None,
                        scale: float | None = None, out: torch.Tensor | None = None,
                        return_lse: bool = False):
    """Causal attention of a batch of sequences over a cache of 4-bit pages: every query of ``q``
    ``[T, heads, head dim]`` sees its own sequence's keys up to itself.

    Key ``j`` of sequence ``b`` is place ``j % 64`` of page ``table[b, j // 64]`` (int32
    ``[B, max pages]``; sequences may share pages, such as those of a voice's prompt, and a page that
    is negative or past the pool has no keys).  Its ``lengths[b]`` keys include those of its new
    tokens.  Its queries are rows ``cu_q[b] .. cu_q[b + 1] - 1``; without ``cu_q`` every sequence has
    ``T / B``.  Rows past ``cu_q[-1]`` are not read, and their rows of ``out`` stay as they are (whatever
    the memory held, without ``out``).  ``max_q`` and ``max_length`` bound the queries and keys of a
    sequence and shape the launch (they default to what one sequence has if the others have a query
    each, and to the table's width); batches that pass them are still computed.  ``scale`` defaults to
    ``head dim ** -0.5``.  A query that sees no key gives zeros.  ``out`` may be ``q`` itself and overlaps
    no other input.  Returns the output, or with ``return_lse`` also the log sums of exponentials, fp32
    ``[T, heads]``."""
    code = _dtype(q, "q")
    n_pages, n_kv, dim, page_stride, head_stride = _pool(pages, q.device)
    size = q.shape
    if len(size) != 3 or size[2] != dim or size[1] % n_kv or size[1] < 1:
        raise ValueError(f"q must be [tokens, heads, {dim}] with heads a multiple of {n_kv}, got "
                         f"{tuple(size)}")
    qs = q.stride()
    if qs[2] != 1:
        raise ValueError("q's last dimension must be contiguous")
    tokens, heads, _ = size
    batch = lengths.numel()
    if batch < 1:
        raise ValueError("lengths is empty")
    len_ptr = _indices(lengths, "lengths", batch, q)
    sizes, ts = table.shape, table.stride()
    if table.dtype is not torch.int32 or table.device != q.device or len(sizes) != 2 \
            or sizes[0] != batch or sizes[1] < 1 or (sizes[1] > 1 and ts[1] != 1):
        raise ValueError(f"table must be an int32 matrix of {batch} rows on {q.device} whose rows are "
                         f"contiguous, got {table.dtype} {tuple(sizes)} on {table.device}")
    max_pages = sizes[1]
    cu_ptr = 0 if cu_q is None else _indices(cu_q, "cu_q", batch + 1, q)
    if cu_q is None:
        if tokens % batch:
            raise ValueError(f"without cu_q the {tokens} rows of q must divide by the {batch} "
                             "sequences")
        max_q = max(tokens // batch, 1)
    elif max_q is None:
        max_q = max(tokens - batch + 1, 1)
    given = out is not None
    if not given:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(size)
    elif out.dtype != q.dtype or out.device != q.device or out.shape != q.shape \
            or out.stride(2) != 1:
        raise ValueError(f"out must be a {q.dtype} tensor {tuple(q.shape)} on {q.device}, its last "
                         "dimension contiguous")
    elif any(out.shape[i] > 1 and out.stride(i) == 0 for i in range(2)):
        raise ValueError("out is expanded: its rows share memory")
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    if tokens == 0:
        return (out, lse) if return_lse else out
    os = out.stride()
    q_ptr, out_ptr, pages_ptr = q.data_ptr(), out.data_ptr(), pages.data_ptr()
    if given:
        rows = (tokens - 1, heads - 1)
        inputs = [("pages", pages, pages_ptr, _reach(pages))]
        if out_ptr != q_ptr or any(n and a != b for n, a, b in zip(rows, qs, os)):
            inputs.append(("q", q, q_ptr, 2 * (rows[0] * qs[0] + rows[1] * qs[1] + dim)))
        _check_apart(out, out_ptr, 2 * (rows[0] * os[0] + rows[1] * os[1] + dim), inputs)
    args = _pack(_ATTENTION, q_ptr, pages_ptr, table.data_ptr(), len_ptr, cu_ptr, out_ptr,
                 0 if lse is None else lse.data_ptr(), qs[0], qs[1], os[0], os[1], page_stride,
                 head_stride, ts[0] if batch > 1 else max_pages, tokens, batch, heads,
                 n_kv, dim, n_pages, max_pages, max_q,
                 PAGE * max_pages if max_length is None else max_length, code,
                 dim ** -0.5 if scale is None else scale)
    need = _entry("fcv_fp4_attention_workspace_bytes", 0)(args)
    fn = _entry("fcv_fp4_attention", 3)
    if need:
        ws = q.new_empty(need, dtype=torch.uint8)
        _launch(fn, q.device.index, args, ws.data_ptr(), need)
    else:
        _launch(fn, q.device.index, args, None, 0)
    return (out, lse) if return_lse else out
