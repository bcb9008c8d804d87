"""Operators of the language model that writes the speech tokens, on libfcvdit.so
(include/fcv_lm.h): the linear layer with its epilogue, per-head norms with the rotation and the
cache append, and attention of a batch whose requests share one voice's prompt.

The reference runs that model in an engine of its own (faster_cosyvoice/llm/engine.py:94-141);
these are a decoder layer's products, rotation, cache append and attention.  Norms of whole rows and
a gate's product with its branch are not among them:

    qkv = fused_linear(x, w_qkv, b_qkv)
    q = qk_norm_rope(qkv, positions, cos, sin, k_cache, v_cache, rows, n_heads=32)
    o = prefix_attention(q, k_cache, v_cache, lengths, prefix_k=voice_k, prefix_v=voice_v)
    x = fused_linear(o.flatten(1), w_out, residual=x)

Calls are asynchronous on the current stream of the tensors' device, compute no gradients, and may
be captured into a graph: lengths, positions and rows are device tensors, and workspaces come from
torch's allocator, which keeps a capture's in the capture's own pool.  Wrong shapes, types and
layouts raise ``ValueError`` before anything is launched; values inside device tensors are not
looked at on the host (include/fcv_lm.h says what the kernels make of each).
"""

from __future__ import annotations

import struct
from operator import mul

import torch

from . import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}  # FCV_LM_F16, FCV_LM_BF16
_F32 = 2                                         # FCV_LM_F32
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

# The argument structs, packed here rather than through ctypes fields: these calls take a few
# microseconds on the GPU, and a ctypes struct of 30 fields takes as long to fill.
_LINEAR = struct.Struct("@5Q4q8i")
_QK_NORM_ROPE = struct.Struct("@10Q8q11if")
_ATTENTION = struct.Struct("@10Q14q11if")
_FNS: dict[str, object] = {}


def _out_of_range(e: struct.error) -> ValueError:
    """What a pack raises (floats past fp32 pack as infinities, which the library refuses)."""
    return ValueError(f"a size is out of its argument's range: {e}")


def _entry(name: str, n_tail: int):
    """The library entry ``name`` taking a packed struct, then workspace, bytes and stream (or as
    many of them as it has)."""
    fn = _FNS.get(name)
    if fn is None:
        restype, argtypes = _lib.SIGNATURES[name]
        proto = _lib.ctypes.CFUNCTYPE(restype, _lib.c_void_p, *argtypes[1:])
        fn = _FNS[name] = proto((name, _lib.load()))
        assert len(argtypes) == 1 + n_tail
    return fn


def _launch(fn, index: int, *args) -> None:
    """Call a library entry on device ``index``'s current stream, with that device current."""
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None or not t.is_cuda:
        raise ValueError(f"{name} must be a float16 or bfloat16 tensor on the GPU, got "
                         f"{t.dtype} on {t.device}")
    return code


def _side(t: torch.Tensor, name: str, like: torch.Tensor, code: int) -> int:
    """The type code of a tensor that may be of ``like``'s type or fp32."""
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if t.dtype == like.dtype:
        return code
    if t.dtype == torch.float32:
        return _F32
    raise ValueError(f"{name} must be {like.dtype} or float32, got {t.dtype}")


def _size(code: int) -> int:
    return 4 if code == _F32 else 2


def _indices(t: torch.Tensor, name: str, n: int, like: torch.Tensor) -> int:
    if t.dtype != torch.int32 or t.device != like.device or t.shape != (n,) \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} on {like.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, width: int) -> tuple[int, int]:
    """Row count and stride of a tensor seen as rows of its last dimension."""
    if t.dim() != 2:
        if t.shape[-1] != width:
            raise ValueError(f"{name} must have {width} columns, got {tuple(t.shape)}")
        try:
            t = t.view(-1, width)
        except RuntimeError as e:
            raise ValueError(f"{name}'s leading dimensions {tuple(t.shape[:-1])} do not lie at one "
                             "stride: make it contiguous") from e
    n, columns = t.shape
    if columns != width:
        raise ValueError(f"{name} must have {width} columns, got {tuple(t.shape)}")
    ld, step = t.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return n, ld if n > 1 else max(ld, width)


def _extent(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size()


def _pieces(t: torch.Tensor, at: int, step: int) -> list[tuple[int, int]]:
    """The ranges of bytes that rows ``step`` apart of a tensor at byte ``at`` take in a period."""
    row = t[0] if t.dim() > 1 else t
    width, starts = _extent(row), [at % step]
    if row.dim() == 2 and row.stride(0):  # heads
        width, stride = _extent(row[0]), row.stride(0) * t.element_size()
        starts = [(at + i * stride) % step for i in range(row.shape[0])]
    if width >= step:
        return [(0, step)]
    ranges = [(first, min(first + width, step)) for first in starts]
    ranges += [(0, first + width - step) for first in starts if first + width > step]
    return sorted(ranges)


def _overlap(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the memory of two tensors may overlap.  Rows at one stride in one buffer whose columns
    or heads lie apart do not; other shapes that interleave are taken to."""
    if t.numel() == 0 or out.numel() == 0:
        return False
    first, other = out.data_ptr(), t.data_ptr()
    if other >= first + _extent(out) or other + _extent(t) <= first:
        return False
    steps = {x.stride(0) * x.element_size() for x in (out, t) if x.dim() > 1 and x.shape[0] > 1}
    if len(steps) > 1 or 0 in steps:
        return True
    step = steps.pop() if steps else 1 << 62  # one row each: no period
    ours, theirs = _pieces(out, 0, step), _pieces(t, other - first, step)
    while ours and theirs:
        if ours[-1][0] >= theirs[-1][1]:
            ours.pop()
        elif theirs[-1][0] >= ours[-1][1]:
            theirs.pop()
        else:
            return True
    return False


def _check_apart(out: torch.Tensor, at: int, reach: int, inputs, rows: bool = False) -> None:
    """Refuses an output over an input.  ``at`` and ``reach``: its address and the bytes from there to
    behind its last element, as in each of ``inputs``, ``(name, tensor, at, reach)``: integers first,
    since a small call takes a few microseconds.  ``rows``: tensors are rows of their last dimension."""
    for name, t, first, length in inputs:
        if first < at + reach and at < first + length:
            ours, theirs = (v.view(-1, v.shape[-1]) if rows else v for v in (out, t))
            if _overlap(ours, theirs):
                raise ValueError(f"out overlaps {name}")


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: products on the matrix cores with fp32 sums, one
    rounding at the end.

    ``x`` ``[..., K]`` and ``weight`` ``[N, K]`` are fp16 or bf16 (the same), ``bias`` ``[N]`` and
    ``residual`` ``[..., N]`` are of that type or fp32; the result is of ``out_dtype`` (``x``'s by
    default, or fp32) or goes to ``out``, which may be ``residual`` itself and overlaps no other
    input.  ``activation``: ``"relu"``, ``"silu"``, ``"gelu"`` (erf), ``"gelu_tanh"`` or none.
    Rows may lie at any stride; many rows go faster where they start on 16-byte
    boundaries."""
    code = _dtype(x, "x")
    device = x.device
    if weight.dtype != x.dtype or weight.device != device or weight.dim() != 2:
        raise ValueError(f"weight must be a {x.dtype} matrix on {device}")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    n, k = weight.shape
    if n < 1 or k < 1:
        raise ValueError(f"weight is empty: {(n, k)}")
    m, ldx = _rows(x, "x", k)
    _, ldw = _rows(weight, "weight", k)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    shape = (m, n) if x.dim() == 2 else (*x.shape[:-1], n)
    given = out is not None
    if not given:
        if out_dtype is None or out_dtype == x.dtype:
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
            raise ValueError(f"residual must have shape {shape}, got "
                             f"{tuple(residual.shape)}")
        _, ldr = _rows(residual, "residual", n)
        res_ptr = residual.data_ptr()
    if m == 0:
        return out
    x_ptr, w_ptr, out_ptr = x.data_ptr(), weight.data_ptr(), out.data_ptr()
    if given:
        inputs = [("x", x, x_ptr, 2 * ((m - 1) * ldx + k)),
                  ("weight", weight, w_ptr, 2 * ((n - 1) * ldw + k))]
        if bias is not None:
            inputs.append(("bias", bias, bias_ptr, _size(bias_code) * n))
        if residual is not None and (res_ptr != out_ptr or (m > 1 and ldr != ldy)
                                     or res_code != out_code):
            inputs.append(("residual", residual, res_ptr, _size(res_code) * ((m - 1) * ldr + n)))
        _check_apart(out, out_ptr, _size(out_code) * ((m - 1) * ldy + n), inputs, rows=True)
    try:
        args = _LINEAR.pack(
            x_ptr, w_ptr, bias_ptr, res_ptr, out_ptr, ldx, ldw, ldr, ldy, m, n, k, code, bias_code,
            res_code, out_code, act)
    except struct.error as e:
        raise _out_of_range(e) from e
    need = _entry("fcv_lm_linear_workspace_bytes", 0)(args)
    fn = _entry("fcv_lm_linear", 3)
    if need:
        ws = x.new_empty(need, dtype=torch.uint8)
        _launch(fn, device.index, args, ws.data_ptr(), need)
    else:
        _launch(fn, device.index, args, None, 0)
    return out


def _caches(k: torch.Tensor, v: torch.Tensor, like: torch.Tensor):
    """Shape of a pair of caches, and their strides."""
    for t, name in ((k, "k_cache"), (v, "v_cache")):
        if t.dtype != like.dtype or t.device != like.device or t.dim() != 4 or t.numel() == 0:
            raise ValueError(f"{name} must be a {like.dtype} tensor [sessions, capacity, kv heads, "
                             f"head dim] on {like.device}")
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if shape != v.shape:
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v.shape)} differ")
    if shape[3] not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {shape[3]}")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the caches' last dimension must be contiguous")
    return shape, ks, vs


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 k_cache: torch.Tensor, v_cache: torch.Tensor, cache_rows: torch.Tensor, *,
                 n_heads: int, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """RMS norms of queries and keys per head, the position rotation and the cache append, in one
    pass over the packed projection ``qkv`` ``[T, (n_heads + 2 kv heads) * head dim]``.

    The caches are ``[sessions, capacity, kv heads, head dim]`` (64 or 128) at any strides; token
    ``t``'s key and value go to row ``cache_rows[t]`` of them, counted over sessions and capacity
    (a negative row or one past the end: nowhere).  ``cos``/``sin`` are fp32 tables
    ``[positions, rotated / 2]``; ``interleaved`` rotates pairs ``(2 i, 2 i + 1)``, otherwise
    ``(i, i + rotated / 2)``.  ``q_weight``/``k_weight`` ``[head dim]`` scale the norms; without
    them heads are not normed.  Returns the queries ``[T, n_heads, head dim]``, in ``out`` if given,
    which may be their own columns of ``qkv`` and overlaps nothing else.  The caches overlap neither
    each other nor an input.  A prompt that a batch shares is written with one session's caches
    (``prefix[None]``)."""
    code = _dtype(qkv, "qkv")
    (sessions, capacity, n_kv, dim), ks, vs = _caches(k_cache, v_cache, qkv)
    if qkv.dim() != 2 or qkv.shape[1] != (n_heads + 2 * n_kv) * dim or n_heads < 1:
        raise ValueError(f"qkv must be [tokens, {(n_heads + 2 * n_kv) * dim}], got "
                         f"{tuple(qkv.shape)}")
    tokens, qkv_row = _rows(qkv, "qkv", qkv.shape[1])
    pos_ptr = _indices(positions, "positions", tokens, qkv)
    row_ptr = _indices(cache_rows, "cache_rows", tokens, qkv)
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype != torch.float32 or t.device != qkv.device or t.dim() != 2 \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 table on {qkv.device}")
    table = cos.shape
    if table != sin.shape or table[0] < 1:
        raise ValueError(f"cos {tuple(table)} and sin {tuple(sin.shape)} must be equal tables")
    w_code = code
    if q_weight is not None and k_weight is not None:
        w_code = _side(q_weight, "q_weight", qkv, code)
        if _side(k_weight, "k_weight", qkv, code) != w_code:
            raise ValueError("q_weight and k_weight must have one type")
        for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if t.shape != (dim,) or t.stride(0) != 1:
                raise ValueError(f"{name} must be a contiguous vector of {dim}")
    elif q_weight is not k_weight:
        raise ValueError("q_weight and k_weight come together")
    if 0 in ks and any(n > 1 and st == 0 for n, st in zip(k_cache.shape, ks)) \
            or 0 in vs and any(n > 1 and st == 0 for n, st in zip(v_cache.shape, vs)):
        raise ValueError("k_cache or v_cache is expanded: its rows share memory")
    given = out is not None
    if not given:
        out = qkv.new_empty((tokens, n_heads, dim))
    elif out.dtype != qkv.dtype or out.device != qkv.device or out.shape != (tokens, n_heads, dim) \
            or out.stride(2) != 1 or (n_heads > 1 and out.stride(1) != dim):
        raise ValueError(f"out must be a {qkv.dtype} tensor {(tokens, n_heads, dim)} on "
                         f"{qkv.device} whose heads are contiguous")
    if tokens == 0:
        return out
    qkv_ptr, out_ptr = qkv.data_ptr(), out.data_ptr()
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    if given:
        size = (sessions - 1, capacity - 1, n_kv - 1)
        inputs = [("k_cache", k_cache, k_ptr, 2 * (sum(map(mul, size, ks)) + dim)),
                  ("v_cache", v_cache, v_ptr, 2 * (sum(map(mul, size, vs)) + dim))]
        if out_ptr != qkv_ptr or (tokens > 1 and out.stride(0) != qkv_row):
            inputs.append(("qkv", qkv, qkv_ptr, 2 * ((tokens - 1) * qkv_row + qkv.shape[1])))
        _check_apart(out, out_ptr, 2 * ((tokens - 1) * out.stride(0) + n_heads * dim), inputs)
    try:
        args = _QK_NORM_ROPE.pack(
            qkv_ptr, pos_ptr, row_ptr, cos.data_ptr(), sin.data_ptr(),
            0 if q_weight is None else q_weight.data_ptr(),
            0 if k_weight is None else k_weight.data_ptr(), out_ptr, k_ptr, v_ptr, qkv_row, out.stride(0) if tokens > 1 else n_heads * dim, *ks[:3],
            *vs[:3], tokens, n_heads, n_kv, dim, 2 * table[1], table[0], sessions, capacity, code,
            w_code, bool(interleaved), eps)
    except struct.error as e:
        raise _out_of_range(e) from e
    _launch(_entry("fcv_lm_qk_norm_rope", 1), qkv.device.index, args)
    return out


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     lengths: torch.Tensor, *, prefix_k: torch.Tensor | None = None,
                     prefix_v: torch.Tensor | None = None, cu_q: torch.Tensor | None = None,
                     max_q: int | None = None, slots: torch.Tensor | None = None,
                     max_length: int | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention of a batch of sequences that share one prompt: every query of ``q``
    ``[T, heads, head dim]`` sees all of ``prefix_k``/``prefix_v`` ``[P, kv heads, head dim]`` and
    its own sequence's cached keys up to itself.  The prompt is read for the rows of the whole batch
    together, or by each sequence with its own keys where these are texts and that is faster.

    The caches are ``[sessions, capacity, kv heads, head dim]`` (64 or 128) at any strides;
    sequence ``b`` reads session ``slots[b]`` (``b`` without ``slots``), its ``lengths[b]`` keys
    include those of its new tokens.  Its queries are rows ``cu_q[b] .. cu_q[b + 1] - 1``; without
    ``cu_q`` every sequence has ``T / len(lengths)``.  Rows past ``cu_q[-1]`` are not read, and
    their rows of ``out`` stay as they are (whatever the memory held, without ``out``).  ``max_q`` and
    ``max_length`` bound the queries and keys of a sequence and shape the launch (they default to
    what one sequence has if the others have a query each, and to the capacity); batches that pass
    them are still computed.
    ``scale`` defaults to ``head dim ** -0.5``.  A query that sees no key gives zeros.  ``out`` may be
    ``q`` itself and overlaps no other input.  Returns the output, or with ``return_lse`` also the
    log sums of exponentials, fp32 ``[T, heads]``."""
    code = _dtype(q, "q")
    (sessions, capacity, n_kv, dim), ks, vs = _caches(k_cache, v_cache, q)
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] % n_kv or q.shape[1] < 1:
        raise ValueError(f"q must be [tokens, heads, {dim}] with heads a multiple of {n_kv}, got "
                         f"{tuple(q.shape)}")
    if q.stride(2) != 1:
        raise ValueError("q's last dimension must be contiguous")
    tokens, heads, _ = q.shape
    batch = lengths.numel()
    if batch < 1:
        raise ValueError("lengths is empty")
    len_ptr = _indices(lengths, "lengths", batch, q)
    cu_ptr = 0 if cu_q is None else _indices(cu_q, "cu_q", batch + 1, q)
    if cu_q is None:
        if tokens % batch:
            raise ValueError(f"without cu_q the {tokens} rows of q must divide by the {batch} "
                             "sequences")
        max_q = max(tokens // batch, 1)
    elif max_q is None:
        max_q = max(tokens - batch + 1, 1)
    slot_ptr = 0 if slots is None else _indices(slots, "slots", batch, q)
    if slots is None and batch > sessions:
        raise ValueError(f"{batch} sequences need slots: the caches hold {sessions} sessions")
    prefix_len, pk_ptr, pv_ptr, pk, pv = 0, 0, 0, (0, 0), (0, 0)
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix_k and prefix_v come together")
    if prefix_k is not None:
        for t, name in ((prefix_k, "prefix_k"), (prefix_v, "prefix_v")):
            if t.dtype != q.dtype or t.device != q.device or t.dim() != 3 \
                    or t.shape[1:] != (n_kv, dim) or t.stride(2) != 1:
                raise ValueError(f"{name} must be a {q.dtype} tensor [keys, {n_kv}, {dim}] on "
                                 f"{q.device}, its last dimension contiguous")
        if prefix_k.shape != prefix_v.shape:
            raise ValueError("prefix_k and prefix_v differ in length")
        prefix_len = prefix_k.shape[0]
        if prefix_len:
            pk_ptr, pv_ptr = prefix_k.data_ptr(), prefix_v.data_ptr()
            pk, pv = prefix_k.stride(), prefix_v.stride()
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.device != q.device or out.shape != q.shape \
            or out.stride(2) != 1:
        raise ValueError(f"out must be a {q.dtype} tensor {tuple(q.shape)} on {q.device}, its last "
                         "dimension contiguous")
    elif any(out.shape[i] > 1 and out.stride(i) == 0 for i in range(2)):
        raise ValueError("out is expanded: its rows share memory")
    lse = None
    if return_lse:
        lse = q.new_empty((tokens, heads), dtype=torch.float32)
    if tokens == 0:
        return (out, lse) if return_lse else out
    qs, os = q.stride(), out.stride()
    q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    if given:
        size, rows = (sessions - 1, capacity - 1, n_kv - 1), (tokens - 1, heads - 1)
        inputs = [("k_cache", k_cache, k_ptr, 2 * (sum(map(mul, size, ks)) + dim)),
                  ("v_cache", v_cache, v_ptr, 2 * (sum(map(mul, size, vs)) + dim))]
        if prefix_len:
            keys = (prefix_len - 1, n_kv - 1)
            inputs += [("prefix_k", prefix_k, pk_ptr, 2 * (sum(map(mul, keys, pk)) + dim)),
                       ("prefix_v", prefix_v, pv_ptr, 2 * (sum(map(mul, keys, pv)) + dim))]
        if out_ptr != q_ptr or any(n and a != b for n, a, b in zip(rows, qs, os)):
            inputs.append(("q", q, q_ptr, 2 * (sum(map(mul, rows, qs)) + dim)))
        _check_apart(out, out_ptr, 2 * (sum(map(mul, rows, os)) + dim), inputs)
    try:
        args = _ATTENTION.pack(
            q_ptr, pk_ptr, pv_ptr, k_ptr, v_ptr, cu_ptr, len_ptr, slot_ptr, out_ptr,
            0 if lse is None else lse.data_ptr(), qs[0], qs[1], os[0], os[1], pk[0], pk[1], pv[0],
            pv[1], *ks[:3], *vs[:3], tokens, batch, heads, n_kv, dim, prefix_len, sessions, capacity,
            max_q, capacity if max_length is None else max_length, code,
            dim ** -0.5 if scale is None else scale)
    except struct.error as e:
        raise _out_of_range(e) from e
    need = _entry("fcv_lm_prefix_attention_workspace_bytes", 0)(args)
    fn = _entry("fcv_lm_prefix_attention", 3)
    if need:
        ws = q.new_empty(need, dtype=torch.uint8)
        _launch(fn, q.device.index, args, ws.data_ptr(), need)
    else:
        _launch(fn, q.device.index, args, None, 0)
    return (out, lse) if return_lse else out
