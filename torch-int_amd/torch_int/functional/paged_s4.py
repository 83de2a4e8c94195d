"""A KV cache of 4 bits in pages: appending to it, attending over it, reading it back.

Beside the INT8 cache (:mod:`torch_int.functional.paged`), whose batches (``block_table``, ``context_lens``, ``cu_new``) it shares:
half the bytes, and no steps to be calibrated, since every token's are found as it is written.  Four tensors hold the cache
(:func:`paged_cache_s4` makes them):

* ``k_cache``, ``v_cache``: uint8 [pages, heads, page_size, head_dim / 2].  Byte j of a row holds the code of column j in its low four
  bits, that of column head_dim / 2 + j in the others.  Any strides that keep the last dimension contiguous, are multiples of
  8 bytes and are the same for both; ``head_dim`` is a multiple of 16 from 32 to 128, ``page_size`` a power of two from 16;
* ``k_scale``, ``v_scale``: int16 [pages, heads, page_size, groups], a word for the whole head (``groups`` 1) or for each half of its
  columns (2).  Bits 4 to 14 are those of an fp16 number, the step; bits 0 to 3 are z, and a value is ``step * (code - z)``.
  The last two dimensions are packed, the other strides multiples of 16 bytes, the same for both.

What the batch's tensors hold cannot be checked on the host; values out of range touch no memory outside the tensors
(``include/torch_int_hip.h`` says what they do instead).
"""
import ctypes

import torch

from .. import _CUDA
from .paged import _Batch, _arrivals, _describe, _on, _raw_stream, _rows

__all__ = ["paged_cache_s4", "paged_kv_append_s4", "paged_attn_s4", "paged_kv_read_s4"]

_lib = _CUDA._lib
_vp, _i64, _i32, _f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


class _Cache(ctypes.Structure):
    """``TiPagedCacheS4`` of include/torch_int_hip.h."""
    _fields_ = ([(n, _vp) for n in ("k", "v", "k_scale", "v_scale")]
                + [(n, _i64) for n in ("pages", "page_size", "heads", "head_dim", "groups", "page", "head", "token", "scale_page",
                                       "scale_head")])


class _Append(ctypes.Structure):
    """``TiPagedAppendS4``."""
    _fields_ = ([(n, _vp) for n in ("key", "value", "query")]
                + [(n, _i64) for n in ("k_row", "k_head", "v_row", "v_head", "q_row", "q_head")]
                + [("q_out", _vp), ("q_heads", _i64), ("cos_sin", _vp), ("rot", _i64), ("positions", _i64), ("type", _i32),
                   ("q_type", _i32), ("neighbours", _i32), ("fill", _i32), ("alpha_q", _f32), ("alpha_k", _f32), ("alpha_v", _f32)])


class _Read(ctypes.Structure):
    """``TiPagedReadS4``."""
    _fields_ = [("key", _vp), ("value", _vp), ("type", _i32), ("fill", _i32), ("alpha_k", _f32), ("alpha_v", _f32)]


class _Attn(ctypes.Structure):
    """``TiPagedAttnS4``."""
    _fields_ = [("q", _vp), ("q_row", _i64), ("q_head", _i64), ("q_heads", _i64), ("out", _vp), ("q_type", _i32), ("out_type", _i32),
                ("fill", _i32), ("alpha_qk", _f32), ("alpha_pv", _f32), ("window", _i64), ("sinks", _i64), ("arrivals", _vp),
                ("arrivals_count", _i64)]


_p = ctypes.POINTER
_lib.ti_paged_kv_append_s4.argtypes = [_p(_Cache), _p(_Batch), _p(_Append), _vp]
_lib.ti_paged_kv_read_s4.argtypes = [_p(_Cache), _p(_Batch), _p(_Read), _vp]
_lib.ti_paged_attn_s4.argtypes = [_p(_Cache), _p(_Batch), _p(_Attn), _vp, _i64, _vp]
_lib.ti_paged_attn_s4_workspace_bytes.argtypes = _lib.ti_paged_attn_s4_arrivals.argtypes = [_i64] * 6
for _f in (_lib.ti_paged_kv_append_s4, _lib.ti_paged_kv_read_s4, _lib.ti_paged_attn_s4):
    _f.restype = ctypes.c_int
_lib.ti_paged_attn_s4_workspace_bytes.restype = _lib.ti_paged_attn_s4_arrivals.restype = _i64
_fast_append = getattr(_CUDA._fast, "paged_append_s4", None)
_fast_read = getattr(_CUDA._fast, "paged_read_s4", None)
_fast_attn = getattr(_CUDA._fast, "paged_attn_s4", None)
_U8, _I8, _I16, _I32, _F32 = torch.uint8, torch.int8, torch.int16, torch.int32, torch.float32
_empty_like, _PACKED = torch.empty_like, torch.contiguous_format
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
_QUERIES = {torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
_ws_need = {}  # shape of a call -> (bytes of workspace, counters) it can use


def _fail(op, msg):
    raise RuntimeError(f"torch_int.functional.paged_s4.{op}: {msg}")


def _status(op, rc):
    _fail(op, f"{_lib.ti_last_error().decode()} (status {rc})")


def paged_cache_s4(pages, heads, page_size, head_dim, groups=1, device="cuda"):
    """A cache of zeros: ``(k_cache, v_cache, k_scale, v_scale)``."""
    op = "paged_cache_s4"
    if page_size < 16 or page_size & (page_size - 1):
        _fail(op, f"a page of {page_size} positions (a power of two from 16 is needed)")
    if head_dim < 32 or head_dim > 128 or head_dim % 16:
        _fail(op, f"head size {head_dim} (a multiple of 16 from 32 to 128 is needed)")
    if groups not in (1, 2):
        _fail(op, f"{groups} groups to a head (1 or 2)")
    codes, words = (pages, heads, page_size, head_dim // 2), (pages, heads, page_size, groups)
    return (torch.zeros(codes, dtype=_U8, device=device), torch.zeros(codes, dtype=_U8, device=device),
            torch.zeros(words, dtype=_I16, device=device), torch.zeros(words, dtype=_I16, device=device))


def _cache_and_batch(op, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, rows):
    """The arguments that all calls begin with, checked.  The usual call passes one expression; whatever does not is looked at
    argument by argument, for the message."""
    try:
        dev = k_cache.get_device()
        if (k_cache.is_cuda and k_cache.dtype is _U8 and v_cache.dtype is _U8 and v_cache.get_device() == dev
                and k_scale.dtype is _I16 and k_scale.get_device() == dev and v_scale.dtype is _I16 and v_scale.get_device() == dev
                and block_table.dtype is _I32 and block_table.get_device() == dev and block_table.is_contiguous()
                and context_lens.dtype is _I32 and context_lens.get_device() == dev and context_lens.is_contiguous()
                and cu_new.dtype is _I32 and cu_new.get_device() == dev and cu_new.is_contiguous()):
            shape = pages, heads, page_size, half = k_cache.shape
            words = k_scale.shape
            groups = words[3]
            strides = page, head, token, last = k_cache.stride()
            word_strides = scale_page, scale_head, scale_token, scale_last = k_scale.stride()
            seqs, per_seq = block_table.shape
            if (v_cache.shape == shape and v_cache.stride() == strides and last == 1 and words == (pages, heads, page_size, groups)
                    and v_scale.shape == words and v_scale.stride() == word_strides and scale_token == groups
                    and (groups == 1 or scale_last == 1)
                    and context_lens.shape == (seqs,) and cu_new.shape == (seqs + 1,)):
                return (k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page_size, heads, 2 * half,
                        groups, page, head, token, 2 * scale_page, 2 * scale_head, block_table.data_ptr(), context_lens.data_ptr(),
                        cu_new.data_ptr(), per_seq, seqs, rows)
    except (AttributeError, TypeError, ValueError, IndexError):
        pass
    for name, t, dtype, ndim in (("k_cache", k_cache, _U8, 4), ("v_cache", v_cache, _U8, 4), ("k_scale", k_scale, _I16, 4),
                                 ("v_scale", v_scale, _I16, 4), ("block_table", block_table, _I32, 2),
                                 ("context_lens", context_lens, _I32, 1), ("cu_new", cu_new, _I32, 1)):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.dim() != ndim:
            _fail(op, f"{name} must be a {ndim}-D {dtype} tensor, got {_describe(t)}")
        if not t.is_cuda:
            _fail(op, f"{name} is on {t.device}; the kernels only run on a HIP (cuda) device")
        if t.device != k_cache.device:
            _fail(op, f"{name} is on {t.device}, expected {k_cache.device}")
    if v_cache.shape != k_cache.shape:
        _fail(op, f"k_cache is {tuple(k_cache.shape)} but v_cache is {tuple(v_cache.shape)}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        _fail(op, "the last dimension of k_cache and v_cache must be contiguous")
    for a, b, name in ((k_cache, v_cache, "k_cache and v_cache"), (k_scale, v_scale, "k_scale and v_scale")):
        if a.shape == b.shape and a.stride() != b.stride():
            _fail(op, f"{name} have strides of {a.stride()} and {b.stride()}, which must be the same")
    if k_scale.shape[:3] != k_cache.shape[:3] or v_scale.shape != k_scale.shape:
        _fail(op, f"k_scale is {tuple(k_scale.shape)} and v_scale {tuple(v_scale.shape)} beside caches of {tuple(k_cache.shape)}")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.stride(2) != t.shape[3] or (t.shape[3] > 1 and t.stride(3) != 1):
            _fail(op, f"the last two dimensions of {name} must be packed")
    seqs = context_lens.shape[0]
    if cu_new.shape[0] != seqs + 1 or block_table.shape[0] != seqs:
        _fail(op, f"context_lens has {seqs} sequences, cu_new {cu_new.shape[0]} entries (one more is needed), block_table "
                  f"{block_table.shape[0]} rows")
    _fail(op, "block_table, context_lens and cu_new must be contiguous")


def _out(op, name, t, dtype, shape, dev):
    """An output that is handed in."""
    _rows(op, name, t, dtype, shape, dev)
    if not t.is_contiguous():
        _fail(op, f"{name} must be contiguous")
    return t


def paged_kv_append_s4(key, value, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, alpha_k=1.0, alpha_v=1.0,
                       query=None, alpha_q=1.0, cos_sin=None, neighbours=False, query_dtype=torch.int8, query_out=None):
    """Writes the new tokens' keys and values into their pages in 4 bits, in one launch.

    ``key``, ``value`` [rows, heads, head_dim] (and ``query`` [rows, q_heads, head_dim]) share one dtype of fp32, fp16, bf16 and int8.
    What is written is ``alpha * x``, or ``alpha`` times its rotation by the token's position (as in
    :func:`~torch_int.functional.paged.paged_kv_append_s8`; ``alpha_k`` and ``alpha_v`` are the steps of int8 inputs), rounded to
    fp32, NaN to 0, cut off at +-57344.  Each group of a head's values gets the smallest step with which 16 levels, 0 among them,
    span it; values go to the nearest level, ties to the even code, so none is off by more than half a step.

    Returns the queries [rows, q_heads, head_dim], rotated: as int8, ``sat_s8(round(alpha_q * y))``, or with a ``query_dtype`` of fp16 or
    bf16 as ``alpha_q * y``; None without ``query``.  Rows of no sequence are zeros in them, or left as they are in a ``query_out``
    that is handed in (whose dtype then counts).  Which tokens are not appended, and that their queries become zeros, is as for
    the INT8 cache."""
    op = "paged_kv_append_s4"
    dtype = key.dtype if isinstance(key, torch.Tensor) else None
    code = _TYPES.get(dtype)
    if code is None or key.dim() != 3:
        _fail(op, f"key must be a 3-D tensor of float32, float16, bfloat16 or int8, got {_describe(key)}")
    rows = key.shape[0]
    args = _cache_and_batch(op, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, rows)
    dev = k_cache.get_device()
    heads, d = args[6], args[7]
    shape = (rows, heads, d)
    k_row, k_head = _rows(op, "key", key, dtype, shape, dev)
    v_row, v_head = _rows(op, "value", value, dtype, shape, dev)
    q_ptr = q_row = q_head = q_heads = out_ptr = 0
    q_code = 3
    out = None
    if query is not None:
        if not isinstance(query, torch.Tensor) or query.dim() != 3:
            _fail(op, f"query must be a 3-D {dtype} tensor, got {_describe(query)}")
        q_heads, q_ptr = query.shape[1], query.data_ptr()
        shape = (rows, q_heads, d)
        q_row, q_head = _rows(op, "query", query, dtype, shape, dev)
        if query_out is not None:
            query_dtype = query_out.dtype if isinstance(query_out, torch.Tensor) else None
        q_code = _QUERIES.get(query_dtype)
        if q_code is None:
            _fail(op, f"queries are made as int8, float16 or bfloat16, not as {query_dtype}")
        if query_out is None:
            out = _empty_like(query, dtype=query_dtype, memory_format=_PACKED)
        else:
            out = _out(op, "query_out", query_out, query_dtype, shape, dev)
            if rows > 0 and out.data_ptr() == q_ptr:
                _fail(op, "query_out must not be the query: its rows are rotated by threads that read each other's elements")
        out_ptr = out.data_ptr()
    elif query_out is not None:
        _fail(op, "query_out without query")
    cs_ptr = rot = positions = 0
    if cos_sin is not None:
        if not isinstance(cos_sin, torch.Tensor) or cos_sin.dtype is not _F32 or cos_sin.dim() != 2:
            _fail(op, f"cos_sin must be a 2-D torch.float32 tensor, got {_describe(cos_sin)}")
        if cos_sin.get_device() != dev or not cos_sin.is_contiguous():
            _fail(op, f"cos_sin must be contiguous and on {k_cache.device}")
        positions, rot = cos_sin.shape
        cs_ptr = cos_sin.data_ptr()
        if rot < 16 or rot > d or rot % 16:
            _fail(op, f"cos_sin rotates {rot} of {d} elements (a multiple of 16 up to the head size is needed)")
        if positions == 0:
            _fail(op, "cos_sin has no positions")
    if rows == 0:
        return out
    tail = (key.data_ptr(), value.data_ptr(), q_ptr, k_row, k_head, v_row, v_head, q_row, q_head, out_ptr, q_heads, cs_ptr, rot,
            positions, code, q_code, 1 if neighbours else 0, 1 if query_out is None else 0, float(alpha_q), float(alpha_k),
            float(alpha_v))
    with _on(dev):
        stream = _raw_stream(dev)
        if _fast_append is not None:
            rc = _fast_append(*args, *tail, stream)
        else:
            rc = _lib.ti_paged_kv_append_s4(_Cache(*args[:14]), _Batch(*args[14:]), _Append(*tail), stream or None)
    if rc:
        _status(op, rc)
    return out


def paged_attn_s4(query, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, alpha_qk, alpha_pv=1.0, window=0, sinks=0,
                  out_dtype=torch.float16, out=None):
    """Causal attention of the new tokens over their sequences' pages: ``alpha_pv * softmax(alpha_qk * q . K) . V``.

    ``query`` [rows, q_heads, head_dim] of int8, fp16 or bf16, ``q_heads`` a multiple of the cache's heads (query head h reads key head
    ``h // (q_heads // heads)``).  A token at position p sees the positions j up to its own, which have to be in the cache already
    (:func:`paged_kv_append_s4`); with a ``window`` only those with ``p - j < window`` and, beside them, the first ``sinks`` of its
    sequence.  Positions that no token of the call sees are not looked at: their pages may be gone from the pool and their entries of
    the block table may be anything.  The result [rows, q_heads, head_dim] is fp16, bf16 or int8 (``sat_s8(round(...))``, for a W8A8
    layer behind it).  A token that sees nothing gets zeros; rows of no sequence are zeros too, or left as they are in an ``out``
    that is handed in, which must not share memory with the inputs.  ``alpha_qk`` is from 1e-30 to 1e4.

    Keys, values and queries are computed with as they are, but for bf16 queries, which become fp16 (infinite beyond 65504, with fewer
    bits below 2^-14); sums and softmax are fp32.  A query that holds an infinity or a NaN gives NaN (0 in int8), in its own row and head.
    Weights have 22 bits in sequences of up to 16 rows (new tokens times ``q_heads // heads``) and, as long as ``query`` has no more
    than 48 to a sequence on average (rows of no sequence counted), in all, some fewer beside values of more than 2^10 times their
    step (``include/torch_int_hip.h``); longer sequences of other batches have weights of 11 bits.  The same batch gives the same bits on any stream and in a recorded graph; beside other sequences the last bits of a
    token's context can differ."""
    op = "paged_attn_s4"
    q_code = _QUERIES.get(query.dtype) if isinstance(query, torch.Tensor) else None
    if q_code is None or query.dim() != 3:
        _fail(op, f"query must be a 3-D tensor of int8, float16 or bfloat16, got {_describe(query)}")
    rows, q_heads, _ = query.shape
    args = _cache_and_batch(op, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, rows)
    dev = k_cache.get_device()
    heads, d, seqs = args[6], args[7], args[18]
    shape = (rows, q_heads, d)
    q_row, q_head = _rows(op, "query", query, query.dtype, shape, dev)
    if heads == 0 or q_heads == 0 or q_heads % heads:
        _fail(op, f"{q_heads} query heads are no multiple of {heads} key heads")
    if not 0 <= window <= 1 << 28 or not 0 <= sinks <= 1 << 28 or (sinks and not window):
        _fail(op, f"a window of {window} keys (0 for all, at most 2^28) beside {sinks} first ones (0 without a window)")
    if out is None:
        fill = 1
        code = _QUERIES.get(out_dtype)
        if code is None:
            _fail(op, f"out_dtype must be torch.int8, torch.float16 or torch.bfloat16, got {out_dtype}")
        out = _empty_like(query, dtype=out_dtype, memory_format=_PACKED)
    else:
        fill = 0
        code = _QUERIES.get(out.dtype) if isinstance(out, torch.Tensor) else None
        if code is None:
            _fail(op, f"out must be a tensor of int8, float16 or bfloat16, got {_describe(out)}")
        _out(op, "out", out, out.dtype, shape, dev)
        if rows > 0 and out.data_ptr() == query.data_ptr():
            _fail(op, "out must not be the query: other workgroups read it while its rows are written")
    if rows == 0:
        return out
    key = (rows, seqs, q_heads, heads, d, args[17] * args[5])
    need = _ws_need.get(key)
    if need is None:
        if len(_ws_need) >= 4096:
            _ws_need.clear()
        need = _ws_need[key] = (int(_lib.ti_paged_attn_s4_workspace_bytes(*key)), int(_lib.ti_paged_attn_s4_arrivals(*key)))
    with _on(dev):
        stream = _raw_stream(dev)
        ws, ws_ptr, ws_bytes = _CUDA._workspace(dev, stream, need[0])
        counters, counters_ptr = _arrivals(dev, stream, need[1]) if need[1] > 0 else (None, 0)
        tail = (query.data_ptr(), q_row, q_head, q_heads, out.data_ptr(), q_code, code, fill, float(alpha_qk), float(alpha_pv), int(window),
                int(sinks), counters_ptr, need[1])
        if _fast_attn is not None:
            rc = _fast_attn(*args, *tail, ws_ptr, ws_bytes, stream)
        else:
            rc = _lib.ti_paged_attn_s4(_Cache(*args[:14]), _Batch(*args[14:]), _Attn(*tail), ws_ptr or None, ws_bytes, stream or None)
    if rc:
        _status(op, rc)
    return out


def paged_kv_read_s4(k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu, rows=None, out_dtype=torch.float16, alpha_k=1.0,
                     alpha_v=1.0, key_out=None, value_out=None):
    """The way back: ``(key, value)`` [rows, heads, head_dim] of ``out_dtype`` fp32, fp16, bf16 or int8, ``alpha`` times the cached values
    (``sat_s8(round(alpha * value))`` for int8).

    The rows ``cu[i]`` to ``cu[i + 1] - 1`` are the last positions of sequence i, those that an append with this ``cu`` as ``cu_new``
    has written; as many as ``context_lens[i]`` are all of them.  Rows of positions that have no page, or are before the first, are
    zeros; so are rows of no sequence, or left as they are in outputs that are handed in (both, of one dtype; ``rows`` is then theirs)."""
    op = "paged_kv_read_s4"
    handed = key_out is not None or value_out is not None
    if handed:
        if not isinstance(key_out, torch.Tensor) or key_out.dim() != 3 or not isinstance(value_out, torch.Tensor):
            _fail(op, f"key_out and value_out must be 3-D tensors, both, got {_describe(key_out)} and {_describe(value_out)}")
        if rows is not None and rows != key_out.shape[0]:
            _fail(op, f"{rows} rows, but key_out has {key_out.shape[0]}")
        rows, out_dtype = key_out.shape[0], key_out.dtype
    elif rows is None or rows < 0:
        _fail(op, f"rows must be given without outputs, got {rows}")
    code = _TYPES.get(out_dtype)
    if code is None:
        _fail(op, f"out_dtype must be torch.float32, torch.float16, torch.bfloat16 or torch.int8, got {out_dtype}")
    args = _cache_and_batch(op, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu, rows)
    dev = k_cache.get_device()
    shape = (rows, args[6], args[7])
    if handed:
        _out(op, "key_out", key_out, out_dtype, shape, dev)
        _out(op, "value_out", value_out, out_dtype, shape, dev)
        if rows > 0 and key_out.data_ptr() == value_out.data_ptr():
            _fail(op, "key_out and value_out must be apart")
    else:
        key_out, value_out = torch.empty((2, *shape), dtype=out_dtype, device=k_cache.device).unbind(0)
    if rows == 0:
        return key_out, value_out
    tail = (key_out.data_ptr(), value_out.data_ptr(), code, 0 if handed else 1, float(alpha_k), float(alpha_v))
    with _on(dev):
        stream = _raw_stream(dev)
        if _fast_read is not None:
            rc = _fast_read(*args, *tail, stream)
        else:
            rc = _lib.ti_paged_kv_read_s4(_Cache(*args[:14]), _Batch(*args[14:]), _Read(*tail), stream or None)
    if rc:
        _status(op, rc)
    return key_out, value_out
