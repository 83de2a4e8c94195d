"""An INT8 KV cache in pages: appending to it and attending over it.

Upstream keeps one growing key and value tensor per batch (``torch_int/models/opt.py:128-133``), so sequences of different
lengths are padded to one and masked.  Here the cache is a pool of pages and a batch is described by three int32 tensors, read
on the device when the kernels run (a recorded graph replays with whatever they hold then):

* ``cu_new`` [seqs + 1]: where each sequence's new tokens begin among the rows of ``key`` / ``value`` / ``query``, ascending
  from 0; rows behind its last entry belong to no sequence;
* ``context_lens`` [seqs]: positions of each sequence, its new tokens counted (new token i of T is at ``context_len - T + i``);
* ``block_table`` [seqs, n]: the pages of each sequence in order.  Entries behind the last position are not read.

``k_cache`` and ``v_cache`` are int8 [pages, heads, page_size, head_dim], of any strides that keep ``head_dim`` contiguous and
multiples of 16 bytes (a permuted [pages, page_size, heads, head_dim] will do); ``page_size`` is a power of two from 16,
``head_dim`` a multiple of 16 up to 128.  What the three tensors hold cannot be checked on the host; values out of range touch no
memory outside the tensors (``include/torch_int_hip.h`` says what they do instead).
"""
import ctypes

import torch

from .. import _CUDA, _hip_ext

__all__ = ["paged_kv_append_s8", "paged_attn_s8"]

_lib = _CUDA._lib
_vp, _i64, _i32, _f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


class _Cache(ctypes.Structure):
    """``TiPagedCache`` of include/torch_int_hip.h."""
    _fields_ = [("k", _vp), ("v", _vp)] + [(n, _i64) for n in ("pages", "page_size", "heads", "head_dim", "k_page", "k_head",
                                                               "k_token", "v_page", "v_head", "v_token")]


class _Batch(ctypes.Structure):
    """``TiPagedBatch``."""
    _fields_ = [(n, _vp) for n in ("block_table", "context_lens", "cu_new")] + [(n, _i64) for n in ("pages_per_seq", "seqs", "rows")]


class _Append(ctypes.Structure):
    """``TiPagedAppend``."""
    _fields_ = ([(n, _vp) for n in ("key", "value", "query")]
                + [(n, _i64) for n in ("k_row", "k_head", "v_row", "v_head", "q_row", "q_head")]
                + [("q_out", _vp), ("q_heads", _i64), ("cos_sin", _vp), ("rot", _i64), ("positions", _i64), ("type", _i32),
                   ("neighbours", _i32), ("fill", _i32), ("alpha_q", _f32), ("alpha_k", _f32), ("alpha_v", _f32)])


class _Attn(ctypes.Structure):
    """``TiPagedAttn``."""
    _fields_ = [("q", _vp), ("q_row", _i64), ("q_head", _i64), ("q_heads", _i64), ("out", _vp), ("out_type", _i32), ("fill", _i32),
                ("alpha_qk", _f32), ("alpha_pv", _f32), ("arrivals", _vp), ("arrivals_count", _i64)]


_lib.ti_paged_kv_append_s8.argtypes = [ctypes.POINTER(_Cache), ctypes.POINTER(_Batch), ctypes.POINTER(_Append), _vp]
_lib.ti_paged_kv_append_s8.restype = ctypes.c_int
_lib.ti_paged_attn_workspace_bytes.argtypes = [_i64] * 6
_lib.ti_paged_attn_workspace_bytes.restype = _i64
_lib.ti_paged_attn_arrivals.argtypes = [_i64] * 6
_lib.ti_paged_attn_arrivals.restype = _i64
_lib.ti_paged_attn_s8.argtypes = [ctypes.POINTER(_Cache), ctypes.POINTER(_Batch), ctypes.POINTER(_Attn), _vp, _i64, _vp]
_lib.ti_paged_attn_s8.restype = ctypes.c_int
_fast_append = getattr(_CUDA._fast, "paged_append", None)
_fast_attn = getattr(_CUDA._fast, "paged_attn", None)
_raw_stream = torch._C._cuda_getCurrentRawStream
_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32
_empty_like, _PACKED = torch.empty_like, torch.contiguous_format
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
_ws_need = {}  # shape of a call -> (bytes of workspace, counters) it can use
_counters = {}  # (device index, stream) -> int32 zeros in which the slices of a call count themselves, zero again behind it


def _arrivals(dev_index, stream, n):
    """Counters for one stream, grown on demand; a recording gets its own, cleared by the recording itself."""
    key = (dev_index, stream)
    t = _counters.get(key)
    capturing = torch.cuda.is_current_stream_capturing()
    if capturing or t is None or t.numel() < n:
        t = torch.zeros(int(n), dtype=_I32, device=torch.device("cuda", dev_index))
        if not capturing:
            _counters[key] = t
    return t, t.data_ptr()


def _fail(op, msg):
    raise RuntimeError(f"torch_int.functional.paged.{op}: {msg}")


def _describe(t):
    return f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__


def _cache_and_batch(op, k_cache, v_cache, block_table, context_lens, cu_new, rows):
    """The arguments that both calls begin with, checked.  The usual call passes one expression; whatever does not is looked at
    argument by argument, for the message."""
    try:
        dev = k_cache.get_device()
        if (k_cache.is_cuda and k_cache.dtype is _I8 and v_cache.dtype is _I8 and v_cache.get_device() == dev
                and block_table.dtype is _I32 and block_table.get_device() == dev and block_table.is_contiguous()
                and context_lens.dtype is _I32 and context_lens.get_device() == dev and context_lens.is_contiguous()
                and cu_new.dtype is _I32 and cu_new.get_device() == dev and cu_new.is_contiguous()):
            shape = pages, heads, page_size, head_dim = k_cache.shape
            kp, kh, kt, kd = k_cache.stride()
            vp, vh, vt, vd = v_cache.stride()
            seqs, per_seq = block_table.shape
            if v_cache.shape == shape and kd == 1 and vd == 1 and context_lens.shape == (seqs,) and cu_new.shape == (seqs + 1,):
                return (k_cache.data_ptr(), v_cache.data_ptr(), pages, page_size, heads, head_dim, kp, kh, kt, vp, vh, vt,
                        block_table.data_ptr(), context_lens.data_ptr(), cu_new.data_ptr(), per_seq, seqs, rows)
    except (AttributeError, TypeError, ValueError):
        pass
    for name, t, dtype, ndim in (("k_cache", k_cache, _I8, 4), ("v_cache", v_cache, _I8, 4), ("block_table", block_table, _I32, 2),
                                 ("context_lens", context_lens, _I32, 1), ("cu_new", cu_new, _I32, 1)):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.dim() != ndim:
            _fail(op, f"{name} must be a {ndim}-D {dtype} tensor, got {_describe(t)}")
        if not t.is_cuda:
            _fail(op, f"{name} is on {t.device}; the INT8 kernels only run on a HIP (cuda) device")
        if t.device != k_cache.device:
            _fail(op, f"{name} is on {t.device}, expected {k_cache.device}")
    shape = k_cache.shape
    if v_cache.shape != shape:
        _fail(op, f"k_cache is {tuple(shape)} but v_cache is {tuple(v_cache.shape)}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        _fail(op, "the last dimension of k_cache and v_cache must be contiguous")
    seqs = context_lens.shape[0]
    if cu_new.shape[0] != seqs + 1 or block_table.shape[0] != seqs:
        _fail(op, f"context_lens has {seqs} sequences, cu_new {cu_new.shape[0]} entries (one more is needed), block_table "
                  f"{block_table.shape[0]} rows")
    _fail(op, "block_table, context_lens and cu_new must be contiguous")


def _rows(op, name, t, dtype, shape, dev):
    """Row and head stride of a tensor of ``shape`` [rows, heads, head_dim] on device number ``dev``, the last dimension contiguous."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev:
        row, head, last = t.stride()
        if last == 1:
            return row, head
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.dim() != 3:
        _fail(op, f"{name} must be a 3-D {dtype} tensor, got {_describe(t)}")
    if t.get_device() != dev:
        _fail(op, f"{name} is on {t.device}, expected cuda:{dev}")
    if t.shape != shape:
        _fail(op, f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    _fail(op, f"the last dimension of {name} must be contiguous")


def _on(dev):
    """Context that makes device number ``dev`` current; free when it already is."""
    return _hip_ext._NO_SWITCH if dev == _hip_ext._current_device() else torch.cuda.device(dev)


def _status(op, rc):
    _fail(op, f"{_lib.ti_last_error().decode()} (status {rc})")


def paged_kv_append_s8(key, value, k_cache, v_cache, block_table, context_lens, cu_new, alpha_k, alpha_v, query=None, alpha_q=1.0,
                       cos_sin=None, neighbours=False, query_out=None):
    """Writes the new tokens' keys and values into their pages, ``sat_s8(round(alpha * y))`` with ``y`` the input or its
    rotation by the token's position, in one launch.

    ``key``, ``value`` [rows, heads, head_dim] (and ``query`` [rows, q_heads, head_dim]) share one dtype of fp32, fp16, bf16
    and int8; ``alpha_*`` is one over the step of the result (for int8 inputs, their step over it).  ``cos_sin`` fp32 [positions,
    rot], the cosines and then the sines, rotates the first ``rot`` elements of keys and queries, pairs ``(j, j + rot / 2)`` or
    with ``neighbours`` ``(2j, 2j + 1)``; values are not rotated.  A token whose position is
    beyond that table, or beyond its sequence's pages in ``block_table``, is not appended, and its query becomes zeros.  The
    rounding is half to even, of the fp64 result; NaN becomes 0.

    Returns the int8 queries [rows, q_heads, head_dim], or None without ``query``.  Rows of no sequence are zeros in them, or
    left as they are in a ``query_out`` that is handed in."""
    op = "paged_kv_append_s8"
    dtype = key.dtype if isinstance(key, torch.Tensor) else None
    code = _TYPES.get(dtype)
    if code is None or key.dim() != 3:
        _fail(op, f"key must be a 3-D tensor of float32, float16, bfloat16 or int8, got {_describe(key)}")
    rows = key.shape[0]
    args = _cache_and_batch(op, k_cache, v_cache, block_table, context_lens, cu_new, rows)
    dev = k_cache.get_device()
    heads, d = args[4], args[5]
    shape = (rows, heads, d)
    k_row, k_head = _rows(op, "key", key, dtype, shape, dev)
    v_row, v_head = _rows(op, "value", value, dtype, shape, dev)
    q_ptr = q_row = q_head = q_heads = out_ptr = 0
    out = None
    if query is not None:
        if not isinstance(query, torch.Tensor) or query.dim() != 3:
            _fail(op, f"query must be a 3-D {dtype} tensor, got {_describe(query)}")
        q_heads, q_ptr = query.shape[1], query.data_ptr()
        shape = (rows, q_heads, d)
        q_row, q_head = _rows(op, "query", query, dtype, shape, dev)
        if query_out is None:
            out = _empty_like(query, dtype=_I8, memory_format=_PACKED)
        else:
            out = query_out
            _rows(op, "query_out", out, _I8, shape, dev)
            if not out.is_contiguous():
                _fail(op, "query_out must be contiguous")
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
            positions, code, 1 if neighbours else 0, 1 if query_out is None else 0, float(alpha_q), float(alpha_k), float(alpha_v))
    with _on(dev):
        stream = _raw_stream(dev)
        if _fast_append is not None:
            rc = _fast_append(*args, *tail, stream)
        else:
            rc = _lib.ti_paged_kv_append_s8(_Cache(*args[:12]), _Batch(*args[12:]), _Append(*tail), stream or None)
    if rc:
        _status(op, rc)
    return out


def paged_attn_s8(query, k_cache, v_cache, block_table, context_lens, cu_new, alpha_qk, alpha_pv, out_dtype=torch.int8, out=None):
    """Causal attention of the new tokens over their sequences' pages: ``alpha_pv * softmax(alpha_qk * q . K) . V``.

    ``query`` int8 [rows, q_heads, head_dim], ``q_heads`` a multiple of the cache's heads (query head h reads key head
    ``h // (q_heads // heads)``).  Every token sees the positions up to its own, which have to be in the cache already
    (:func:`paged_kv_append_s8`).  The result [rows, q_heads, head_dim] is fp16, bf16 or int8 (``sat_s8(round(...))``, for a W8A8
    layer behind it).  A token that sees nothing gets zeros; rows of no sequence are zeros too, or left as they are in an
    ``out`` that is handed in, which must not share memory with the inputs.  ``alpha_qk`` is positive and at most 0.25.

    Weights have 22 bits in sequences of up to 16 rows (new tokens times ``q_heads // heads``) and, as long as a batch has no more
    than 16 on average, in all; longer sequences of other batches have weights of 11 bits.  The same batch gives the same bits on any
    stream and in a recorded graph; beside other sequences the last bits of a token's context can differ."""
    op = "paged_attn_s8"
    if not isinstance(query, torch.Tensor) or query.dim() != 3:
        _fail(op, f"query must be a 3-D torch.int8 tensor, got {_describe(query)}")
    rows, q_heads, _ = query.shape
    args = _cache_and_batch(op, k_cache, v_cache, block_table, context_lens, cu_new, rows)
    dev = k_cache.get_device()
    heads, d, seqs = args[4], args[5], args[16]
    shape = (rows, q_heads, d)
    q_row, q_head = _rows(op, "query", query, _I8, shape, dev)
    if heads == 0 or q_heads == 0 or q_heads % heads:
        _fail(op, f"{q_heads} query heads are no multiple of {heads} key heads")
    if out is None:
        fill = 1
        code = _TYPES.get(out_dtype)
        if code is None or code == 0:
            _fail(op, f"out_dtype must be torch.int8, torch.float16 or torch.bfloat16, got {out_dtype}")
        out = _empty_like(query, dtype=out_dtype, memory_format=_PACKED)
    else:
        fill = 0
        code = _TYPES.get(out.dtype) if isinstance(out, torch.Tensor) else None
        if code is None or code == 0:
            _fail(op, f"out must be a tensor of int8, float16 or bfloat16, got {_describe(out)}")
        _rows(op, "out", out, out.dtype, shape, dev)
        if not out.is_contiguous():
            _fail(op, "out must be contiguous")
        if rows > 0 and out.data_ptr() == query.data_ptr():
            _fail(op, "out must not be the query: other workgroups read it while its rows are written")
    if rows == 0:
        return out
    key = (rows, seqs, q_heads, heads, d, args[15] * args[3])
    need = _ws_need.get(key)
    if need is None:
        if len(_ws_need) >= 4096:
            _ws_need.clear()
        need = _ws_need[key] = (int(_lib.ti_paged_attn_workspace_bytes(*key)), int(_lib.ti_paged_attn_arrivals(*key)))
    with _on(dev):
        stream = _raw_stream(dev)
        ws, ws_ptr, ws_bytes = _CUDA._workspace(dev, stream, need[0])
        counters, counters_ptr = _arrivals(dev, stream, need[1]) if need[1] > 0 else (None, 0)
        tail = (query.data_ptr(), q_row, q_head, q_heads, out.data_ptr(), code, fill, float(alpha_qk), float(alpha_pv), counters_ptr,
                need[1])
        if _fast_attn is not None:
            rc = _fast_attn(*args, *tail, ws_ptr, ws_bytes, stream)
        else:
            rc = _lib.ti_paged_attn_s8(_Cache(*args[:12]), _Batch(*args[12:]), _Attn(*tail), ws_ptr or None, ws_bytes, stream or None)
    if rc:
        _status(op, rc)
    return out
