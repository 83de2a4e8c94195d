"""Modules around the paged KV caches (:mod:`torch_int.functional.paged` in INT8, :mod:`torch_int.functional.paged_s4` in 4 bits):
scales as 0-dim fp32 buffers, as the modules around the batched products keep theirs."""
import torch

from ..functional import paged, paged_s4
from ._scalars import ScalarCacheMixin


def _as_tensor(x):
    return x if torch.is_tensor(x) else torch.tensor(float(x))


class PagedKVAppend_S8(ScalarCacheMixin, torch.nn.Module):
    """Quantises new keys and values into their pages and, where there are some, the queries beside them.  ``a_k``, ``a_v`` and
    ``a_q`` are one over the steps (for int8 inputs, the inputs' step over them)."""

    def __init__(self, alpha_k=1.0, alpha_v=1.0, alpha_q=1.0, neighbours=False):
        super().__init__()
        self.neighbours = neighbours
        self.register_buffer("a_k", torch.tensor(float(alpha_k)))
        self.register_buffer("a_v", torch.tensor(float(alpha_v)))
        self.register_buffer("a_q", torch.tensor(float(alpha_q)))

    def forward(self, key, value, k_cache, v_cache, block_table, context_lens, cu_new, query=None, cos_sin=None, query_out=None):
        """Returns the int8 queries, or None without ``query``."""
        return paged.paged_kv_append_s8(key, value, k_cache, v_cache, block_table, context_lens, cu_new, self._scalar("a_k"),
                                        self._scalar("a_v"), query, self._scalar("a_q"), cos_sin, self.neighbours, query_out)

    @staticmethod
    def from_scale(k_scale, v_scale, q_scale=1.0, neighbours=False):
        """From the steps of the cached keys and values and of the int8 queries."""
        mod = PagedKVAppend_S8(neighbours=neighbours)
        mod.a_k, mod.a_v, mod.a_q = (_as_tensor(1.0 / s) for s in (k_scale, v_scale, q_scale))
        return mod


class PagedAttn_S8(ScalarCacheMixin, torch.nn.Module):
    """Causal attention of new tokens over their pages, ``b * softmax(a * q . K) . V`` in ``out_dtype``.  ``a`` is at most 0.25, which
    a module keeps until its scales are set or loaded."""

    def __init__(self, alpha_qk=0.25, alpha_pv=1.0, out_dtype=torch.int8):
        super().__init__()
        self.out_dtype = out_dtype
        self.register_buffer("a", torch.tensor(float(alpha_qk)))
        self.register_buffer("b", torch.tensor(float(alpha_pv)))

    def forward(self, query, k_cache, v_cache, block_table, context_lens, cu_new, out=None):
        """query: int8 [rows, heads, head_dim]; returns the same shape."""
        return paged.paged_attn_s8(query, k_cache, v_cache, block_table, context_lens, cu_new, self._scalar("a"), self._scalar("b"),
                                   self.out_dtype, out)

    @staticmethod
    def from_scale(q_scale, k_scale, v_scale, output_scale=None, softmax_scale=1.0, out_dtype=None):
        """From the steps of queries, keys and values.  With an ``output_scale`` the output is int8 in steps of it, without one
        ``out_dtype`` (fp16 unless given)."""
        mod = PagedAttn_S8(out_dtype=out_dtype or (torch.float16 if output_scale is None else torch.int8))
        mod.a = _as_tensor(q_scale * k_scale * softmax_scale)
        mod.b = _as_tensor(v_scale if output_scale is None else v_scale / output_scale)
        return mod


class PagedKVAppend_S4(ScalarCacheMixin, torch.nn.Module):
    """Writes new keys and values into their pages in 4 bits and, where there are some, rotates the queries beside them.  ``a_k`` and
    ``a_v`` are factors of the inputs (int8 inputs' steps); ``a_q`` is one over the step of int8 queries (for int8 inputs, their step
    over it), or a factor of those in ``query_dtype`` fp16 or bf16 (int8 inputs' step)."""

    def __init__(self, alpha_k=1.0, alpha_v=1.0, alpha_q=1.0, neighbours=False, query_dtype=torch.int8):
        super().__init__()
        self.neighbours, self.query_dtype = neighbours, query_dtype
        self.register_buffer("a_k", torch.tensor(float(alpha_k)))
        self.register_buffer("a_v", torch.tensor(float(alpha_v)))
        self.register_buffer("a_q", torch.tensor(float(alpha_q)))

    def forward(self, key, value, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, query=None, cos_sin=None,
                query_out=None):
        """Returns the queries, or None without ``query``."""
        return paged_s4.paged_kv_append_s4(key, value, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new,
                                           self._scalar("a_k"), self._scalar("a_v"), query, self._scalar("a_q"), cos_sin, self.neighbours,
                                           self.query_dtype, query_out)

    @staticmethod
    def from_scale(q_scale=None, k_input_scale=1.0, v_input_scale=1.0, neighbours=False, query_dtype=torch.float16, q_input_scale=1.0):
        """From the step of int8 queries (without one they are made in ``query_dtype``) and, for int8 keys, values and queries, their
        inputs'."""
        mod = PagedKVAppend_S4(neighbours=neighbours, query_dtype=query_dtype if q_scale is None else torch.int8)
        mod.a_k, mod.a_v = _as_tensor(k_input_scale), _as_tensor(v_input_scale)
        mod.a_q = _as_tensor(q_input_scale if q_scale is None else q_input_scale / q_scale)
        return mod


class PagedAttn_S4(ScalarCacheMixin, torch.nn.Module):
    """Causal attention of new tokens over their pages in 4 bits, ``b * softmax(a * q . K) . V`` in ``out_dtype``; with a ``window`` over
    the last positions up to a token's own and the first ``sinks`` of its sequence."""

    def __init__(self, alpha_qk=1.0, alpha_pv=1.0, window=0, sinks=0, out_dtype=torch.float16):
        super().__init__()
        self.window, self.sinks, self.out_dtype = window, sinks, out_dtype
        self.register_buffer("a", torch.tensor(float(alpha_qk)))
        self.register_buffer("b", torch.tensor(float(alpha_pv)))

    def forward(self, query, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, out=None):
        """query: [rows, heads, head_dim] of int8, fp16 or bf16; returns the same shape."""
        return paged_s4.paged_attn_s4(query, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu_new, self._scalar("a"),
                                      self._scalar("b"), self.window, self.sinks, self.out_dtype, out)

    @staticmethod
    def from_scale(q_scale=1.0, output_scale=None, softmax_scale=1.0, window=0, sinks=0, out_dtype=None):
        """From the step of int8 queries (1 for others).  With an ``output_scale`` the output is int8 in steps of it, without one
        ``out_dtype`` (fp16 unless given)."""
        mod = PagedAttn_S4(window=window, sinks=sinks, out_dtype=out_dtype or (torch.float16 if output_scale is None else torch.int8))
        mod.a = _as_tensor(q_scale * softmax_scale)
        mod.b = _as_tensor(1.0 if output_scale is None else 1.0 / output_scale)
        return mod


class PagedKVRead_S4(ScalarCacheMixin, torch.nn.Module):
    """Cached keys and values as rows of ``out_dtype``, times ``a_k`` and ``a_v`` (one over the steps of int8 rows)."""

    def __init__(self, alpha_k=1.0, alpha_v=1.0, out_dtype=torch.float16):
        super().__init__()
        self.out_dtype = out_dtype
        self.register_buffer("a_k", torch.tensor(float(alpha_k)))
        self.register_buffer("a_v", torch.tensor(float(alpha_v)))

    def forward(self, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu, rows=None, key_out=None, value_out=None):
        """Returns keys and values [rows, heads, head_dim]."""
        return paged_s4.paged_kv_read_s4(k_cache, v_cache, k_scale, v_scale, block_table, context_lens, cu, rows, self.out_dtype,
                                         self._scalar("a_k"), self._scalar("a_v"), key_out, value_out)

    @staticmethod
    def from_scale(k_scale, v_scale):
        """int8 rows in these steps."""
        mod = PagedKVRead_S4(out_dtype=torch.int8)
        mod.a_k, mod.a_v = _as_tensor(1.0 / k_scale), _as_tensor(1.0 / v_scale)
        return mod
