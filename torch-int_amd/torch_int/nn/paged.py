"""Modules around the paged INT8 KV cache (:mod:`torch_int.functional.paged`): scales as 0-dim fp32 buffers, as the modules
around the batched products keep theirs."""
import torch

from ..functional import paged
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
