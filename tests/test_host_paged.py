"""What the paged cache's functions refuse, on the host: nothing is launched here."""
import ctypes

import pytest
import torch

from tests import _paged_oracle as orc


def _lib():
    import torch_int.functional.paged as P
    return P, P._lib


def _good():
    """C structures that are right but for their pointers, which nothing reads: there are no rows to work on."""
    P, _ = _lib()
    c = P._Cache(4096, 8192, 8, 16, 2, 64, 2 * 16 * 64, 16 * 64, 64, 2 * 16 * 64, 16 * 64, 64)
    b = P._Batch(4096, 4096, 4096, 4, 2, 2)
    return c, b


@pytest.mark.parametrize("field,value,word", [
    ("page_size", 8, b"page of 8"), ("page_size", 24, b"page of 24"), ("page_size", 1 << 17, b"power of two"),
    ("head_dim", 72, b"head size 72"), ("head_dim", 144, b"head size 144"), ("head_dim", 0, b"head size 0"),
    ("heads", 0, b"0 heads"), ("heads", 5000, b"5000 heads"), ("pages", -1, b"pages"), ("k", 4097, b"k_cache is not aligned"),
    ("k", None, b"k_cache is NULL"), ("v", 8, b"v_cache is not aligned"), ("k_token", 32, b"step over"), ("k_token", 72, b"multiples of 16"),
    ("v_head", 0, b"step over"), ("v_head", 128, b"overlap"), ("k_page", 1024, b"overlap"), ("v_page", -2048, b"step over")])
def test_pools_that_are_refused(field, value, word):
    P, lib = _lib()
    c, b = _good()
    setattr(c, field, value)
    w = P._Attn(4096, 128, 64, 2, 4096, 3, 1, 1e-3, 1.0, None, 0)
    assert lib.ti_paged_attn_s8(c, b, w, None, 0, None) in (1, 2) and word in lib.ti_last_error()
    a = P._Append(4096, 4096, None, 128, 64, 128, 64, 0, 0, None, 0, None, 0, 0, 0, 0, 0, 1.0, 1.0, 1.0)
    assert lib.ti_paged_kv_append_s8(c, b, a, None) in (1, 2) and word in lib.ti_last_error()


@pytest.mark.parametrize("field,value,word", [
    ("rows", -1, b"rows"), ("rows", (1 << 23) + 1, b"rows"), ("seqs", (1 << 20) + 1, b"sequences"), ("pages_per_seq", 1 << 25, b"positions"),
    ("block_table", None, b"block_table is NULL"), ("context_lens", 4098, b"context_lens is not aligned"), ("cu_new", None, b"cu_new is NULL")])
def test_batches_that_are_refused(field, value, word):
    P, lib = _lib()
    c, b = _good()
    setattr(b, field, value)
    w = P._Attn(4096, 128, 64, 2, 4096, 3, 1, 1e-3, 1.0, None, 0)
    assert lib.ti_paged_attn_s8(c, b, w, None, 0, None) in (1, 2) and word in lib.ti_last_error()


@pytest.mark.parametrize("field,value,word", [
    ("q", 4104, b"q is not aligned"), ("q_row", 72, b"multiples of 16 bytes"), ("q_row", -64, b"multiples"), ("q_heads", 3, b"3 query heads"),
    ("q_heads", 0, b"0 query heads"), ("out", None, b"out is NULL"), ("out_type", 0, b"output type 0"), ("out_type", 4, b"output type"),
    ("alpha_qk", 0.0, b"alpha_qk"), ("alpha_qk", -1.0, b"alpha_qk"), ("alpha_qk", float("nan"), b"alpha_qk"),
    ("alpha_qk", float("inf"), b"alpha_qk"), ("alpha_qk", 0.26, b"alpha_qk")])
def test_attention_that_is_refused(field, value, word):
    P, lib = _lib()
    c, b = _good()
    w = P._Attn(4096, 128, 64, 2, 4096, 3, 1, 1e-3, 1.0, None, 0)
    setattr(w, field, value)
    assert lib.ti_paged_attn_s8(c, b, w, None, 0, None) in (1, 2) and word in lib.ti_last_error()
    w = P._Attn(4096, 128, 64, 2, 4096, 3, 1, 1e-3, 1.0, None, 0)
    assert lib.ti_paged_attn_s8(c, b, w, 4100, 64, None) == 2 and lib.ti_paged_attn_s8(c, b, w, None, -1, None) == 1
    assert lib.ti_paged_attn_s8(None, b, w, None, 0, None) == 1 and lib.ti_paged_attn_s8(c, b, None, None, 0, None) == 1


@pytest.mark.parametrize("field,value,word", [
    ("key", None, b"key is NULL"), ("value", 4100, b"value is not aligned"), ("query", 4100, b"query is not aligned"),
    ("q_out", None, b"q_out is NULL"), ("q_heads", 0, b"0 query heads"), ("type", 4, b"type 4"), ("rot", 24, b"24 of 64"),
    ("rot", 80, b"80 of 64"), ("rot", 0, b"0 of 64"), ("k_row", 2, b"multiples of 16 bytes"), ("cos_sin", 4100, b"cos_sin is not aligned")])
def test_appending_that_is_refused(field, value, word):
    P, lib = _lib()
    c, b = _good()
    a = P._Append(4096, 4096, 4096, 128, 64, 128, 64, 128, 64, 4096, 2, 4096, 32, 100, 1, 0, 1, 1.0, 1.0, 1.0)
    setattr(a, field, value)
    assert lib.ti_paged_kv_append_s8(c, b, a, None) in (1, 2) and word in lib.ti_last_error()


def test_no_rows_are_no_work():
    P, lib = _lib()
    c, b = _good()
    b.rows = 0
    assert lib.ti_paged_attn_s8(c, b, P._Attn(None, 0, 0, 2, None, 3, 1, 1e-3, 1.0), None, 0, None) == 0
    assert lib.ti_paged_kv_append_s8(c, b, P._Append(), None) == 0


def test_workspace_is_for_sequences_that_are_cut():
    _, lib = _lib()
    need = lib.ti_paged_attn_workspace_bytes
    assert need(1, 1, 12, 12, 64, 256) == 0                      # too short to be cut
    assert need(0, 0, 12, 12, 64, 4096) == 0 and need(4, 4, 12, 5, 64, 4096) == 0
    assert 0 < need(1, 1, 12, 12, 64, 4096) < need(64, 64, 32, 32, 128, 4096) < 2 ** 28


def test_python_refuses_before_any_launch():
    P, _ = _lib()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    t, n, cu = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="only run on a HIP"):
        P.paged_attn_s8(q, k, k, t, n, cu, 1e-3, 1.0)
    with pytest.raises(RuntimeError, match="only run on a HIP"):
        P.paged_kv_append_s8(q, q, k, k, t, n, cu, 1.0, 1.0)
    f = {"k_cache": _Fake(k), "v_cache": _Fake(k), "block_table": _Fake(t), "context_lens": _Fake(n), "cu_new": _Fake(cu)}
    for name, t, word in (("block_table", t.long(), "2-D torch.int32"), ("v_cache", k[:3], "v_cache is"), ("cu_new", cu[:1], "sequences"),
                          ("block_table", t[:, ::2], "contiguous"), ("k_cache", k.transpose(2, 3), "v_cache is|contiguous"),
                          ("context_lens", n[0], "1-D"), ("k_cache", None, "NoneType")):
        with pytest.raises(RuntimeError, match=word):
            P._cache_and_batch("x", rows=1, **{**f, name: _Fake(t) if t is not None else None})
    with pytest.raises(RuntimeError, match="query must be a 3-D"):
        P.paged_attn_s8(q[0], k, k, t, n, cu, 1e-3, 1.0)
    with pytest.raises(RuntimeError, match="key must be a 3-D"):
        P.paged_kv_append_s8(q.double(), q, k, k, t, n, cu, 1.0, 1.0)


class _Fake(torch.Tensor):
    """A CPU tensor that says it is on a HIP device, for checks that come after that one."""
    @staticmethod
    def __new__(cls, t):
        return t.as_subclass(cls)

    is_cuda = True


def test_the_oracle_agrees_with_dense_attention():
    # one sequence whose pages are in order: softmax over a causal mask, head by head
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randint(-9, 10, (3, 2, 16, 16), generator=g).to(torch.int8) for _ in range(2))
    q = torch.randint(-9, 10, (5, 4, 16), generator=g).to(torch.int8)
    table, lens, cu = torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([40], dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    got, size, _ = orc.attention(q, k, v, table, lens, cu, 0.01, 0.5)
    kk, vv = (x.transpose(1, 2).reshape(48, 2, 16)[:40].double().repeat_interleave(2, 1) for x in (k, v))
    s = torch.einsum("thd,shd->hts", q.double(), kk) * float(torch.tensor(0.01))
    s = s.masked_fill(torch.ones(5, 40).triu(36).bool(), float("-inf"))
    want = 0.5 * torch.einsum("hts,shd->thd", torch.softmax(s, -1), vv)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12) and (size >= got.abs() - 1e-12).all()


def test_modules_keep_their_scales_as_buffers():
    from torch_int.nn import PagedAttn_S8, PagedKVAppend_S8
    append = PagedKVAppend_S8.from_scale(torch.tensor(0.25), 0.5, 0.125, neighbours=True)
    assert {n: float(t) for n, t in append.state_dict().items()} == {"a_k": 4.0, "a_v": 2.0, "a_q": 8.0} and append.neighbours
    attend = PagedAttn_S8.from_scale(0.125, torch.tensor(0.25), 0.5, softmax_scale=0.5)
    assert {n: float(t) for n, t in attend.state_dict().items()} == {"a": 1 / 64, "b": 0.5} and attend.out_dtype is torch.float16
    attend = PagedAttn_S8.from_scale(0.125, 0.25, 0.5, 0.25)
    assert float(attend.b) == 2.0 and attend.out_dtype is torch.int8
    other = PagedAttn_S8()
    other.load_state_dict(attend.state_dict())
    assert other._scalar("a") == 1 / 32 and other._scalar("b") == 2.0
