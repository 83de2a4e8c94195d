"""What the 4-bit paged cache's functions refuse, and its format, on the host: nothing is launched here."""
import pytest
import torch

from tests import _paged_s4_oracle as orc
from tests.test_host_paged import _Fake


def _lib():
    import torch_int.functional.paged_s4 as P
    return P, P._lib


def _good():
    """C structures that are right but for their pointers, which nothing reads: there are no rows to work on."""
    P, _ = _lib()
    c = P._Cache(4096, 8192, 16384, 32768, 8, 16, 2, 64, 2, 2 * 16 * 32, 16 * 32, 32, 128, 64)
    b = P._Batch(4096, 4096, 4096, 4, 2, 2)
    return c, b


def _attn(**kw):
    P, _ = _lib()
    w = P._Attn(4096, 128, 64, 2, 4096, 3, 1, 1, 0.1, 1.0, 0, 0, None, 0)
    for name, value in kw.items():
        setattr(w, name, value)
    return w


def _append():
    P, _ = _lib()
    return P._Append(4096, 4096, 4096, 128, 64, 128, 64, 128, 64, 4096, 2, 4096, 32, 100, 1, 3, 0, 1, 1.0, 1.0, 1.0)


def _refused(c, b, word):
    P, lib = _lib()
    for rc in (lambda: lib.ti_paged_attn_s4(c, b, _attn(), None, 0, None), lambda: lib.ti_paged_kv_append_s4(c, b, _append(), None),
               lambda: lib.ti_paged_kv_read_s4(c, b, P._Read(4096, 8192, 1, 1, 1.0, 1.0), None)):
        assert rc() in (1, 2) and word in lib.ti_last_error(), lib.ti_last_error()


@pytest.mark.parametrize("field,value,word", [
    ("page_size", 8, b"page of 8"), ("page_size", 24, b"page of 24"), ("page_size", 1 << 17, b"power of two"),
    ("head_dim", 72, b"head size 72"), ("head_dim", 144, b"head size 144"), ("head_dim", 16, b"head size 16"), ("groups", 0, b"0 groups"),
    ("groups", 4, b"4 groups"), ("heads", 0, b"0 heads"), ("heads", 5000, b"5000 heads"), ("pages", -1, b"pages"),
    ("k", 4097, b"k_cache is not aligned"), ("k", None, b"k_cache is NULL"), ("v", 8, b"v_cache is not aligned"),
    ("k_scale", None, b"k_scale is NULL"), ("v_scale", 4104, b"v_scale is not aligned"), ("token", 16, b"step over"),
    ("token", 36, b"multiples of 8"), ("head", 0, b"step over"), ("head", 64, b"overlap"), ("page", 512, b"overlap"),
    ("page", -2048, b"step over"), ("scale_head", 32, b"step over"), ("scale_page", 64, b"overlap"),
    ("scale_head", 72, b"multiples of 16"), ("scale_page", 0, b"step over")])
def test_pools_that_are_refused(field, value, word):
    c, b = _good()
    setattr(c, field, value)
    _refused(c, b, word)


@pytest.mark.parametrize("field,value,word", [
    ("rows", -1, b"rows"), ("rows", (1 << 23) + 1, b"rows"), ("seqs", (1 << 20) + 1, b"sequences"), ("pages_per_seq", 1 << 25, b"positions"),
    ("block_table", None, b"block_table is NULL"), ("context_lens", 4098, b"context_lens is not aligned"), ("cu_new", None, b"cu_new is NULL")])
def test_batches_that_are_refused(field, value, word):
    c, b = _good()
    setattr(b, field, value)
    _refused(c, b, word)


@pytest.mark.parametrize("kw,word", [
    (dict(q=4104), b"q is not aligned"), (dict(q_row=72), b"multiples of 16 bytes"), (dict(q_row=-64), b"multiples"),
    (dict(q_row=72, q_type=0), b"query type 0"), (dict(q_row=68, q_type=1), b"multiples of 16 bytes"), (dict(q_type=4), b"query type 4"),
    (dict(q_heads=3), b"3 query heads"), (dict(q_heads=0), b"0 query heads"), (dict(out=None), b"out is NULL"),
    (dict(out_type=0), b"output type 0"), (dict(out_type=4), b"output type"), (dict(alpha_qk=0.0), b"alpha_qk"), (dict(alpha_qk=-1.0), b"alpha_qk"),
    (dict(alpha_qk=float("nan")), b"alpha_qk"), (dict(alpha_qk=float("inf")), b"alpha_qk"), (dict(alpha_qk=1.1e4), b"alpha_qk"),
    (dict(window=-1), b"window of -1"), (dict(window=(1 << 28) + 1), b"window"), (dict(window=5, sinks=-1), b"first ones"),
    (dict(window=5, sinks=(1 << 28) + 1), b"first ones"), (dict(sinks=4), b"0 without a window"), (dict(arrivals=4098), b"arrivals is not aligned")])
def test_attention_that_is_refused(kw, word):
    _, lib = _lib()
    c, b = _good()
    assert lib.ti_paged_attn_s4(c, b, _attn(**kw), None, 0, None) in (1, 2) and word in lib.ti_last_error()
    assert lib.ti_paged_attn_s4(c, b, _attn(), 4100, 64, None) == 2 and lib.ti_paged_attn_s4(c, b, _attn(), None, -1, None) == 1
    assert lib.ti_paged_attn_s4(None, b, _attn(), None, 0, None) == 1 and lib.ti_paged_attn_s4(c, b, None, None, 0, None) == 1


@pytest.mark.parametrize("field,value,word", [
    ("key", None, b"key is NULL"), ("value", 4100, b"value is not aligned"), ("query", 4100, b"query is not aligned"),
    ("q_out", None, b"q_out is NULL"), ("q_heads", 0, b"0 query heads"), ("type", 4, b"type 4"), ("q_type", 0, b"query type 0"), ("rot", 24, b"24 of 64"),
    ("rot", 80, b"80 of 64"), ("rot", 0, b"0 of 64"), ("k_row", 2, b"multiples of 16 bytes"), ("cos_sin", 4100, b"cos_sin is not aligned")])
def test_appending_that_is_refused(field, value, word):
    _, lib = _lib()
    c, b = _good()
    a = _append()
    setattr(a, field, value)
    assert lib.ti_paged_kv_append_s4(c, b, a, None) in (1, 2) and word in lib.ti_last_error()


@pytest.mark.parametrize("field,value,word", [("key", None, b"key is NULL"), ("value", 8200, b"value is not aligned"), ("type", 4, b"type 4"),
                                              ("type", -1, b"type -1")])
def test_reading_that_is_refused(field, value, word):
    P, lib = _lib()
    c, b = _good()
    r = P._Read(4096, 8192, 1, 1, 1.0, 1.0)
    setattr(r, field, value)
    assert lib.ti_paged_kv_read_s4(c, b, r, None) in (1, 2) and word in lib.ti_last_error()
    assert lib.ti_paged_kv_read_s4(c, b, None, None) == 1


def test_no_rows_are_no_work():
    P, lib = _lib()
    c, b = _good()
    b.rows = 0
    assert lib.ti_paged_attn_s4(c, b, P._Attn(None, 0, 0, 2, None, 3, 3, 1, 1e-3, 1.0), None, 0, None) == 0
    assert lib.ti_paged_kv_append_s4(c, b, P._Append(), None) == 0 and lib.ti_paged_kv_read_s4(c, b, P._Read(), None) == 0


def test_workspace_is_for_sequences_that_are_cut_and_does_not_grow_with_the_batch():
    _, lib = _lib()
    need, counters = lib.ti_paged_attn_s4_workspace_bytes, lib.ti_paged_attn_s4_arrivals
    assert need(1, 1, 12, 12, 64, 256) == 0 and counters(1, 1, 12, 12, 64, 256) == 0
    assert need(0, 0, 12, 12, 64, 4096) == 0 and need(4, 4, 12, 5, 64, 4096) == 0
    assert 0 < need(1, 1, 12, 12, 64, 4096) < need(64, 64, 32, 32, 128, 4096) < 2 ** 28
    for rows, seqs, q_heads, heads in ((64, 64, 32, 32), (4096, 4096, 64, 8), (600, 64, 8, 2), (1 << 20, 4000, 8, 1), (100000, 1, 4, 1)):
        assert need(rows, seqs, q_heads, heads, 128, 1 << 16) <= 2 ** 27 and counters(rows, seqs, q_heads, heads, 128, 1 << 16) <= 2048


def test_python_refuses_before_any_launch():
    P, _ = _lib()
    k, v, ks, vs = P.paged_cache_s4(4, 2, 16, 64, 2, "cpu")
    t, n, cu = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.int8)
    for call in (lambda: P.paged_attn_s4(q, k, v, ks, vs, t, n, cu, 1e-3), lambda: P.paged_kv_append_s4(q, q, k, v, ks, vs, t, n, cu),
                 lambda: P.paged_kv_read_s4(k, v, ks, vs, t, n, cu, 1)):
        with pytest.raises(RuntimeError, match="only run on a HIP"):
            call()
    f = {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs, "block_table": t, "context_lens": n, "cu_new": cu}
    for name, bad, word in (("block_table", t.long(), "2-D torch.int32"), ("v_cache", v[:3], "v_cache is"), ("cu_new", cu[:1], "sequences"),
                            ("block_table", t[:, ::2], "contiguous"), ("k_cache", k.transpose(2, 3), "v_cache is|contiguous"),
                            ("context_lens", n[0], "1-D"), ("k_cache", None, "NoneType"), ("k_cache", k.view(torch.int8), "4-D torch.uint8"),
                            ("k_scale", ks.view(torch.float16), "4-D torch.int16"), ("k_scale", ks[:, :, :8], "beside caches"),
                            ("v_scale", vs[..., :1], "beside caches"), ("v_scale", vs.transpose(2, 3).contiguous().transpose(2, 3), "the same"),
                            ("v_cache", v.transpose(1, 2).contiguous().transpose(1, 2), "the same")):
        with pytest.raises(RuntimeError, match=word):
            P._cache_and_batch("x", rows=1, **{m: _Fake(x) if x is not None else None for m, x in {**f, name: bad}.items()})
    apart = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (ks, vs)]
    with pytest.raises(RuntimeError, match="packed"):
        P._cache_and_batch("x", rows=1, **{m: _Fake(x) for m, x in {**f, "k_scale": apart[0], "v_scale": apart[1]}.items()})
    with pytest.raises(RuntimeError, match="query must be a 3-D"):
        P.paged_attn_s4(q[0], k, v, ks, vs, t, n, cu, 1e-3)
    with pytest.raises(RuntimeError, match="query must be a 3-D"):
        P.paged_attn_s4(q.float(), k, v, ks, vs, t, n, cu, 1e-3)
    with pytest.raises(RuntimeError, match="key must be a 3-D"):
        P.paged_kv_append_s4(q.double(), q, k, v, ks, vs, t, n, cu)
    with pytest.raises(RuntimeError, match="rows must be given"):
        P.paged_kv_read_s4(k, v, ks, vs, t, n, cu)
    with pytest.raises(RuntimeError, match="both"):
        P.paged_kv_read_s4(k, v, ks, vs, t, n, cu, key_out=q)
    with pytest.raises(RuntimeError, match="out_dtype must be"):
        P.paged_kv_read_s4(k, v, ks, vs, t, n, cu, 1, torch.float64)
    for bad in ((4, 2, 8, 64, 1), (4, 2, 24, 64, 1), (4, 2, 16, 16, 1), (4, 2, 16, 72, 1), (4, 2, 16, 64, 3)):
        with pytest.raises(RuntimeError, match="paged_cache_s4"):
            P.paged_cache_s4(*bad, "cpu")


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("size", [2.0 ** -16, 1e-3, 1.0, 1e4])
def test_no_value_is_further_than_half_a_step_from_its_own(groups, size):
    # the oracle's format: every value, 0 among them, and no step of half the size would do
    g = torch.Generator().manual_seed(3)
    y = (torch.randn(200, 96, generator=g) * size).double()
    y[::3] = y[::3].abs()
    y[1] = 0.0
    codes, words = orc.quantise(y, groups)
    assert codes.dtype is torch.uint8 and words.dtype is torch.int16 and (words >= 0).all()
    back = orc.values(codes, words)
    step = orc.STEPS[(words >> 4).long()].repeat_interleave(96 // groups, 1)
    assert ((back - y).abs() <= step / 2 * (1 + 1e-12)).all() and (back[1] == 0).all()
    assert torch.equal(back.half().double(), back)          # exact in fp16
    span = (y.unflatten(1, (groups, -1)).amax(-1).clamp(min=0) - y.unflatten(1, (groups, -1)).amin(-1).clamp(max=0))
    s = orc.STEPS[(words >> 4).long()]
    assert (15 * s >= span).all() and (s <= span / 15 * (1 + 1 / 64) + 2.0 ** -20).all()


def test_the_oracle_agrees_with_dense_attention():
    g = torch.Generator().manual_seed(1)
    caches = [orc.quantise(torch.randn(3, 2, 16, 32, generator=g).double(), 1) for _ in range(2)]
    caches = (caches[0][0], caches[1][0], caches[0][1], caches[1][1])
    q = torch.randn(5, 4, 32, generator=g).half()
    table, lens, cu = torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([40], dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    kk, vv = (orc.values(c, w).transpose(1, 2).reshape(48, 2, 32)[:40].repeat_interleave(2, 1) for c, w in ((caches[0], caches[2]), (caches[1], caches[3])))
    i, j = torch.arange(35, 40)[:, None], torch.arange(40)[None, :]
    for window, sinks in ((0, 0), (7, 0), (7, 3), (50, 2)):
        got, about = orc.attention(q, caches, table, lens, cu, 0.2, 0.5, window, sinks)
        s = torch.matmul(q.double().transpose(0, 1), kk.permute(1, 2, 0)) * orc.f32(0.2)
        sees = (j <= i) & ((i - j < window) | (j < sinks) if window else j >= 0)
        want = 0.5 * torch.matmul(torch.softmax(s.masked_fill(~sees, float("-inf")), -1), vv.transpose(0, 1)).transpose(0, 1)
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12) and (about[0] >= got.abs() - 1e-12).all()


def test_modules_keep_their_scales_as_buffers():
    from torch_int.nn import PagedAttn_S4, PagedKVAppend_S4, PagedKVRead_S4
    append = PagedKVAppend_S4.from_scale(torch.tensor(0.25), 0.5, 0.125, neighbours=True)
    assert {n: float(t) for n, t in append.state_dict().items()} == {"a_k": 0.5, "a_v": 0.125, "a_q": 4.0}
    assert append.neighbours and append.query_dtype is torch.int8 and PagedKVAppend_S4.from_scale().query_dtype is torch.float16
    attend = PagedAttn_S4.from_scale(0.125, softmax_scale=0.5, window=9, sinks=2)
    assert {n: float(t) for n, t in attend.state_dict().items()} == {"a": 1 / 16, "b": 1.0} and attend.out_dtype is torch.float16
    attend = PagedAttn_S4.from_scale(0.125, 0.25)
    assert float(attend.b) == 4.0 and attend.out_dtype is torch.int8 and (attend.window, attend.sinks) == (0, 0)
    read = PagedKVRead_S4.from_scale(0.25, torch.tensor(0.5))
    assert float(read.a_k) == 4.0 and float(read.a_v) == 2.0 and read.out_dtype is torch.int8
    other = PagedAttn_S4()
    other.load_state_dict(attend.state_dict())
    assert other._scalar("a") == 1 / 8 and other._scalar("b") == 4.0
