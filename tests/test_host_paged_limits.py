"""The paged cache's defaults and bounds, on the host: nothing is launched here."""
from tests.test_host_paged import _good, _lib


def test_the_default_scales_are_taken():
    from torch_int.nn import PagedAttn_S8, PagedKVAppend_S8
    P, lib = _lib()
    c, b = _good()
    b.rows = 0
    attend, append = PagedAttn_S8(), PagedKVAppend_S8()
    w = P._Attn(None, 0, 0, 2, None, 3, 1, attend._scalar("a"), attend._scalar("b"))
    assert lib.ti_paged_attn_s8(c, b, w, None, 0, None) == 0, lib.ti_last_error()
    assert [append._scalar(n) for n in ("a_k", "a_v", "a_q")] == [1.0, 1.0, 1.0]
