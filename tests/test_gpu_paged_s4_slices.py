"""The 4-bit paged cache's attention: few long items of many rows, cut into more slices than 16, against fp64 on the CPU."""
import pytest
import torch

from tests import _paged_s4_oracle as orc
from tests.test_gpu_paged import _batch
from tests.test_gpu_paged_s4 import DEV, ONE_FP16, _alpha, _attend, _cache, _device, _paged, _query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,d,groups,lens,new,window,sinks", [
    (10, 1, 32, 1, [70000], [5], 0, 0), (5, 1, 32, 2, [36000], [10], 0, 0), (4, 2, 32, 2, [37000, 34000], [26, 25], 0, 0),
    (6, 1, 48, 1, [34000, 33000, 35000], [9, 11, 12], 0, 0), (10, 1, 32, 1, [60000], [7], 40000, 9), (12, 1, 32, 1, [65536, 33000, 50], [11, 1, 1], 0, 0)])
def test_few_long_items_of_many_rows(hq, hk, d, groups, lens, new, window, sinks, monkeypatch):
    P = _paged()
    g = torch.Generator().manual_seed(sum(new))
    cu, lens_t, table, pages, rows = _batch(g, lens, new, 64)
    assert rows * hq > 48 * len(lens) * hk
    caches = _cache(g, pages, hk, 64, d, groups)
    q = _query(g, rows, hq, d, torch.float16)
    a_qk = _alpha(d, torch.float16)
    first = _attend((lens, new, window), q, caches, table, lens_t, cu, a_qk, 30.0, window, sinks, ONE_FP16, out_dtype=torch.float16).to(DEV)
    args = (q.to(DEV), *_device(caches), table.to(DEV), lens_t.to(DEV), cu.to(DEV), a_qk, 30.0, window, sinks)
    assert all(torch.equal(P.paged_attn_s4(*args), first) for _ in range(3))
    monkeypatch.setattr(P._CUDA, "_workspace", lambda *a: (None, 0, 0))     # nothing is cut
    got = P.paged_attn_s4(*args).cpu()
    want, about = orc.attention(q, caches, table, lens_t, cu, a_qk, 30.0, window, sinks)
    assert orc.attention_error(got, want, about, ONE_FP16) <= 1.0
