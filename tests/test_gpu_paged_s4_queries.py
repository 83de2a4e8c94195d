"""The 4-bit paged cache's attention: queries that hold an infinity, also where all of their scores are minus infinity."""
import pytest
import torch

from tests import _paged_s4_oracle as orc
from tests.test_gpu_paged import _batch
from tests.test_gpu_paged_s4 import DEV, _cache, _device, _paged, _query

pytestmark = pytest.mark.gpu


# query heads, key heads, head size, groups, context lengths, new tokens, window, first keys
ROWS = [
    (2, 2, 64, 1, [1], [1], 0, 0),
    (8, 2, 128, 2, [300, 40], [2, 1], 0, 0),
    (4, 1, 80, 1, [5000], [1], 0, 0),                # slices that meet in the launch
    (32, 2, 128, 2, [9000], [1], 0, 0),              # ... and behind it
    (2, 1, 64, 2, [400], [130], 0, 0),               # tiles
    (4, 2, 96, 1, [3000, 20], [70, 1], 0, 0),        # tiles in slices
    (4, 2, 128, 2, [700, 200], [100, 2], 60, 3),
]


@pytest.mark.parametrize("query", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("i", range(len(ROWS)))
def test_a_row_whose_scores_are_all_minus_infinity_is_no_number(i, query):
    hq, hk, d, groups, lens, new, window, sinks = ROWS[i]
    print("minus infinity", ROWS[i], query, flush=True)
    g = torch.Generator().manual_seed(i)
    cu, lens, table, pages, rows = _batch(g, lens, new, 16)
    caches = _cache(g, pages, hk, 16, d, groups)
    y = torch.randn(pages, hk, 16, d, generator=g)
    y[..., 7] = -2.0 - y[..., 7].abs()                # a column of negative keys, so that an infinity there is one in every score
    caches = (orc.quantise(y.double(), groups)[0], caches[1], orc.quantise(y.double(), groups)[1], caches[3])
    assert (orc.values(caches[0], caches[2])[..., 7] < 0).all()
    q = _query(g, rows, hq, d, query)
    args = (*_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), 0.2, 1.0, window, sinks)
    want = _paged().paged_attn_s4(q.to(DEV), *args)
    spoilt = torch.rand(rows, hq, generator=g) < 0.3
    spoilt[0, 0] = True
    q[..., 7] = torch.where(spoilt, float("inf"), q[..., 7])
    got = _paged().paged_attn_s4(q.to(DEV), *args)
    spoilt = spoilt.to(DEV)
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])
    none = torch.zeros_like(lens)                     # a token that sees nothing gets zeros all the same
    got = _paged().paged_attn_s4(q.to(DEV), *args[:5], none.to(DEV), *args[6:])
    assert (got == 0).all()
