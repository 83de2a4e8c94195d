"""The modules around the 4-bit paged cache whose inputs are int8, against fp64 on the CPU (tests/_paged_s4_oracle.py)."""
import pytest
import torch

from tests import _paged_s4_oracle as orc
from tests.test_gpu_paged import _angles, _batch, _s8
from tests.test_gpu_paged_s4 import DEV, _cache, _device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rot", [0, 64])
@pytest.mark.parametrize("q_scale,query_dtype", [(0.02, torch.int8), (0.031, torch.int8), (None, torch.float16), (None, torch.bfloat16)])
def test_int8_inputs_have_steps_of_their_own(q_scale, query_dtype, rot):
    from torch_int.nn import PagedKVAppend_S4
    g = torch.Generator().manual_seed(rot)
    cu, lens, table, pages, rows = _batch(g, [40, 21], [5, 1], 16)
    caches = _cache(g, pages, 2, 16, 64, 2)
    q, k, v = (_s8(g, rows, h, 64, spread=30) for h in (4, 2, 2))
    cs = _angles(64, rot) if rot else None
    steps = dict(q_input_scale=0.02, k_input_scale=0.05, v_input_scale=0.0625)
    append = PagedKVAppend_S4.from_scale(q_scale, **steps, query_dtype=query_dtype if q_scale is None else torch.float16).to(DEV)
    alpha = 0.02 if q_scale is None else float(append.a_q)
    assert alpha == pytest.approx(0.02 / (q_scale or 1.0), rel=1e-6)
    want, want_q = orc.append(k, v, caches, table, lens, cu, 0.05, 0.0625, q, alpha, cs, query_dtype=query_dtype)
    dev = _device(caches)
    got = append(k.to(DEV), v.to(DEV), *dev, table.to(DEV), lens.to(DEV), cu.to(DEV), query=q.to(DEV), cos_sin=None if cs is None else cs.to(DEV))
    assert got.dtype is query_dtype and torch.equal(got.cpu(), want_q)
    assert all(torch.equal(t.cpu(), w) for t, w in zip(dev, want))
    if q_scale == 0.02 and not rot:
        assert torch.equal(got.cpu(), q)      # the same step before and behind
