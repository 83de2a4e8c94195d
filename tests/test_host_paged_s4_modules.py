"""The scales of the modules around the 4-bit paged cache, on the host: nothing is launched here."""
import pytest
import torch


@pytest.mark.parametrize("q_scale,q_input,want", [(None, 1.0, 1.0), (None, 0.02, 0.02), (0.25, 1.0, 4.0), (0.02, 0.02, 1.0), (0.5, 0.125, 0.25)])
def test_int8_queries_have_a_step_of_their_own(q_scale, q_input, want):
    from torch_int.nn import PagedKVAppend_S4
    for one in (lambda x: x, lambda x: None if x is None else torch.tensor(x)):
        mod = PagedKVAppend_S4.from_scale(one(q_scale), 0.5, 0.125, q_input_scale=one(q_input))
        assert float(mod.a_q) == pytest.approx(want, rel=1e-6) and float(mod.a_k) == 0.5 and float(mod.a_v) == 0.125
        assert mod.query_dtype is (torch.float16 if q_scale is None else torch.int8) and mod.a_q.dim() == 0
