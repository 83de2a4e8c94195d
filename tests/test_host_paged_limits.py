"""The paged cache's defaults and bounds, on the host: nothing is launched here."""
import pytest
import torch

from tests import _paged_cancelling as data
from tests import _paged_oracle as orc
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


def test_the_workspace_does_not_grow_with_the_batch():
    # slices of what is cut: at most 1032 of 16 rows, or 520 of 128 rows and 264 of 16, or 1032 of 128 rows
    _, lib = _lib()
    need, counters = lib.ti_paged_attn_workspace_bytes, lib.ti_paged_attn_arrivals
    for seqs in (64, 512, 1024, 4096):
        assert need(seqs, seqs, 32, 32, 128, 4096) == 1032 * 16 * 130 * 4
        assert counters(seqs, seqs, 32, 32, 128, 4096) == 1032
        assert need(seqs, seqs, 64, 64, 128, 1 << 20) == 1032 * 16 * 130 * 4
    for rows, seqs, q_heads, heads in ((600, 64, 8, 2), (4000, 1000, 32, 8), (5000, 4096, 64, 8), (2048, 1, 32, 8), (1 << 20, 4000, 8, 1),
                                       (100000, 1, 4, 1)):
        assert need(rows, seqs, q_heads, heads, 128, 1 << 16) <= 1032 * 128 * 130 * 4
        assert counters(rows, seqs, q_heads, heads, 128, 1 << 16) <= 1032


@pytest.mark.parametrize("keys", [64, 160])
def test_the_bound_tells_weights_of_11_bits_from_weights_of_22(keys):
    # the kernels' way of holding a weight, on the CPU: the largest is 2^8, in one fp16 number or in the sum of two
    g = torch.Generator().manual_seed(keys)
    q, k, v, at = data.sequence(g, keys, keys)
    want, size, most = data.wanted(q, k, v, at)
    x = (q.double() @ k.double().T).float()
    c = torch.tensor(data.ALPHA, dtype=torch.float32) * torch.tensor(1.44269504088896341, dtype=torch.float32)
    e = torch.exp2((x.double() * c.double() + (8 - x.amax(1, keepdim=True) * c).double()).float().double()).float()
    one = e.half().double()
    two = one + (e.double() - one).half().double()
    off = [orc.attention_error(((w @ v.double()) / w.sum(1, keepdim=True)).half(), want, size, most, keys, 2.0 ** -22) for w in (one, two)]
    print("error over its bound, 11 bits and 22", off)
    assert off[0] > 2.0 and off[1] <= 1.0
