"""That the inputs of tests/_paged_s4_cancelling.py tell weights of 11 bits from weights of 22, on the host: nothing is launched here."""
import pytest
import torch

from tests import _paged_oracle as orc
from tests import _paged_s4_cancelling as data
from tests import _paged_s4_oracle as s4


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("keys,new", [(64, 1), (160, 1), (66, 2), (300, 5)])
def test_the_bound_tells_weights_of_11_bits_from_weights_of_22(keys, new, d):
    # the kernels' way of holding a weight times its value's step, on the CPU: the largest is 2^8, in one fp16 number or in the sum of two
    g = torch.Generator().manual_seed(keys + d)
    heavy = 64
    q, k, v, at = data.sequence(g, keys, heavy, new, 8, d)
    want, size, most = data.wanted(q, k, v, at)
    sees = torch.arange(keys)[None, None] <= torch.arange(keys - new, keys)[:, None, None]
    x = (data.K_STEP * (q.double() @ k.double().T)).float().masked_fill(~sees, float("-inf"))
    c = torch.tensor(data.ALPHA, dtype=torch.float32) * torch.tensor(1.44269504088896341, dtype=torch.float32)
    e = torch.exp2((x.double() * c.double() + (8 - x.amax(-1, keepdim=True) * c).double()).float().double()).float()
    one = e.half().double()
    two = one + (e.double() - one).half().double()
    off = [orc.attention_error((data.V_STEP * (w @ v.double()) / e.double().sum(-1, keepdim=True)).half(), want, size, most, heavy, 2.0 ** -22)
           for w in (one, two)]
    print("error over its bound, 11 bits and 22", off)
    assert off[0] > 2.0 and off[1] <= 1.0


def test_codes_and_words_stand_for_the_values():
    g = torch.Generator().manual_seed(2)
    _, k, v, _ = data.sequence(g, 80, 64, 3, 4, 96)
    for x, step in ((k, data.K_STEP), (v, data.V_STEP)):
        for groups in (1, 2):
            words = torch.full((80, groups), data.word(step), dtype=torch.int16)
            assert torch.equal(s4.values(data.codes(x), words), step * x.double())
