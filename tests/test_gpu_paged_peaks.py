"""The paged INT8 KV cache's attention in tiles where a key's score passes all before it by many powers of two and its values are 0, so
that the context is what the keys before it have left."""
import pytest
import torch

from tests import _paged_oracle as orc
from tests.test_gpu_paged import DEV, _batch, _paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("at", [37, 69, 100])
@pytest.mark.parametrize("powers", [8, 20, 24, 25, 27, 30])
def test_weights_far_below_the_largest_are_the_fp16_numbers_that_they_are_called(powers, at, hq, hk, d):
    # The largest weight counts 2^8 at least, so another is off by 2^-11 of itself, or by 2^-25 / 2^8 of the largest
    g = torch.Generator().manual_seed(powers + at)
    n, new, alpha, scale = 230, 60, 0.25 * 0.6931471805599453, 2.0 ** (powers - 4)   # four units of a score are a power of two
    cu, lens, table, pages, rows = _batch(g, [n], [new], 16)
    keys, values = torch.zeros(n, d), torch.zeros(n, d)
    keys[at, 0] = 4 * powers
    values[: n - new] = torch.randint(0, 100, (n - new, d), generator=g).float()
    values[at] = 0
    k, v = (torch.zeros(pages, hk, 16, d, dtype=torch.int8) for _ in range(2))
    pos = torch.arange(n)
    where = (table[0].long()[pos // 16], slice(None), pos % 16)
    k[where], v[where] = keys.to(torch.int8)[:, None], values.to(torch.int8)[:, None]
    q = torch.zeros(rows, hq, d, dtype=torch.int8)
    q[..., 0] = 1
    args = (q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens.to(DEV), cu.to(DEV), alpha, scale)
    got = _paged().paged_attn_s8(*args, out_dtype=torch.float16).cpu().double()
    want, size, most = orc.attention(q, k, v, table, lens, cu, alpha, scale)
    share = 2 * (most * 2.0 ** -22 * 0.7 + 2.0 ** -22 + 2.0 ** -11) + n * 2.0 ** -24 + 2.0 ** -20      # as in attention_error
    bound = 2.0 ** -11 * want.abs() * (1 + 1e-3) + share * size + 2.0 ** -25 + scale * 2.0 ** -32 * values.abs().sum(0)
    worst = float(((got - want).abs() / bound).max())
    print("peak", powers, at, hq, d, "error over its bound", worst, flush=True)
    assert worst <= 1.0
