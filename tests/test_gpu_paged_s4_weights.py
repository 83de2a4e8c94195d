"""The 4-bit paged cache's attention: which weights have 22 bits, on inputs where weights of 11 bits break the bound
(tests/_paged_s4_cancelling.py, shown on the CPU by tests/test_host_paged_s4_weights.py)."""
import pytest
import torch

from tests import _paged_oracle as orc
from tests import _paged_s4_cancelling as data
from tests.test_gpu_paged import _batch, _s8
from tests.test_gpu_paged_s4 import DEV, ONE_FP16, TWO_FP16, _attend, _cache, _device, _paged

pytestmark = pytest.mark.gpu


def _cancelling(g, hq, hk, d, groups, lens, new, heavy, pad=0, chunk=0):
    """A batch of such sequences, ``pad`` rows of nobody behind them and, where asked, a chunk of another kind of keys: the
    arguments of a call but for its window, and what the sequences' rows are to be."""
    cu, lens_t, table, pages, rows = _batch(g, lens + [chunk] * (chunk > 0), new + [chunk] * (chunk > 0), 16, pad=pad)
    caches = _cache(g, pages, hk, 16, d, groups)
    q = _s8(g, rows, hq, d, spread=30)
    wants = []
    for b, (n, t) in enumerate(zip(lens, new)):
        mine = slice(int(cu[b]), int(cu[b + 1]))
        q[mine], k, v, at = data.sequence(g, n, heavy, t, hq, d)
        pos = torch.arange(n)
        where = table[b].long()[pos // 16], slice(None), pos % 16
        for codes, words, x, step in ((caches[0], caches[2], k, data.K_STEP), (caches[1], caches[3], v, data.V_STEP)):
            codes[where], words[where] = data.codes(x)[:, None], data.word(step)
        wants.append((mine, data.wanted(q[mine], k, v, at)))
    return (q, caches, table, lens_t, cu), wants


def _check(case, args, wants, heavy, query, monkeypatch):
    P = _paged()
    q, caches, table, lens, cu = args
    call = (q.to(query).to(DEV), *_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), data.ALPHA, 1.0)
    for where in ("in the launch", "behind it"):
        got = P.paged_attn_s4(*call, out_dtype=torch.float16).cpu()
        for mine, (want, size, most) in wants:
            worst = orc.attention_error(got[mine], want, size, most, heavy, TWO_FP16)
            print("22 bits", case, where, "rows", mine, "error over its bound", worst, flush=True)
            assert worst <= 1.0
        assert (got[int(cu[-1]):] == 0).all()
        monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))


# query heads, key heads, head size, context lengths, new tokens, a chunk
EXACT = [
    (8, 8, 64, [64], [1], 0),
    (8, 1, 128, [160, 64, 90], [1, 1, 2], 0),           # up to 16 rows
    (16, 1, 80, [3000], [1], 0),                        # 16 rows, in slices
    (8, 2, 96, [3000, 700, 5000], [1, 4, 2], 0),
    (8, 1, 64, [3000, 500], [2, 1], 40),                # up to 16 rows beside a chunk
    (8, 1, 128, [300, 200], [5, 6], 0),                 # 40 and 48 rows, 44 on average
    (8, 2, 64, [4000, 80, 90, 100], [30, 1, 1, 1], 0),  # 120 rows, 33 on average
    (4, 4, 80, [130], [40], 0),
]


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("i", range(len(EXACT)))
def test_weights_of_22_bits(i, groups, monkeypatch):
    hq, hk, d, lens, new, chunk = EXACT[i]
    args, wants = _cancelling(torch.Generator().manual_seed(i), hq, hk, d, groups, lens, new, 64, 0, chunk)
    _check((EXACT[i], groups), args, wants, 64, [torch.int8, torch.float16, torch.bfloat16][i % 3], monkeypatch)


# query heads, key heads, head size, context lengths, new tokens, rows of nobody: more than 48 rows to a sequence, as the host counts
SPARE = [
    (16, 1, 128, [400], [1], 3),
    (16, 1, 64, [20000], [1], 3),
    (64, 8, 128, [5000], [1], 6),
    (28, 4, 80, [3000], [2], 7),
    (8, 1, 96, [3000], [2], 5),
    (4, 4, 64, [200], [16], 60),
    (16, 1, 128, [3000, 90], [1, 1], 5),
    (8, 1, 64, [700, 3000, 66], [1, 1, 2], 17),
    (2, 1, 64, [100], [1], 3000),
]


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("i", range(len(SPARE)))
def test_spare_rows_do_not_take_bits_from_weights(i, groups, monkeypatch):
    # rows of nobody behind a recorded step's sequences: those still have up to 16 rows, and weights of 22 bits
    hq, hk, d, lens, new, pad = SPARE[i]
    assert (sum(new) + pad) * hq > 48 * len(lens) * hk and max(new) * hq <= 16 * hk
    args, wants = _cancelling(torch.Generator().manual_seed(50 + i), hq, hk, d, groups, lens, new, 64, pad)
    _check((SPARE[i], groups), args, wants, 64, [torch.int8, torch.float16, torch.bfloat16][i % 3], monkeypatch)


@pytest.mark.parametrize("hq,hk,d,groups,n,new,pad,window,sinks", [
    (16, 1, 128, 2, 6000, 1, 4, 0, 0), (8, 1, 80, 1, 2000, 2, 30, 700, 5), (28, 4, 64, 1, 1, 1, 8, 0, 0), (64, 8, 128, 2, 40, 0, 7, 0, 0),
    (8, 1, 128, 1, 3000, 40, 9, 0, 0), (4, 2, 64, 2, 900, 300, 40, 100, 3)])
def test_one_sequence_and_spare_rows(hq, hk, d, groups, n, new, pad, window, sinks):
    g = torch.Generator().manual_seed(n + pad)
    cu, lens, table, pages, rows = _batch(g, [n], [new], 16, pad=pad)
    caches = _cache(g, pages, hk, 16, d, groups)
    q = torch.randn(rows, hq, d, generator=g).half()
    got = _attend((hq, hk, d, n, new, pad), q, caches, table, lens, cu, 2.0 / d ** 0.5, 1.0, window, sinks,
                  TWO_FP16 if new * hq <= 16 * hk else ONE_FP16, out_dtype=torch.bfloat16)
    assert (got[new:] == 0).all()


@pytest.mark.parametrize("hq,hk,d,groups,lens,new", [(8, 2, 64, 2, [300], [2]), (16, 1, 128, 1, [3000, 90], [1, 1]), (4, 4, 96, 2, [200], [30])])
@pytest.mark.parametrize("powers", [3, 10, 14, 17])
def test_values_of_larger_steps_beside_take_bits_that_are_stated(powers, hq, hk, d, groups, lens, new):
    # a light key in front of the others whose values' step is 2^powers of theirs: a weight is off by 2^-22 of itself, or by 2^-32 of the
    # largest weight times that, which here is as large as all the others but for some powers of two
    P = _paged()
    (q, caches, table, lens_t, cu), wants = _cancelling(torch.Generator().manual_seed(powers), hq, hk, d, groups, lens, new, 64)
    heavy = 64
    for b in range(len(lens)):
        at = heavy // 2           # behind the first heavy keys
        caches[3][int(table[b, at // 16]), :, at % 16] = data.word(data.V_STEP * 2.0 ** (powers - 10))
        pos = [j for j in range(lens[b]) if j != at]
        for j in pos:
            caches[3][int(table[b, j // 16]), :, j % 16] = data.word(data.V_STEP * 2.0 ** -10)
    got = P.paged_attn_s4(q.to(DEV), *_device(caches), table.to(DEV), lens_t.to(DEV), cu.to(DEV), data.ALPHA, 1024.0, out_dtype=torch.float16).cpu()
    for mine, (want, size, most) in wants:
        # (scores are within 2^(3 * 16 * 15 / 256) = 2^2.9 of one another, so the sum of weights is 64 / 2^2.9 of the largest at least)
        error = max(TWO_FP16, 2.0 ** -32 * 2.0 ** powers * 2.0 ** 2.9)
        worst = orc.attention_error(got[mine], want, size, most, heavy, error)
        print("steps", powers, hq, d, "error over its bound", worst, flush=True)
        assert worst <= 1.0
