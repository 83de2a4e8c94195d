"""The paged KV cache in 4 bits (paged_kv_append_s4, paged_attn_s4, paged_kv_read_s4) against fp64 on the CPU: codes, words and what
is read back exactly, the attention within the bound that its arithmetic gives (tests/_paged_s4_oracle.py)."""
import pytest
import torch

from tests import _paged_s4_oracle as orc
from tests.test_gpu_paged import _angles, _batch, _s8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TWO_FP16, ONE_FP16 = 2.0 ** -22, 2.0 ** -11    # relative errors of weights


def _paged():
    from torch_int.functional import paged_s4
    return paged_s4


def _normal(g, *shape, dtype=torch.float32, spread=1.0):
    return (torch.randn(*shape, generator=g) * spread).to(dtype)


def _query(g, rows, heads, d, dtype):
    return _s8(g, rows, heads, d, spread=30) if dtype is torch.int8 else _normal(g, rows, heads, d, dtype=dtype)


def _alpha(d, dtype):
    return 2.0 / ((30 if dtype is torch.int8 else 1) * d ** 0.5)


def _cache(g, pages, heads, page, d, groups, spread=1.0):
    """A full cache of normal values, with a head or two of another size."""
    out = []
    for _ in range(2):
        y = torch.randn(pages, heads, page, d, generator=g) * spread
        y[:, 0] *= 3.0
        y[:, :, :, 5] += 2.0 * spread
        out.append(orc.quantise(y.double(), groups))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _device(caches, token_major=False):
    """On the device, [pages, heads, page, n], the codes in memory as [pages, page, heads, n] where asked."""
    c = [t.to(DEV) for t in caches]
    if token_major:
        c[:2] = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in c[:2]]
    return tuple(c)


def _attend(case, q, caches, table, lens, cu, a_qk, a_pv=1.0, window=0, sinks=0, weight_error=TWO_FP16, token_major=False, **kw):
    got = _paged().paged_attn_s4(q.to(DEV), *_device(caches, token_major), table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, a_pv, window, sinks,
                                 **kw).cpu()
    want, about = orc.attention(q, caches, table, lens, cu, a_qk, a_pv, window, sinks)
    worst = orc.attention_error(got, want, about, weight_error)
    print("attention", case, "error over its bound", worst, flush=True)
    assert worst <= 1.0
    return got


# query heads, key heads, head size, groups, page, context lengths, new tokens, window, first keys
ATTENTION = [
    (1, 1, 32, 1, 16, [1], [1], 0, 0),
    (2, 2, 48, 2, 16, [0, 1, 15, 16, 17], [0, 1, 1, 1, 1], 0, 0),
    (12, 12, 64, 1, 16, [500], [1], 0, 0),
    (4, 4, 80, 2, 32, [31, 32, 33, 600], [1, 2, 3, 5], 0, 0),
    (8, 2, 112, 1, 64, [64, 65, 0, 130], [1, 1, 0, 1], 0, 0),
    (8, 1, 128, 2, 16, [1000, 3], [2, 3], 0, 0),
    (7, 1, 128, 1, 128, [127, 128, 129], [5, 1, 9], 0, 0),
    (16, 1, 128, 2, 32, [513, 511], [1, 1], 0, 0),
    (24, 8, 64, 2, 16, [257, 255, 254, 31], [4, 1, 2, 31], 0, 0),
    (3, 3, 96, 1, 16, [5, 40], [9, 2], 0, 0),                     # more new tokens than positions: those in front see nothing
    (4, 2, 128, 2, 16, [5000], [1], 0, 0),                        # cut into slices
    (2, 1, 64, 1, 64, [2049, 9, 1030], [3, 1, 17], 0, 0),
    (1, 1, 32, 2, 256, [4097, 4096], [1, 40], 0, 0),
    # windows: of one key, inside a block, over block and page borders, beside first keys, longer than the sequence
    (2, 2, 64, 1, 16, [1, 40, 700], [1, 1, 1], 1, 0),
    (4, 2, 128, 2, 16, [100, 17, 333], [1, 3, 5], 16, 4),
    (8, 1, 80, 1, 32, [600, 64, 31], [2, 1, 31], 50, 1),
    (4, 4, 128, 1, 64, [3000, 90], [1, 4], 1000, 70),
    (3, 1, 48, 2, 16, [400, 400, 8], [7, 1, 8], 33, 16),
    (2, 2, 112, 2, 128, [50, 200], [9, 2], 1000, 20),
    (1, 1, 128, 1, 16, [6000], [2], 4100, 300),                   # a window that is cut into slices
    (5, 5, 32, 2, 16, [20, 90], [40, 3], 12, 3),                  # more new tokens than positions
    # prompts and chunks, single tokens among them, rows and keys that end inside a tile
    (1, 1, 128, 1, 16, [128], [128], 0, 0),
    (8, 2, 128, 2, 16, [700, 130, 64, 0], [300, 130, 1, 0], 0, 0),
    (12, 12, 64, 1, 32, [257, 1], [257, 1], 0, 0),
    (3, 3, 80, 2, 16, [200, 40], [150, 33], 0, 0),
    (5, 1, 48, 1, 64, [65, 300], [64, 13], 0, 0),
    (16, 2, 112, 2, 128, [500, 129, 17], [9, 129, 17], 0, 0),
    (4, 4, 96, 1, 16, [20, 90], [60, 80], 0, 0),
    (2, 1, 128, 2, 16, [6000], [64], 0, 0),
    (24, 8, 64, 2, 256, [3000, 2], [5, 2], 0, 0),
    (8, 2, 128, 2, 16, [700, 130, 64], [300, 130, 1], 100, 5),
    (2, 2, 64, 1, 16, [1000, 300], [500, 300], 17, 0),
    (4, 1, 80, 2, 32, [2000], [130], 700, 40),
    (1, 1, 128, 1, 64, [900], [900], 300, 300),
    # some tens of rows to a sequence, and one over the line
    (8, 2, 128, 2, 16, [300, 77, 12], [12, 11, 12], 0, 0),
    (6, 1, 64, 1, 32, [500], [8], 0, 0),
    (7, 1, 64, 1, 32, [500], [7], 0, 0),
    (12, 4, 80, 2, 64, [200, 90], [16, 15], 60, 3),
]


@pytest.mark.parametrize("query", [torch.int8, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("i", range(len(ATTENTION)))
def test_attention(i, query):
    hq, hk, d, groups, page, lens, new, window, sinks = ATTENTION[i]
    out = [torch.int8, torch.float16, torch.bfloat16][(i + [torch.int8, torch.float16, torch.bfloat16].index(query)) % 3]
    g = torch.Generator().manual_seed(i)
    cu, lens, table, pages, rows = _batch(g, lens, new, page)
    caches = _cache(g, pages, hk, page, d, groups)
    _attend((i, query, out), _query(g, rows, hq, d, query), caches, table, lens, cu, _alpha(d, query), 60.0 if out is torch.int8 else 0.7, window,
            sinks, ONE_FP16, i % 2 == 1, out_dtype=out)


@pytest.mark.parametrize("a_qk", [1e-30, 1e-3, 1.0, 1e4])
def test_attention_of_flat_and_of_peaked_scores(a_qk):
    # from weights that are all equal to one weight that is all
    g = torch.Generator().manual_seed(7)
    cu, lens, table, pages, rows = _batch(g, [700, 90], [1, 3], 16)
    caches = _cache(g, pages, 2, 16, 128, 2)
    for query in (torch.int8, torch.float16):
        q = _query(g, rows, 4, 128, query)
        q[0] = q[0] * 0 - 3
        _attend((a_qk, query), q, caches, table, lens, cu, a_qk, 0.5, out_dtype=torch.float16)


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (100, 5)])
def test_keys_that_outweigh_those_before_them(window, sinks):
    # peaked rows, whose reference moves by 20 powers of two and more from one block of keys to the next; where the heaviest keys'
    # values are 0, as those of 4 bits often are, the context is what the keys before them have left
    g = torch.Generator().manual_seed(1)
    for lens, new in (([700], [300]), ([700, 90], [1, 2])):
        cu, lens, table, pages, rows = _batch(g, lens, new, 16)
        caches = _cache(g, pages, 2, 16, 128, 2)
        q = _query(g, rows, 8, 128, torch.float16)
        _attend((lens, new, window), q, caches, table, lens, cu, 3 * _alpha(128, torch.float16), 1.0, window, sinks,
                ONE_FP16 if rows > 3 else TWO_FP16)


@pytest.mark.parametrize("size", [2.0 ** -17, 2.0 ** -12, 3e-3, 300.0, 3000.0])
def test_values_of_any_size(size):
    # steps from the smallest on, where keys and values are subnormal numbers of fp16, to the largest
    g = torch.Generator().manual_seed(29)
    cu, lens, table, pages, rows = _batch(g, [300, 40], [1, 20], 16)
    caches = _cache(g, pages, 2, 16, 64, 1, spread=size)
    q = _query(g, rows, 4, 64, torch.float16)
    _attend(size, q, caches, table, lens, cu, min(0.25 / size, 1e4), 1.0 / size, out_dtype=torch.bfloat16, weight_error=ONE_FP16)


def test_few_rows_have_weights_of_22_bits():
    g = torch.Generator().manual_seed(3)
    cu, lens, table, pages, rows = _batch(g, [4000, 300], [1, 1], 16)
    caches = _cache(g, pages, 4, 16, 128, 2)
    _attend("22 bits", _query(g, rows, 16, 128, torch.float16), caches, table, lens, cu, 0.05, 30.0, out_dtype=torch.float16)


def test_rows_of_nobody_and_an_output_that_is_handed_in():
    g = torch.Generator().manual_seed(11)
    cu, lens, table, pages, rows = _batch(g, [33, 70], [1, 2], 16, pad=5)
    caches = _cache(g, pages, 2, 16, 64, 2)
    q = _query(g, rows, 4, 64, torch.bfloat16)
    got = _attend("pad", q, caches, table, lens, cu, 0.2)
    assert (got[3:] == 0).all()
    out = torch.full((rows, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    again = _attend("handed in", q[:3], caches, table, lens, cu, 0.2, out=out[:3])
    assert torch.equal(again, got[:3]) and (out[3:] == 7).all()
    out.fill_(7.0)
    args = (q.to(DEV), *_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), 0.2)
    assert _paged().paged_attn_s4(*args, out=out) is out
    assert torch.equal(out[:3].cpu(), got[:3]) and (out[3:] == 7).all()
    cu0 = torch.tensor([2, 3, 5], dtype=torch.int32)      # rows in front of the first sequence are nobody's either
    got = _attend("front", q, caches, table, lens, cu0, 0.2, out_dtype=torch.bfloat16)
    assert (got[:2] == 0).all() and (got[5:] == 0).all()
    none = torch.zeros(1, dtype=torch.int32, device=DEV)  # no sequence at all
    got = _paged().paged_attn_s4(q.to(DEV), *_device(caches), table[:0].to(DEV), none[:0], none, 0.2)
    assert got.dtype is torch.float16 and (got == 0).all()
    empty = _paged().paged_cache_s4(0, 2, 16, 64, 2, DEV)  # a pool without pages
    got = _paged().paged_attn_s4(q.to(DEV), *empty, table.to(DEV), lens.to(DEV), cu.to(DEV), 0.2)
    assert (got == 0).all()


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 5), (300, 0)])
@pytest.mark.parametrize("new", [[1, 1], [1, 300]])
def test_what_no_token_sees_may_be_anything(groups, window, sinks, new):
    # codes and words behind the last position, and outside the windows, of any bits (infinite steps, NaN); tables without pages there
    g = torch.Generator().manual_seed(19)
    page = 16
    cu, lens, table, pages, rows = _batch(g, [700, 333], new, page)
    caches = _cache(g, pages, 2, page, 80, groups)
    q = _query(g, rows, 4, 80, torch.float16)
    want = _attend("clean", q, caches, table, lens, cu, 0.2, 1.0, window, sinks, ONE_FP16)
    dirty = [t.clone() for t in caches]
    bad_table = table.clone()
    for b in range(2):
        n, t = int(lens[b]), int(cu[b + 1] - cu[b])
        first = max(0, n - t - window + 1) if window else 0
        hidden = [j for j in range(-(-n // page) * page) if j >= n or (sinks <= j < first)]
        for j in hidden:
            at = int(table[b, j // page])
            for i, bits in ((0, 0xA5), (1, 0xFF)):
                dirty[i][at, :, j % page] = bits
            for i, bits in ((2, 0x7E0F), (3, -1)):
                dirty[i][at, :, j % page] = bits
        for i in range(table.shape[1]):
            if all(j in hidden for j in range(i * page, (i + 1) * page)):
                bad_table[b, i] = [-1, 2 ** 31 - 1, pages, 0][i % 4]
    got = _attend("dirty", q, dirty, bad_table, lens, cu, 0.2, 1.0, window, sinks, ONE_FP16)
    assert torch.equal(got, want)


def test_a_query_with_infinities_or_nan_spoils_its_own_rows():
    g = torch.Generator().manual_seed(43)
    cu, lens, table, pages, rows = _batch(g, [400, 50, 90], [1, 1, 40], 16)
    caches = _cache(g, pages, 2, 16, 64, 1)
    q = _query(g, rows, 4, 64, torch.float16)
    args = (*_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), 0.2)
    want = _paged().paged_attn_s4(q.to(DEV), *args)
    q[0, 1, 3], q[1, 0, 0], q[5, 2, 7] = float("nan"), float("inf"), -float("inf")
    got = _paged().paged_attn_s4(q.to(DEV), *args)
    spoilt = torch.zeros(rows, 4, dtype=torch.bool, device=DEV)
    spoilt[0, 1] = spoilt[1, 0] = spoilt[5, 2] = True
    assert torch.equal(got[~spoilt], want[~spoilt]) and got[spoilt].isnan().all()


def test_values_out_of_range_touch_nothing_else():
    # pages that the pool does not have, lengths beyond the table, rows beyond the tensor, bounds that descend
    g = torch.Generator().manual_seed(13)
    cu, lens, table, pages, rows = _batch(g, [200, 90, 64], [2, 1, 4], 16)
    caches = _cache(g, pages, 2, 16, 80, 2)
    q = _query(g, rows, 4, 80, torch.float16)
    table[0, 2], table[0, 12], table[1, 0], table[2, :] = -1, pages, 2 ** 31 - 1, -(2 ** 31)
    for window, sinks in ((0, 0), (60, 9)):
        got = _attend("pages", q, caches, table, lens, cu, 0.2, 1.0, window, sinks)
        assert (got[3:] == 0).all()
        q2, cu2, lens2 = _query(g, 90, 8, 80, torch.int8), torch.tensor([0, 60, 61, 90], dtype=torch.int32), lens + 60
        got = _attend("pages, chunks", q2, caches, table, lens2, cu2, 0.01, 1.0, window, sinks, ONE_FP16)
        assert (got[61:] == 0).all()
        for bad_lens in ([2 ** 31 - 1, -5, 64], [10 ** 6, 0, -(2 ** 31)]):
            _attend("lens", q, caches, table, torch.tensor(bad_lens, dtype=torch.int32), cu, 0.2, 1.0, window, sinks)
        for bad_cu in ([0, 2, 3, 10 ** 9], [0, 7, 3, 5], [-4, 2, -9, 2 ** 31 - 1], [5, 0, 7, 6]):
            out = torch.zeros(rows + 2, 4, 80, dtype=torch.float16, device=DEV)
            out[rows:] = 7
            _paged().paged_attn_s4(q.to(DEV), *_device(caches), table.to(DEV), lens.to(DEV), torch.tensor(bad_cu, dtype=torch.int32, device=DEV),
                                   0.2, 1.0, window, sinks, out=out[:rows])
            assert torch.isfinite(out).all() and (out[rows:] == 7).all()


def test_strides_and_offsets_beyond_32_bits():
    # queries inside a fused projection's output, pools whose pages are far apart: the last one begins beyond 2^32
    g = torch.Generator().manual_seed(17)
    cu, lens, table, pages, rows = _batch(g, [300], [2], 16)
    pages = 20
    table[0] = torch.randperm(pages, generator=g)[: table.shape[1]].int()
    table[0, 0] = pages - 1
    big = torch.empty(2 ** 28 * (pages - 1) + 4096, dtype=torch.uint8, device=DEV)
    caches = _cache(g, pages, 2, 16, 80, 2)
    row, words = 2 * 16 * 40, 2 * 16 * 2
    k, v = (big.as_strided((pages, 2, 16, 40), (2 ** 28, 16 * 40, 40, 1), i * row) for i in range(2))
    ks, vs = (big.view(torch.int16).as_strided((pages, 2, 16, 2), (2 ** 27, 32, 2, 1), row + i * words) for i in range(2))
    far = (k, v, ks, vs)
    for t, c in zip(far, caches):
        t.copy_(c)
    fused = _query(g, rows, 8, 80, torch.float16).to(DEV)
    got = _paged().paged_attn_s4(fused[:, 2:6], *far, table.to(DEV), lens.to(DEV), cu.to(DEV), 0.2).cpu()
    want, about = orc.attention(fused[:, 2:6].cpu(), caches, table, lens, cu, 0.2)
    assert orc.attention_error(got, want, about, TWO_FP16) <= 1.0
    kn = torch.randn(rows, 8, 80, generator=g)
    ref, _ = orc.append(kn[:, 1:3], kn[:, 3:5], caches, table, lens, cu, 1.0, 1.5)
    kd = kn.to(DEV)
    _paged().paged_kv_append_s4(kd[:, 1:3], kd[:, 3:5], *far, table.to(DEV), lens.to(DEV), cu.to(DEV), 1.0, 1.5)
    assert all(torch.equal(t.cpu(), r) for t, r in zip(far, ref))
    whole = torch.tensor([0, 300], dtype=torch.int32)
    for a, b in zip(_paged().paged_kv_read_s4(*far, table.to(DEV), lens.to(DEV), whole.to(DEV), 300),
                    orc.read(ref, table, lens, whole, 300, torch.float16)):
        assert torch.equal(a.cpu(), b)


# ---------------------------------------------------------------- appending and reading back
# query heads, key heads, head size, groups, page, context lengths, new tokens, dtype, rotated elements, neighbours, query dtype
APPEND = [
    (12, 12, 64, 1, 16, [500], [1], torch.int8, 0, False, torch.int8),
    (4, 4, 80, 2, 16, [17, 0, 33], [17, 0, 2], torch.float32, 80, False, torch.float16),
    (8, 2, 128, 1, 32, [40, 32, 31], [8, 1, 31], torch.float16, 128, False, torch.int8),
    (8, 2, 128, 2, 32, [40, 32, 31], [8, 1, 31], torch.bfloat16, 64, True, torch.bfloat16),
    (3, 1, 48, 2, 64, [64, 65], [64, 3], torch.float32, 16, True, torch.int8),
    (2, 2, 32, 1, 16, [3, 100], [9, 1], torch.float16, 16, False, torch.bfloat16),      # more new tokens than positions
    (5, 1, 112, 1, 16, [200], [150], torch.bfloat16, 112, False, torch.float16),
    (2, 2, 96, 2, 128, [100, 5], [3, 5], torch.int8, 96, False, torch.int8),            # int8 in, rotated
    (1, 1, 128, 2, 16, [16] * 130, [1] * 130, torch.float32, 32, False, torch.float16),
    (40, 40, 128, 1, 16, [9, 1], [7, 1], torch.float16, 48, False, torch.int8),         # more heads than a block has lanes for
    (64, 8, 64, 2, 16, [21], [21], torch.bfloat16, 64, True, torch.float16),
]


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_and_read_are_exact(i):
    hq, hk, d, groups, page, lens, new, dtype, rot, neighbours, q_dtype = APPEND[i]
    print("append", APPEND[i], flush=True)
    g = torch.Generator().manual_seed(100 + i)
    cu, lens, table, pages, rows = _batch(g, lens, new, page, pad=3)
    caches = _cache(g, pages, hk, page, d, groups)
    if dtype is torch.int8:
        q, kn, vn = (_s8(g, rows, h, d) for h in (hq, hk, hk))
        alphas = (0.7, 0.03, 1.0)
    else:
        q, kn, vn = (_normal(g, rows, h, d, dtype=dtype, spread=1.5) for h in (hq, hk, hk))
        alphas = (31.0 if q_dtype is torch.int8 else 1.0, 1.0, 0.37 if i % 2 else 1.0)
        kn.view(-1)[:3] = torch.tensor([float("nan"), float("inf"), -float("inf")]).to(dtype)
        vn.view(-1)[:4] = torch.tensor([float("nan"), float("inf"), 0.5, 1e4]).to(dtype)
        # a group of zeros, of one value, of one sign, of the smallest numbers, of ties (odd multiples of half a step of 1)
        last = rows - 4
        vn[last, 0] = 0.0
        kn[last, -1] = 2.25
        if last > 0:
            vn[last - 1, 0] = vn[last - 1, 0].abs() + 0.5
            kn[last - 1, -1] = kn[last - 1, -1] * 2.0 ** -21
            vn[last - 1, -1] = (torch.arange(d) % 30 - 14).to(dtype) / 2
            vn[last - 1, -1, 0] = vn[last - 1, -1, d // 2] = 8.0
            vn[last - 1, -1, 1] = vn[last - 1, -1, d // 2 + 1] = -7.0
    cos_sin = _angles(max(lens.tolist()) + 1, rot) if rot else None
    want, want_q = orc.append(kn, vn, caches, table, lens, cu, alphas[1], alphas[2], q, alphas[0], cos_sin, neighbours, q_dtype)
    dev = _device(caches, i % 2 == 0)
    args = (kn.to(DEV), vn.to(DEV), *dev, table.to(DEV), lens.to(DEV), cu.to(DEV), alphas[1], alphas[2])
    kw = dict(alpha_q=alphas[0], cos_sin=None if cos_sin is None else cos_sin.to(DEV), neighbours=neighbours)
    got = _paged().paged_kv_append_s4(*args, query=q.to(DEV), query_dtype=q_dtype, **kw)
    for t, w in zip(dev, want):
        assert torch.equal(t.cpu(), w)
    assert got.dtype is q_dtype and torch.equal(got.cpu(), want_q)
    out = torch.full((rows, hq, d), 9, dtype=q_dtype, device=DEV)
    assert _paged().paged_kv_append_s4(*args, query=q.to(DEV), query_out=out, **kw) is out
    mine = int(cu[-1])
    assert torch.equal(out[:mine].cpu(), want_q[:mine]) and (out[mine:] == 9).all()
    assert _paged().paged_kv_append_s4(*args, **kw) is None
    for t, w in zip(dev, want):
        assert torch.equal(t.cpu(), w)
    batch = (table.to(DEV), lens.to(DEV), cu.to(DEV))
    for out_dtype, alpha in ((torch.float32, 1.0), (torch.float16, 1.0), (torch.bfloat16, 0.3), (torch.int8, 29.7)):
        wanted = orc.read(want, table, lens, cu, rows, out_dtype, alpha, 2 * alpha)
        back = _paged().paged_kv_read_s4(*dev, *batch, rows, out_dtype, alpha, 2 * alpha)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(back, wanted))
        handed = [torch.full((rows, hk, d), 5, dtype=out_dtype, device=DEV) for _ in range(2)]
        _paged().paged_kv_read_s4(*dev, *batch, alpha_k=alpha, alpha_v=2 * alpha, key_out=handed[0], value_out=handed[1])
        assert all(torch.equal(a[:mine].cpu(), b[:mine]) and (a[mine:] == 5).all() for a, b in zip(handed, wanted))


def test_ties_and_borders_go_to_the_even_code():
    # values at and beside every border between two codes, for steps of all 64 mantissas, in fp32 and as numbers of 16 bits
    g = torch.Generator().manual_seed(5)
    rows, d = 128, 128
    steps = orc.STEPS[(15 << 6) + torch.arange(rows) % 64]                     # from 1 on, and halves of them below
    steps[64:] /= 64
    y = torch.zeros(rows, 1, d, dtype=torch.float64)
    at = (torch.arange(d) % 31 - 15).double() / 2 + 0.25 * 0                   # borders and whole steps from -7.5 to 7.5
    y[:, 0] = steps[:, None] * at
    y[:, 0, 0], y[:, 0, 1] = -7.0 * steps, 8.0 * steps
    nudged = y.float()
    up, down = torch.nextafter(nudged, nudged + 1), torch.nextafter(nudged, nudged - 1)
    which = torch.randint(0, 3, nudged.shape, generator=g)
    nudged = torch.where(which == 0, up, torch.where(which == 1, down, nudged))
    nudged[:, 0, :2] = y[:, 0, :2].float()
    cu, lens, table, pages, _ = _batch(g, [rows], [rows], 16)
    for x in (y.float(), nudged, y.to(torch.bfloat16), y.half()):
        caches = _paged().paged_cache_s4(pages, 1, 16, d, 1, "cpu")
        want, _ = orc.append(x, -x, caches, table, lens, cu)
        dev = _device(caches)
        _paged().paged_kv_append_s4(x.to(DEV), (-x).to(DEV), *dev, table.to(DEV), lens.to(DEV), cu.to(DEV))
        assert all(torch.equal(t.cpu(), w) for t, w in zip(dev, want))


def test_append_and_read_out_of_range_touch_nothing_else():
    g = torch.Generator().manual_seed(23)
    cu, lens, table, pages, rows = _batch(g, [40, 20, 90], [4, 5, 3], 16)
    caches = _cache(g, pages, 2, 16, 64, 1)
    kn, vn, q = (torch.randn(rows, 2, 64, generator=g) for _ in range(3))
    cos_sin = _angles(89, 32)      # the third sequence's last token is beyond it
    table[0, 2], table[1, 1] = -1, pages
    for bad_lens, bad_cu in (([40, 20, 90], [0, 4, 9, 12]), ([10 ** 9, -7, 2], [0, 4, 9, 12]), ([40, 20, 90], [0, 4, 9, 10 ** 9]),
                             ([40, 20, 90], [-3, 4, 2, 12])):
        bl, bc = torch.tensor(bad_lens, dtype=torch.int32), torch.tensor(bad_cu, dtype=torch.int32)
        print("out of range", bad_lens, bad_cu, flush=True)
        want, want_q = orc.append(kn, vn, caches, table, bl, bc, 1.0, 1.0, q, 30.0, cos_sin)
        dev = _device(caches)
        batch = (table.to(DEV), bl.to(DEV), bc.to(DEV))
        got = _paged().paged_kv_append_s4(kn.to(DEV), vn.to(DEV), *dev, *batch, query=q.to(DEV), alpha_q=30.0, cos_sin=cos_sin.to(DEV))
        back = _paged().paged_kv_read_s4(*dev, *batch, rows, torch.float32)
        if bad_cu == sorted(bad_cu):
            assert all(torch.equal(t.cpu(), w) for t, w in zip(dev, want)) and torch.equal(got.cpu(), want_q)
            # (a length beyond the table is cut off where positions are looked up, so such rows have none)
            if bad_lens[0] < 10 ** 6:
                assert all(torch.equal(a.cpu(), b) for a, b in zip(back, orc.read(want, table, bl, bc, rows, torch.float32)))


# ---------------------------------------------------------------- the three together, streams and graphs
class _Server:
    """Sequences that grow: a prompt in chunks, then token by token, beside the same in fp64."""

    def __init__(self, seqs, per, page, hq, hk, d, groups, window, sinks, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.hq, self.hk, self.d, self.window, self.sinks = hq, hk, d, window, sinks
        self.table = torch.randperm(seqs * per, generator=self.g).int().view(seqs, per)
        self.lens = torch.zeros(seqs, dtype=torch.int32)
        self.caches = _paged().paged_cache_s4(seqs * per, hk, page, d, groups, "cpu")
        self.dev, self.td = _device(self.caches), self.table.to(DEV)
        self.cs = _angles(per * page, d)
        self.csd = self.cs.to(DEV)

    def step(self, new):
        rows = sum(new)
        self.lens += torch.tensor(new, dtype=torch.int32)
        cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int()
        q, k, v = (_normal(self.g, rows, h, self.d, dtype=torch.float16) for h in (self.hq, self.hk, self.hk))
        batch = (self.td, self.lens.to(DEV), cu.to(DEV))
        qd = _paged().paged_kv_append_s4(k.to(DEV), v.to(DEV), *self.dev, *batch, query=q.to(DEV), cos_sin=self.csd, query_dtype=torch.float16)
        alpha = 2.0 / self.d ** 0.5
        got = _paged().paged_attn_s4(qd, *self.dev, *batch, alpha, 1.0, self.window, self.sinks).cpu()
        self.caches, qs = orc.append(k, v, self.caches, self.table, self.lens, cu, query=q, cos_sin=self.cs, query_dtype=torch.float16)
        assert torch.equal(qd.cpu(), qs) and all(torch.equal(t.cpu(), w) for t, w in zip(self.dev, self.caches))
        want, about = orc.attention(qs, self.caches, self.table, self.lens, cu, alpha, 1.0, self.window, self.sinks)
        worst = orc.attention_error(got, want, about, ONE_FP16)
        print("step", new, worst, flush=True)
        assert worst <= 1.0
        total = int(self.lens.sum())
        whole = torch.cat([torch.zeros(1, dtype=torch.int32), self.lens.cumsum(0).int()])
        back = _paged().paged_kv_read_s4(*self.dev, batch[0], batch[1], whole.to(DEV), total, torch.bfloat16)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(back, orc.read(self.caches, self.table, self.lens, whole, total, torch.bfloat16)))


@pytest.mark.parametrize("hq,hk,d,page,groups,window,sinks", [(8, 2, 64, 16, 1, 0, 0), (4, 4, 128, 32, 2, 50, 4), (6, 1, 80, 64, 1, 20, 0)])
def test_prompts_in_chunks_then_tokens(hq, hk, d, page, groups, window, sinks):
    s = _Server(3, 256 // page, page, hq, hk, d, groups, window, sinks, hq)
    for new in ([40, 7, 1], [64, 100, 0], [1, 1, 33], [1, 1, 1], [3, 1, 2], [0, 1, 0]):
        s.step(new)


def test_the_same_inputs_give_the_same_bits_on_any_stream():
    g = torch.Generator().manual_seed(31)
    cu, lens, table, pages, rows = _batch(g, [6000, 900, 40], [1, 20, 1], 16)
    caches = _device(_cache(g, pages, 2, 16, 128, 2))
    q = _query(g, rows, 8, 128, torch.float16).to(DEV)
    args = (q, *caches, table.to(DEV), lens.to(DEV), cu.to(DEV), 0.1)
    first = _paged().paged_attn_s4(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_paged().paged_attn_s4(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)


@pytest.mark.parametrize("seqs,low,high,long,chunks,window", [
    (65, 1, 200, 0, 0, 0), (70, 1000, 5000, 0, 0, 0), (130, 0, 300, 9000, 0, 0), (256, 1500, 2700, 0, 0, 700),
    (257, 0, 300, 6000, 0, 0), (90, 100, 4000, 9000, 8, 0), (300, 0, 200, 5000, 5, 150), (520, 0, 60, 2000, 0, 0)])
def test_more_sequences_than_a_wave_looks_at(seqs, low, high, long, chunks, window, monkeypatch):
    # short and long ones, some without tokens or keys, one of `long` keys in their middle, chunks among single tokens: against
    # fp64, and the same bits when slices are joined behind the launch
    P = _paged()
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(low, high + 1, (seqs,), generator=g).tolist()
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    if long:
        lens[seqs // 2], new[seqs // 2] = long, 1
    for i in range(chunks):
        new[(i + 1) * seqs // (chunks + 2)] = 40 + 30 * i
    cu, lens, table, pages, rows = _batch(g, lens, new, 16)
    caches = _cache(g, pages, 2, 16, 32, 1)
    q = _query(g, rows, 6, 32, torch.bfloat16)
    a_qk, sinks = _alpha(32, torch.bfloat16), 3 if window else 0
    first = _attend(("many", seqs), q, caches, table, lens, cu, a_qk, 1.0, window, sinks, ONE_FP16).to(DEV)
    args = (q.to(DEV), *_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, 1.0, window, sinks)
    monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))
    assert torch.equal(P.paged_attn_s4(*args), first)


@pytest.mark.parametrize("hq,hk,d,lens,new,window", [
    (1, 1, 128, [70000], [1], 0), (8, 1, 64, [9000, 2, 700], [1, 1, 1], 0), (4, 2, 80, [3000, 2900], [9, 1], 0),
    (32, 2, 128, [5000, 40, 6001], [1, 1, 2], 0), (12, 12, 64, [1025], [1], 0), (4, 2, 128, [4000, 70], [100, 1], 0),
    (1, 1, 64, [3000], [200], 0), (8, 8, 80, [1500], [33], 0), (2, 1, 128, [9000, 50], [1, 1], 5000), (4, 2, 64, [4000, 3000], [70, 3], 2000),
    (8, 2, 128, [4000, 900], [12, 7], 0), (12, 4, 64, [6000], [16], 0), (8, 2, 80, [5000, 4000, 3], [15, 9, 3], 3000)])
def test_slices_that_meet_in_the_launch_or_behind_it(hq, hk, d, lens, new, window, monkeypatch):
    # the same bits with the counters, without them (a second launch), again and again, and after calls whose tables hold
    # nonsense: the counters are zero behind every call; against fp64 as well
    P = _paged()
    from torch_int.functional import paged
    g = torch.Generator().manual_seed(41 + hq)
    cu, lens, table, pages, rows = _batch(g, lens, new, 16)
    caches = _cache(g, pages, hk, 16, d, 2)
    q = _query(g, rows, hq, d, torch.bfloat16)
    a_qk = _alpha(d, torch.bfloat16)
    first = _attend(("meet", hq, hk, d), q, caches, table, lens, cu, a_qk, 1.0, window, 3 if window else 0, ONE_FP16).to(DEV)
    args = (q.to(DEV), *_device(caches), table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, 1.0, window, 3 if window else 0)
    for i in range(30):
        assert torch.equal(P.paged_attn_s4(*args), first), i
    for bad in ([0] + [rows, 0] * len(lens), [-7, 2 ** 31 - 1] * len(lens)):
        bad_cu = torch.tensor(bad[: len(lens) + 1], dtype=torch.int32, device=DEV)
        P.paged_attn_s4(*args[:6], torch.full_like(args[6], 2 ** 31 - 1), bad_cu, *args[8:])
        assert all(int(t.abs().max()) == 0 for t in paged._counters.values())
        assert torch.equal(P.paged_attn_s4(*args), first)
    monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))
    assert torch.equal(P.paged_attn_s4(*args), first)
    monkeypatch.setattr(P._CUDA, "_workspace", lambda *a: (None, 0, 0))     # nothing is cut
    got = P.paged_attn_s4(*args).cpu()
    want, about = orc.attention(q, caches, table, lens, cu, a_qk, 1.0, window, 3 if window else 0)
    assert orc.attention_error(got, want, about, ONE_FP16) <= 1.0


def test_recorded_steps_read_the_batch_when_they_replay():
    from torch_int.nn import PagedAttn_S4, PagedKVAppend_S4, PagedKVRead_S4
    g = torch.Generator().manual_seed(37)
    seqs, per, page, hq, hk, d = 3, 100, 16, 8, 2, 128
    table = torch.randperm(seqs * per, generator=g).int().view(seqs, per).to(DEV)
    cs = _angles(per * page, d).to(DEV)
    lens = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device=DEV)
    rows = 4
    q, k, v = (torch.zeros(rows, h, d, dtype=torch.float16, device=DEV) for h in (hq, hk, hk))
    pools = _device(_cache(g, seqs * per, hk, page, d, 2))
    append, attend = PagedKVAppend_S4.from_scale(1 / 30), PagedAttn_S4.from_scale(1 / 30, softmax_scale=0.1, window=600, sinks=4)
    read = PagedKVRead_S4.from_scale(1 / 30, 1 / 30)
    for m in (append, attend, read):
        m.to(DEV)

    def step(c):
        qs = append(k, v, *c, table, lens, cu, query=q, cos_sin=cs)
        return (qs, attend(qs, *c, table, lens, cu), *read(*c, table, lens, cu, rows))

    recorded = []
    step(tuple(t.clone() for t in pools))
    for _ in range(2):          # two graphs, each with pools of its own
        c = tuple(t.clone() for t in pools)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(c)
        recorded.append((graph, c, out))
    for at, new in (([1, 700, 33], [1, 1, 1]), ([1590, 2, 900], [0, 1, 2]), ([5, 6, 1600], [2, 0, 1]), ([3, 1, 1], [1, 1, 1])):
        lens.copy_(torch.tensor(at, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int())
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).half())
        mine = tuple(t.clone() for t in recorded[0][1])
        want = step(mine)
        torch.cuda.synchronize()
        for graph, _, _ in recorded:
            graph.replay()
        torch.cuda.synchronize()
        for _, c, out in recorded:
            assert all(torch.equal(a, b) for a, b in zip((*c, *out), (*mine, *want)))
