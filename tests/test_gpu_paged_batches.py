"""The paged INT8 KV cache in larger batches and behind its modules: more sequences than a wave looks at at once, so many tiles
that none is cut, values on and next to the borders of a rounding, and both operators as a layer uses them."""
import pytest
import torch

from tests import _paged_oracle as orc
from tests.test_gpu_paged import DEV, FP16_WEIGHTS, _angles, _attend, _batch, _paged, _pool, _s8

pytestmark = pytest.mark.gpu


def _many(g, seqs, longest, rows):
    """Lengths and new tokens of many sequences: single tokens, some of a few rows, some chunks, one that is empty."""
    new = [1] * seqs
    for i in range(0, seqs, 5):
        new[i] = int(torch.randint(2, 20, (1,), generator=g))
    for i in range(3, seqs, 16):
        new[i] = rows - i % 7
    lens = [n + int(torch.randint(0, 60, (1,), generator=g)) for n in new]
    lens[seqs // 2] = longest
    lens[-2], new[-2] = 0, 0
    return lens, new


@pytest.mark.parametrize("seqs,hq,hk,d,longest,rows", [(65, 4, 1, 64, 70, 40), (130, 2, 2, 32, 3000, 70), (64, 8, 2, 128, 2500, 140),
                                                       (200, 3, 3, 16, 1500, 33)])
def test_attention_of_many_sequences(seqs, hq, hk, d, longest, rows):
    g = torch.Generator().manual_seed(seqs)
    lens, new = _many(g, seqs, longest, rows)
    cu, lens, table, pages, n = _batch(g, lens, new, 16, pad=3)
    k, v = (_pool(_s8(g, pages, hk, 16, d, spread=30), False) for _ in range(2))
    q = _s8(g, n, hq, d, spread=30)
    _attend((seqs, hq, hk, d), q, k, v, table, lens, cu, 2.0 / (900 * d ** 0.5), 0.02, FP16_WEIGHTS, out_dtype=torch.float16)


def test_so_many_tiles_that_none_is_cut():
    # 26 heads of 64 chunks: over 2048 tiles, so a sequence of 900 keys among them stays whole
    g = torch.Generator().manual_seed(5)
    lens, new = [40] * 63 + [900], [33] * 64
    cu, lens, table, pages, n = _batch(g, lens, new, 16)
    k, v = (_pool(_s8(g, pages, 26, 16, 16, spread=30), False) for _ in range(2))
    q = _s8(g, n, 26, 16, spread=30)
    _attend("whole", q, k, v, table, lens, cu, 5e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.float16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("alpha", [1.0, 0.5, 3.0, 2.0 ** -20, 1e30, 1e-38])
def test_append_next_to_the_borders(dtype, neighbours, alpha):
    # halves of a step and the numbers next to them, unrotated, turned by nothing (position 0), by a quarter, by 45 degrees, where a
    # product nearly cancels the other; the largest and the smallest numbers; what is no number
    g = torch.Generator().manual_seed(17)
    d, page = 64, 16
    cu, lens, table, pages, rows = _batch(g, [32, 7], [32, 7], page)
    kn, vn, q = (torch.randint(-40, 41, (rows, 2, d), generator=g).float() / 2 / min(max(alpha, 1e-20), 1e20) for _ in range(3))
    if dtype is torch.int8:
        kn, vn, q = (torch.randint(-128, 128, (rows, 2, d), generator=g).float() for _ in range(3))
    else:
        for t in (kn, vn, q):
            step = torch.randint(-2, 3, t.shape, generator=g).float()
            t.mul_(1 + step * torch.finfo(dtype).eps)
            flat = t.view(-1)
            flat[3::97] = float("nan")
            flat[5::89] = float("inf")
            flat[9::83] = -3e38
            flat[11::79] = 1e-40
            flat[12::73] = -0.0
    kn, vn, q = (t.to(dtype) for t in (kn, vn, q))
    cs = _angles(40, 32)
    cs[0, :16], cs[0, 16:] = 1.0, 0.0
    cs[1, :16], cs[1, 16:] = 0.0, 1.0
    cs[2:20] = 2.0 ** -0.5
    cs[4, :16] = -(2.0 ** -0.5)
    k, v = (_s8(g, pages, 2, page, d) for _ in range(2))
    want = orc.append(kn, vn, k, v, table, lens, cu, alpha, alpha, q, alpha, cs, neighbours)
    kd, vd = k.to(DEV), v.to(DEV)
    got = _paged().paged_kv_append_s8(kn.to(DEV), vn.to(DEV), kd, vd, table.to(DEV), lens.to(DEV), cu.to(DEV), alpha, alpha,
                                      query=q.to(DEV), alpha_q=alpha, cos_sin=cs.to(DEV), neighbours=neighbours)
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(got.cpu(), want[2])


@pytest.mark.parametrize("out", [torch.int8, torch.float16])
def test_modules_do_what_the_functions_do(out):
    from torch_int.nn import PagedAttn_S8, PagedKVAppend_S8
    g = torch.Generator().manual_seed(23)
    cu, lens, table, pages, rows = _batch(g, [40, 3], [5, 3], 16)
    q, kn, vn = (torch.randn(rows, h, 64, generator=g).half().to(DEV) for h in (4, 2, 2))
    pools = [_s8(g, pages, 2, 16, 64, spread=30).to(DEV) for _ in range(2)]
    batch = (table.to(DEV), lens.to(DEV), cu.to(DEV))
    append = PagedKVAppend_S8.from_scale(torch.tensor(1 / 32), 1 / 16, 1 / 64).to(DEV)
    attend = PagedAttn_S8.from_scale(1 / 64, 1 / 32, 1 / 16, 1 / 64 if out is torch.int8 else None, softmax_scale=0.125).to(DEV)
    a, b = [p.clone() for p in pools], [p.clone() for p in pools]
    qs = append(kn, vn, *a, *batch, query=q, cos_sin=_angles(64, 64).to(DEV))
    got = attend(qs, *a, *batch)
    want_q = _paged().paged_kv_append_s8(kn, vn, *b, *batch, 32.0, 16.0, query=q, alpha_q=64.0, cos_sin=_angles(64, 64).to(DEV))
    want = _paged().paged_attn_s8(want_q, *b, *batch, 2.0 ** -14, 4.0 if out is torch.int8 else 1 / 16, out_dtype=out)
    assert got.dtype is out and torch.equal(qs, want_q) and torch.equal(got, want)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert append(kn, vn, *a, *batch) is None
    into = torch.empty_like(got)
    assert attend(qs, *b, *batch, out=into) is into and torch.equal(into, want)


def test_the_query_is_refused_as_output_and_taken_as_quantised_query():
    g = torch.Generator().manual_seed(29)
    cu, lens, table, pages, rows = _batch(g, [40, 3], [5, 3], 16)
    q, kn, vn = (_s8(g, rows, h, 64, spread=30).to(DEV) for h in (4, 2, 2))
    pools = [_s8(g, pages, 2, 16, 64, spread=30).to(DEV) for _ in range(2)]
    batch = (table.to(DEV), lens.to(DEV), cu.to(DEV))
    with pytest.raises(RuntimeError, match="must not be the query"):
        _paged().paged_attn_s8(q, *pools, *batch, 1e-3, 1.0, out=q)
    kw = dict(alpha_q=0.7, cos_sin=_angles(64, 32).to(DEV))
    want = _paged().paged_kv_append_s8(kn, vn, *[p.clone() for p in pools], *batch, 0.5, 0.5, query=q, **kw)
    assert _paged().paged_kv_append_s8(kn, vn, *pools, *batch, 0.5, 0.5, query=q, query_out=q, **kw) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("new", [1, 40])
def test_a_pool_without_pages(new):
    g = torch.Generator().manual_seed(31)
    lens, cu = torch.tensor([100, 100], dtype=torch.int32), torch.tensor([0, new, 2 * new], dtype=torch.int32)
    table = torch.zeros(2, 7, dtype=torch.int32)
    q, kn, vn = (_s8(g, 2 * new, h, 64, spread=30) for h in (4, 2, 2))
    empty = torch.empty(0, 2, 16, 64, dtype=torch.int8)
    batch = (table.to(DEV), lens.to(DEV), cu.to(DEV))
    pools = (empty.to(DEV), empty.to(DEV))
    got = _paged().paged_kv_append_s8(kn.to(DEV), vn.to(DEV), *pools, *batch, 1.0, 1.0, query=q.to(DEV), alpha_q=0.5)
    assert torch.equal(got.cpu(), orc.append(kn, vn, empty, empty, table, lens, cu, 1.0, 1.0, q, 0.5)[2])
    out = _paged().paged_attn_s8(got, *pools, *batch, 1e-3, 1.0, out_dtype=torch.float16)
    assert out.shape == q.shape and not out.any()


@pytest.mark.parametrize("rows", [5, 300])
def test_rows_without_a_sequence(rows):
    g = torch.Generator().manual_seed(33)
    q, kn, vn = (_s8(g, rows, h, 64, spread=30).to(DEV) for h in (4, 2, 2))
    pools = [_s8(g, 3, 2, 16, 64, spread=30).to(DEV) for _ in range(2)]
    before = [p.clone() for p in pools]
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    batch = (none.view(0, 1).expand(0, 100).contiguous(), none, torch.zeros(1, dtype=torch.int32, device=DEV))
    got = _paged().paged_kv_append_s8(kn, vn, *pools, *batch, 1.0, 1.0, query=q)
    assert not got.any() and torch.equal(pools[0], before[0]) and torch.equal(pools[1], before[1])
    assert not _paged().paged_attn_s8(q, *pools, *batch, 1e-3, 1.0, out_dtype=torch.float16).any()
