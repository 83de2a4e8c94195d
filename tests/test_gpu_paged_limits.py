"""The paged INT8 KV cache at its limits: contexts that are longer than their pages, batches without a sequence,
many sequences of which some are cut."""
import pytest
import torch

from tests import _paged_cancelling as data
from tests import _paged_oracle as orc
from tests.test_gpu_paged import DEV, EXACT_WEIGHTS, FP16_WEIGHTS, _angles, _attend, _batch, _paged, _s8

pytestmark = pytest.mark.gpu


def _one_by_one(cu, lens, table, rows, capacity):
    """The batch with every row a sequence of its own, as long as the row's position makes it, so that no length passes the pages: a
    row whose position does gets no position, as a row at a negative position or of no sequence."""
    own = torch.zeros(rows, dtype=torch.int32)
    whose = torch.zeros(rows, dtype=torch.long)
    for b, n in enumerate(lens.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        for i in range(lo, hi):
            p = n - (hi - i)
            whose[i], own[i] = b, p + 1 if 0 <= p < capacity else 0
    return torch.arange(rows + 1, dtype=torch.int32), own, table[whose].contiguous()


# query heads, key heads, head size, page, pages of a sequence, context lengths, new tokens
BEYOND = [
    (4, 2, 64, 16, 2, [34, 32, 33, 5], [4, 1, 1, 2]),        # the second page ends in the middle of the new tokens
    (2, 1, 128, 16, 3, [2 ** 31 - 1, 48, 10 ** 9], [3, 2, 1]),
    (4, 1, 80, 16, 6, [130, 96, 7], [60, 40, 7]),
    (1, 1, 128, 64, 5, [321, 2 ** 31 - 1], [200, 150]),
]


@pytest.mark.parametrize("rot", [0, 16])
@pytest.mark.parametrize("i", range(len(BEYOND)))
def test_tokens_beyond_the_pages_are_not_appended(i, rot):
    hq, hk, d, page, per, lens, new = BEYOND[i]
    print("beyond", BEYOND[i], flush=True)
    g = torch.Generator().manual_seed(50 + i)
    cu, _, table, pages, rows = _batch(g, [per * page] * len(lens), new, page, pad=2)
    lens = torch.tensor(lens, dtype=torch.int32)
    k, v = _s8(g, pages, hk, page, d), _s8(g, pages, hk, page, d)
    q, kn, vn = (torch.randn(rows, h, d, generator=g) for h in (hq, hk, hk))
    cs = _angles(2 * per * page, rot) if rot else None
    cu1, lens1, table1 = _one_by_one(cu, lens, table, rows, per * page)
    want = orc.append(kn, vn, k, v, table1, lens1, cu1, 30.0, 31.0, q, 29.0, cs)
    kd, vd = k.to(DEV), v.to(DEV)
    got = _paged().paged_kv_append_s8(kn.to(DEV), vn.to(DEV), kd, vd, table.to(DEV), lens.to(DEV), cu.to(DEV), 30.0, 31.0,
                                      query=q.to(DEV), alpha_q=29.0, cos_sin=None if cs is None else cs.to(DEV))
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(got.cpu(), want[2])


@pytest.mark.parametrize("out_type,size", [(1, 2), (3, 1)])
@pytest.mark.parametrize("rows", [5, 300])
def test_no_sequence_beside_a_workspace(rows, out_type, size):
    # through the C entry point, which takes a workspace that nothing needs: rows of nobody become zeros, or stay
    P = _paged()
    g = torch.Generator().manual_seed(rows)
    k, v = (_s8(g, 3, 2, 16, 64).to(DEV) for _ in range(2))
    q = _s8(g, rows, 4, 64).to(DEV)
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    ws = torch.empty(1 << 25, dtype=torch.int8, device=DEV)
    counters = torch.zeros(1 << 12, dtype=torch.int32, device=DEV)
    strides = (2 * 16 * 64, 16 * 64, 64)
    cache = P._Cache(k.data_ptr(), v.data_ptr(), 3, 16, 2, 64, *strides, *strides)
    batch = P._Batch(None, None, cu.data_ptr(), 100, 0, rows)
    for fill in (1, 0):
        out = torch.full((rows * 4 * 64 * size,), 7, dtype=torch.int8, device=DEV)
        what = P._Attn(q.data_ptr(), 4 * 64, 64, 4, out.data_ptr(), out_type, fill, 1e-3, 1.0, counters.data_ptr(), counters.numel())
        rc = P._lib.ti_paged_attn_s8(cache, batch, what, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream or None)
        assert rc == 0, P._lib.ti_last_error()
        torch.cuda.synchronize()
        assert bool((out == (0 if fill else 7)).all()) and not counters.any()


def test_a_module_as_it_is_constructed():
    from torch_int.nn import PagedAttn_S8
    g = torch.Generator().manual_seed(3)
    cu, lens, table, pages, rows = _batch(g, [40, 3], [5, 3], 16)
    k, v = (_s8(g, pages, 2, 16, 64, spread=30).to(DEV) for _ in range(2))
    args = (_s8(g, rows, 4, 64, spread=30).to(DEV), k, v, table.to(DEV), lens.to(DEV), cu.to(DEV))
    assert torch.equal(PagedAttn_S8().to(DEV)(*args), _paged().paged_attn_s8(*args, 0.25, 1.0))


# query heads, key heads, head size, sequences, context lengths of some of them, new tokens of some of them
SOME_CUT = [
    (8, 8, 16, 60, dict.fromkeys(range(60), 2000), {}),                                  # as many slices as there are places for
    (4, 4, 64, 300, {5: 4000, 70: 3000, 131: 900, 299: 3500}, {}),                       # over several looks of 64 sequences
    (2, 1, 128, 129, {0: 2500, 64: 2600, 128: 2700}, {64: 5}),
    (8, 1, 32, 70, {3: 3000, 66: 2500}, {3: 100, 66: 100}),                              # tiles that are cut
    (16, 2, 128, 66, {0: 1500, 1: 40, 30: 1800, 65: 1700}, {0: 40, 1: 20, 30: 64}),      # tiles and few rows, both cut
]


@pytest.mark.parametrize("i", range(len(SOME_CUT)))
def test_slices_of_some_sequences_among_many(i, monkeypatch):
    # the places of the slices are counted apart from the items: right, the same again and again and whoever joins them
    P = _paged()
    hq, hk, d, seqs, longs, news = SOME_CUT[i]
    print("some cut", hq, hk, d, seqs, flush=True)
    g = torch.Generator().manual_seed(70 + i)
    new = [news.get(b, 1) for b in range(seqs)]
    lens = [longs.get(b, 0) or new[b] + int(torch.randint(0, 60, (1,), generator=g)) for b in range(seqs)]
    cu, lens, table, pages, rows = _batch(g, lens, new, 16, pad=1)
    k, v = (_s8(g, pages, hk, 16, d, spread=30).to(DEV) for _ in range(2))
    q = _s8(g, rows, hq, d, spread=30)
    a_qk = 2.0 / (900 * d ** 0.5)
    first = _attend(SOME_CUT[i][:4], q, k, v, table, lens, cu, a_qk, 0.02, FP16_WEIGHTS, out_dtype=torch.float16).to(DEV)
    args = (q.to(DEV), k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, 0.02)
    for _ in range(5):
        assert torch.equal(P.paged_attn_s8(*args, out_dtype=torch.float16), first)
    assert all(int(t.abs().max()) == 0 for t in P._counters.values())
    monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))
    assert torch.equal(P.paged_attn_s8(*args, out_dtype=torch.float16), first)


def test_bounds_that_descend_leave_places_and_counters_alone():
    # cu_new counts its rows many times over: more items and slices than there are workgroups or places for
    P = _paged()
    g = torch.Generator().manual_seed(81)
    for seqs, rows, hq, hk in ((200, 100, 8, 8), (66, 300, 8, 1)):
        cu, lens, table, pages, _ = _batch(g, [3000] + [20] * (seqs - 1), [1] * seqs, 16)
        table[:] = table[0]
        k, v = (_s8(g, pages, hk, 16, 64, spread=30).to(DEV) for _ in range(2))
        q = _s8(g, rows, hq, 64, spread=30).to(DEV)
        cu = torch.tensor([0, rows] * (seqs // 2) + [rows], dtype=torch.int32, device=DEV)
        lens = torch.where(torch.arange(seqs) % 20 == 0, 3000, rows + 20).int().to(DEV)
        out = torch.zeros(rows + 2, hq, 64, dtype=torch.float16, device=DEV)
        out[rows:] = 7
        print("descending", seqs, rows, flush=True)
        P.paged_attn_s8(q, k, v, table.to(DEV), lens, cu, 3e-4, 0.02, out=out[:rows])
        assert torch.isfinite(out).all() and (out[rows:] == 7).all()
        assert all(int(t.abs().max()) == 0 for t in P._counters.values())


@pytest.mark.parametrize("hk", [1, data.HEADS])
@pytest.mark.parametrize("lens,heavy,chunk", [([64], 64, 0), ([160, 64, 31], 64, 0), ([3000], 80, 0), ([3000, 700, 5000], 80, 0),
                                              ([3000, 64], 64, 40)])
def test_single_tokens_have_weights_of_22_bits(lens, heavy, chunk, hk, monkeypatch):
    # whole, in slices that meet in the launch or behind it, beside a chunk that goes by tiles
    P = _paged()
    g = torch.Generator().manual_seed(sum(lens) + heavy)
    hq, d = data.HEADS, data.D
    new = [1] * len(lens) + [chunk] * (chunk > 0)
    cu, lens_t, table, pages, rows = _batch(g, lens + [chunk] * (chunk > 0), new, 16)
    k, v, q = (_s8(g, *shape, spread=30) for shape in ((pages, hk, 16, d), (pages, hk, 16, d), (rows, hq, d)))
    wants = []
    for b, n in enumerate(lens):
        q[b], kk, vv, at = data.sequence(g, n // 2 * 2, min(heavy, n // 2 * 2))
        pos = torch.arange(n // 2 * 2)
        lens_t[b] = len(pos)
        k[table[b].long()[pos // 16], :, pos % 16], v[table[b].long()[pos // 16], :, pos % 16] = kk[:, None], vv[:, None]
        wants.append((data.wanted(q[b], kk, vv, at), len(at)))
    args = (q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens_t.to(DEV), cu.to(DEV), data.ALPHA, 1.0)
    for where in ("in the launch", "behind it"):
        got = P.paged_attn_s8(*args, out_dtype=torch.float16).cpu()
        for b, ((want, size, most), keys) in enumerate(wants):
            worst = orc.attention_error(got[b], want, size, most, keys, EXACT_WEIGHTS)
            print("22 bits", lens[b], hk, where, "error over its bound", worst, flush=True)
            assert worst <= 1.0
        monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))
