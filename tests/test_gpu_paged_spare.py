"""The paged INT8 KV cache's attention with rows of nobody behind its sequences, as a recorded step of fixed size has them."""
import pytest
import torch

from tests import _paged_cancelling as data
from tests import _paged_oracle as orc
from tests.test_gpu_paged import DEV, EXACT_WEIGHTS, FP16_WEIGHTS, _attend, _batch, _paged, _s8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk,lens,heavy,pad", [(1, [64], 64, 2), (1, [3000], 80, 2), (2, [700], 64, 5), (8, [5000], 64, 17), (1, [20000], 80, 3),
                                               (1, [300], 64, 3000), (1, [3000, 700], 80, 4), (2, [3000, 64, 90], 64, 20)])
def test_spare_rows_do_not_take_bits_from_weights(hk, lens, heavy, pad, monkeypatch):
    # more than 16 rows to a sequence, as the host counts, in sequences of one token: weights of 22 bits, and the bits of a batch without
    P = _paged()
    g = torch.Generator().manual_seed(sum(lens) + pad)
    hq, d = data.HEADS, data.D
    cu, lens_t, table, pages, rows = _batch(g, lens, [1] * len(lens), 16, pad=pad)
    assert rows * hq > 16 * len(lens) * hk
    k, v, q = (_s8(g, *shape, spread=30) for shape in ((pages, hk, 16, d), (pages, hk, 16, d), (rows, hq, d)))
    wants = []
    for b, n in enumerate(lens):
        q[b], kk, vv, at = data.sequence(g, n, heavy)
        pos = torch.arange(n)
        k[table[b].long()[pos // 16], :, pos % 16], v[table[b].long()[pos // 16], :, pos % 16] = kk[:, None], vv[:, None]
        wants.append(data.wanted(q[b], kk, vv, at))
    args = (q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens_t.to(DEV), cu.to(DEV), data.ALPHA, 1.0)
    alone = P.paged_attn_s8(args[0][:len(lens)], *args[1:], out_dtype=torch.float16)
    for where in ("in the launch", "behind it"):
        got = P.paged_attn_s8(*args, out_dtype=torch.float16).cpu()
        for b, (want, size, most) in enumerate(wants):
            worst = orc.attention_error(got[b], want, size, most, heavy, EXACT_WEIGHTS)
            print("22 bits", lens[b], hk, pad, where, "error over its bound", worst, flush=True)
            assert worst <= 1.0
        assert (got[len(lens):] == 0).all()
        if len(lens) == 1:
            assert torch.equal(got[:1], alone.cpu())
        monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))


@pytest.mark.parametrize("hq,hk,d,n,new,pad", [(8, 1, 128, 3000, 40, 9), (4, 2, 64, 900, 300, 40), (64, 8, 128, 40, 0, 7), (28, 4, 80, 1, 1, 8),
                                               (2, 1, 64, 6000, 8, 100), (2, 1, 64, 6000, 9, 100)])
def test_one_sequence_and_spare_rows(hq, hk, d, n, new, pad):
    g = torch.Generator().manual_seed(n + pad)
    cu, lens, table, pages, rows = _batch(g, [n], [new], 16, pad=pad)
    k, v = (_s8(g, pages, hk, 16, d, spread=30).to(DEV) for _ in range(2))
    got = _attend((hq, hk, d, n, new, pad), _s8(g, rows, hq, d, spread=30), k, v, table, lens, cu, 2.0 / (900 * d ** 0.5), 0.02,
                  EXACT_WEIGHTS if new * hq <= 16 * hk else FP16_WEIGHTS, out_dtype=torch.bfloat16)
    assert (got[new:] == 0).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_a_recorded_step_of_one_sequence_is_of_either_kind_when_it_replays(bits):
    # 40 rows, of which a replay's sequence has one, some or all: eager calls, two graphs and their replays in turn
    g = torch.Generator().manual_seed(bits)
    rows, hq, hk, d, page, per = 40, 8, 1, 128, 16, 400
    table = torch.randperm(per, generator=g).int().view(1, per).to(DEV)
    lens, cu = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    q = _s8(g, rows, hq, d, spread=30).to(DEV)
    if bits == 8:
        k, v = (_s8(g, per, hk, page, d, spread=30).to(DEV) for _ in range(2))
        step = lambda: _paged().paged_attn_s8(q, k, v, table, lens, cu, 2e-4, 0.02, out_dtype=torch.float16)  # noqa: E731
    else:
        from tests.test_gpu_paged_s4 import _cache, _device
        from torch_int.functional import paged_s4
        pools = _device(_cache(g, per, hk, page, d, 2))
        step = lambda: paged_s4.paged_attn_s4(q, *pools, table, lens, cu, 6e-3)  # noqa: E731
    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for n, new in ((6000, 1), (6000, 40), (700, 2), (6400, 3), (40, 40), (5000, 0), (6399, 17), (1, 1)):
        lens.fill_(n)
        cu[1] = new
        want = step()
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert (want[new:] == 0).all() and all(torch.equal(out, want) for _, out in graphs), (n, new)
        assert bool(want[:new].any()) or new == 0
