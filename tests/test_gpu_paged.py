"""The paged INT8 KV cache (paged_kv_append_s8, paged_attn_s8) against fp64 on the CPU: the appended bytes exactly, the
attention within the bound that its arithmetic gives (tests/_paged_oracle.py)."""
import pytest
import torch

from tests import _paged_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EXACT_WEIGHTS, FP16_WEIGHTS = 2.0 ** -22, 2.0 ** -11


def _paged():
    from torch_int.functional import paged
    return paged


def _s8(g, *shape, spread=None):
    if spread is None:
        return torch.randint(-128, 128, shape, dtype=torch.int8, generator=g)
    return (torch.randn(*shape, generator=g) * spread).round().clamp(-127, 127).to(torch.int8)


def _batch(g, lens, new, page, spare=2, pad=0):
    """cu_new, context_lens, block_table with pages dealt at random, number of pages, rows."""
    per = max([1] + [-(-n // page) for n in lens])
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    at = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), per), -1, dtype=torch.int32)
    k = 0
    for b, n in enumerate(need):
        table[b, :n] = at[k:k + n].int()
        k += n
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    return (torch.tensor(cu, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), table, pages, cu[-1] + pad)


def _pool(t, token_major):
    """The pool on the device, [pages, heads, page, d], in memory as [pages, page, heads, d] where asked."""
    t = t.to(DEV)
    return t.transpose(1, 2).contiguous().transpose(1, 2) if token_major else t


def _attend(case, q, k, v, table, lens, cu, a_qk, a_pv, weight_error, **kw):
    got = _paged().paged_attn_s8(q.to(DEV), k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, a_pv, **kw).cpu()
    want, size, most = orc.attention(q, k.cpu(), v.cpu(), table, lens, cu, a_qk, a_pv)
    worst = orc.attention_error(got, want, size, most, int(max([1] + lens.tolist())), weight_error)
    print("attention", case, "error over its bound", worst, flush=True)
    assert worst <= 1.0
    return got


# query heads, key heads, head size, page, context lengths, new tokens
ATTENTION = [
    (1, 1, 16, 16, [1], [1]),
    (2, 2, 48, 16, [0, 1, 15, 16, 17], [0, 1, 1, 1, 1]),
    (12, 12, 64, 16, [500], [1]),
    (4, 4, 80, 32, [31, 32, 33, 600], [1, 2, 3, 5]),
    (8, 2, 112, 64, [64, 65, 0, 130], [1, 1, 0, 1]),
    (8, 1, 128, 16, [1000, 3], [2, 3]),
    (7, 1, 128, 128, [127, 128, 129], [5, 1, 9]),
    (16, 1, 128, 32, [513, 511], [1, 1]),
    (24, 8, 64, 16, [257, 255, 254, 31], [4, 1, 2, 31]),
    (3, 3, 96, 16, [5, 40], [9, 2]),                     # more new tokens than positions: those in front see nothing
    (4, 2, 128, 16, [5000], [1]),                        # cut into slices
    (2, 1, 64, 64, [2049, 9, 1030], [3, 1, 17]),
    (1, 1, 32, 256, [4097, 4096], [1, 40]),
    # tiles of 128 rows: whole prompts, chunks, single tokens among them, rows and keys that end inside a tile
    (1, 1, 128, 16, [128], [128]),
    (8, 2, 128, 16, [700, 130, 64, 0], [300, 130, 1, 0]),
    (12, 12, 64, 32, [257, 1], [257, 1]),
    (3, 3, 80, 16, [200, 40], [150, 33]),
    (5, 1, 48, 64, [65, 300], [64, 13]),
    (16, 2, 112, 128, [500, 129, 17], [9, 129, 17]),
    (4, 4, 96, 16, [20, 90], [60, 80]),                  # more new tokens than positions
    (2, 1, 128, 16, [6000], [64]),                       # cut into slices
    (24, 8, 64, 256, [3000, 2], [5, 2]),
]


@pytest.mark.parametrize("out", [torch.int8, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("i", range(len(ATTENTION)))
def test_attention(i, out):
    hq, hk, d, page, lens, new = ATTENTION[i]
    g = torch.Generator().manual_seed(i)
    cu, lens, table, pages, rows = _batch(g, lens, new, page)
    k, v = (_pool(_s8(g, pages, hk, page, d, spread=30), i % 2 == 1) for _ in range(2))
    q = _s8(g, rows, hq, d, spread=30)
    a_qk = 2.0 / (900 * d ** 0.5)
    _attend((i, out), q, k, v, table, lens, cu, a_qk, 6.0 if out is torch.int8 else 0.02, FP16_WEIGHTS, out_dtype=out)


@pytest.mark.parametrize("a_qk", [1e-30, 1e-6, 3e-3, 0.25])
def test_attention_of_flat_and_of_peaked_scores(a_qk):
    # values over the whole range of int8; from weights that are all equal to one weight that is all; scores up to 2^21
    g = torch.Generator().manual_seed(7)
    cu, lens, table, pages, rows = _batch(g, [700, 90], [1, 3], 16)
    k, v = (_pool(_s8(g, pages, 2, 16, 128), False) for _ in range(2))
    k[int(table[0, 3]), :, 5] = -128
    q = _s8(g, rows, 4, 128)
    q[0] = -128
    _attend(a_qk, q, k, v, table, lens, cu, a_qk, 0.5, FP16_WEIGHTS, out_dtype=torch.float16)
    _attend(a_qk, q, k, v, table, lens, cu, a_qk, 1.0, FP16_WEIGHTS)


def test_few_rows_have_weights_of_22_bits():
    # one key among 4000 that outweighs the rest, and values whose sum nearly cancels: fp16 weights would show
    g = torch.Generator().manual_seed(3)
    cu, lens, table, pages, rows = _batch(g, [4000, 300], [1, 1], 16)
    k, v = (_pool(_s8(g, pages, 4, 16, 128, spread=30), False) for _ in range(2))
    q = _s8(g, rows, 16, 128, spread=30)
    _attend("22 bits", q, k, v, table, lens, cu, 1e-4, 2e-2, EXACT_WEIGHTS, out_dtype=torch.float16)


def test_rows_of_nobody_and_an_output_that_is_handed_in():
    g = torch.Generator().manual_seed(11)
    cu, lens, table, pages, rows = _batch(g, [33, 70], [1, 2], 16, pad=5)
    k, v = (_pool(_s8(g, pages, 2, 16, 64, spread=30), False) for _ in range(2))
    q = _s8(g, rows, 4, 64, spread=30)
    got = _attend("pad", q, k, v, table, lens, cu, 3e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.float16)
    assert (got[3:] == 0).all()
    out = torch.full((rows, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    again = _attend("handed in", q[:3], k, v, table, lens, cu, 3e-4, 0.02, FP16_WEIGHTS, out=out[:3])
    assert torch.equal(again, got[:3]) and (out[3:] == 7).all()
    out.fill_(7.0)
    args = (q.to(DEV), k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), 3e-4, 0.02)
    assert _paged().paged_attn_s8(*args, out=out) is out
    assert torch.equal(out[:3].cpu(), got[:3]) and (out[3:] == 7).all()
    cu0 = torch.tensor([2, 3, 5], dtype=torch.int32)      # rows in front of the first sequence are nobody's either
    got = _attend("front", q, k, v, table, lens, cu0, 3e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.bfloat16)
    assert (got[:2] == 0).all() and (got[5:] == 0).all()
    none = torch.zeros(1, dtype=torch.int32, device=DEV)  # no sequence at all
    got = _paged().paged_attn_s8(q.to(DEV), k, v, table[:0].to(DEV), none[:0], none, 3e-4, 0.02)
    assert got.dtype is torch.int8 and (got == 0).all()


def test_values_out_of_range_touch_nothing_else():
    # pages that the pool does not have, lengths beyond the table, rows beyond the tensor, bounds that descend
    g = torch.Generator().manual_seed(13)
    cu, lens, table, pages, rows = _batch(g, [200, 90, 64], [2, 1, 4], 16)
    k, v = (_pool(_s8(g, pages, 2, 16, 80, spread=30), False) for _ in range(2))
    q = _s8(g, rows, 4, 80, spread=30)
    table[0, 2], table[0, 12], table[1, 0], table[2, :] = -1, pages, 2 ** 31 - 1, -(2 ** 31)
    got = _attend("pages", q, k, v, table, lens, cu, 3e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.float16)
    assert (got[3:] == 0).all()
    q128, cu128, lens128 = _s8(g, 90, 8, 80, spread=30), torch.tensor([0, 60, 61, 90], dtype=torch.int32), lens + 60
    got = _attend("pages, tiles", q128, k, v, table, lens128, cu128, 3e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.float16)
    assert (got[61:] == 0).all()
    for bad_lens in ([2 ** 31 - 1, -5, 64], [10 ** 6, 0, -(2 ** 31)]):
        _attend("lens", q, k, v, table, torch.tensor(bad_lens, dtype=torch.int32), cu, 3e-4, 0.02, FP16_WEIGHTS, out_dtype=torch.float16)
    for bad_cu in ([0, 2, 3, 10 ** 9], [0, 7, 3, 5], [-4, 2, -9, 2 ** 31 - 1], [5, 0, 7, 6]):
        out = torch.zeros(rows + 2, 4, 80, dtype=torch.float16, device=DEV)
        out[rows:] = 7
        _paged().paged_attn_s8(q.to(DEV), k, v, table.to(DEV), lens.to(DEV), torch.tensor(bad_cu, dtype=torch.int32, device=DEV),
                               3e-4, 0.02, out=out[:rows])
        assert torch.isfinite(out).all() and (out[rows:] == 7).all()


def test_strides_and_offsets_beyond_32_bits():
    # queries inside a fused projection's output, a pool whose pages are 2^28 bytes apart: the last one begins beyond 2^32
    g = torch.Generator().manual_seed(17)
    cu, lens, table, pages, rows = _batch(g, [300], [2], 16)
    pages = 20
    table[0] = torch.randperm(pages, generator=g)[: table.shape[1]].int()
    table[0, 0] = pages - 1
    big = torch.empty(2 ** 28 * (pages - 1) + 2 * 2 * 16 * 64, dtype=torch.int8, device=DEV)
    k = big.as_strided((pages, 2, 16, 64), (2 ** 28, 16 * 64, 64, 1))
    v = big.as_strided((pages, 2, 16, 64), (2 ** 28, 16 * 64, 64, 1), 2 * 16 * 64)
    k.copy_(_s8(g, pages, 2, 16, 64, spread=30))
    v.copy_(_s8(g, pages, 2, 16, 64, spread=30))
    fused = _s8(g, rows, 8, 64, spread=30).to(DEV)
    q = fused[:, 2:6]
    got = _paged().paged_attn_s8(q, k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), 3e-4, 0.02, out_dtype=torch.float16).cpu()
    want, size, most = orc.attention(q.cpu(), k.cpu(), v.cpu(), table, lens, cu, 3e-4, 0.02)
    assert orc.attention_error(got, want, size, most, 300, FP16_WEIGHTS) <= 1.0
    kn = torch.randn(rows, 8, 64, generator=g, dtype=torch.float32)
    k_ref, v_ref, _ = orc.append(kn[:, 1:3], kn[:, 3:5], k.cpu(), v.cpu(), table, lens, cu, 30.0, 31.0)
    kd = kn.to(DEV)
    _paged().paged_kv_append_s8(kd[:, 1:3], kd[:, 3:5], k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), 30.0, 31.0)
    assert torch.equal(k.cpu(), k_ref) and torch.equal(v.cpu(), v_ref)


# ---------------------------------------------------------------- appending
# query heads, key heads, head size, page, context lengths, new tokens, dtype, rotated elements, neighbours
APPEND = [
    (12, 12, 64, 16, [500], [1], torch.int8, 0, False),
    (4, 4, 80, 16, [17, 0, 33], [17, 0, 2], torch.float32, 80, False),
    (8, 2, 128, 32, [40, 32, 31], [8, 1, 31], torch.float16, 128, False),
    (8, 2, 128, 32, [40, 32, 31], [8, 1, 31], torch.bfloat16, 64, True),
    (3, 1, 48, 64, [64, 65], [64, 3], torch.float32, 16, True),
    (2, 2, 16, 16, [3, 100], [9, 1], torch.float16, 16, True),      # more new tokens than positions
    (5, 1, 112, 16, [200], [150], torch.bfloat16, 112, False),
    (2, 2, 96, 128, [100, 5], [3, 5], torch.int8, 96, False),       # int8 in, rotated
    (1, 1, 128, 16, [16] * 130, [1] * 130, torch.float32, 32, False),
]


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_is_exact(i):
    hq, hk, d, page, lens, new, dtype, rot, neighbours = APPEND[i]
    print("append", APPEND[i], flush=True)
    g = torch.Generator().manual_seed(100 + i)
    cu, lens, table, pages, rows = _batch(g, lens, new, page, pad=3)
    k, v = _s8(g, pages, hk, page, d), _s8(g, pages, hk, page, d)
    if dtype is torch.int8:
        q, kn, vn = (_s8(g, rows, h, d) for h in (hq, hk, hk))
        alphas = (1.0, 0.7, 1.0)
    else:
        q, kn, vn = ((torch.randn(rows, h, d, generator=g) * 1.5).to(dtype) for h in (hq, hk, hk))
        alphas = (31.0, 47.3, 29.0)
        kn.view(-1)[:3] = torch.tensor([float("nan"), float("inf"), -float("inf")]).to(dtype)
        vn.view(-1)[:4] = torch.tensor([float("nan"), float("inf"), 0.5, 1e4]).to(dtype)
        q.view(-1)[5] = float("nan")
        # ties, to even: 0.5 and 1.5 steps
        vn[1, 0, 8:12] = torch.tensor([0.5, 1.5, -0.5, -2.5]).to(dtype)
        alphas = (31.0, 47.3, 1.0) if i % 2 else alphas
    cos_sin = None
    if rot:
        angle = torch.arange(max(lens.tolist()) + 1, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(rot // 2).double() / rot)
        cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    want = orc.append(kn, vn, k, v, table, lens, cu, alphas[1], alphas[2], q, alphas[0], cos_sin, neighbours)
    kd, vd = _pool(k, i % 2 == 0), _pool(v, i % 3 == 0)
    args = (kn.to(DEV), vn.to(DEV), kd, vd, table.to(DEV), lens.to(DEV), cu.to(DEV), alphas[1], alphas[2])
    kw = dict(alpha_q=alphas[0], cos_sin=None if cos_sin is None else cos_sin.to(DEV), neighbours=neighbours)
    got = _paged().paged_kv_append_s8(*args, query=q.to(DEV), **kw)
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(got.cpu(), want[2])
    out = torch.full((rows, hq, d), 9, dtype=torch.int8, device=DEV)
    assert _paged().paged_kv_append_s8(*args, query=q.to(DEV), query_out=out, **kw) is out
    assert torch.equal(out[: int(cu[-1])].cpu(), want[2][: int(cu[-1])]) and (out[int(cu[-1]):] == 9).all()
    assert _paged().paged_kv_append_s8(*args, **kw) is None
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])


def test_append_out_of_range_writes_nothing_else():
    g = torch.Generator().manual_seed(23)
    cu, lens, table, pages, rows = _batch(g, [40, 20, 90], [4, 5, 3], 16)
    k, v = _s8(g, pages, 2, 16, 64), _s8(g, pages, 2, 16, 64)
    kn, vn, q = (torch.randn(rows, 2, 64, generator=g) for _ in range(3))
    angle = torch.arange(89, dtype=torch.float64)[:, None] * torch.ones(16)      # the third sequence's last token is beyond it
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    table[0, 2], table[1, 1] = -1, pages
    for bad_lens, bad_cu in (([40, 20, 90], [0, 4, 9, 12]), ([10 ** 9, -7, 2], [0, 4, 9, 12]), ([40, 20, 90], [0, 4, 9, 10 ** 9]),
                             ([40, 20, 90], [-3, 4, 2, 12])):
        bl, bc = torch.tensor(bad_lens, dtype=torch.int32), torch.tensor(bad_cu, dtype=torch.int32)
        print("append out of range", bad_lens, bad_cu, flush=True)
        want = orc.append(kn, vn, k, v, table, bl, bc, 30.0, 30.0, q, 30.0, cos_sin)
        kd, vd = k.to(DEV), v.to(DEV)
        got = _paged().paged_kv_append_s8(kn.to(DEV), vn.to(DEV), kd, vd, table.to(DEV), bl.to(DEV), bc.to(DEV), 30.0, 30.0,
                                          query=q.to(DEV), alpha_q=30.0, cos_sin=cos_sin.to(DEV))
        if bad_cu == sorted(bad_cu):
            assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(got.cpu(), want[2])


# ---------------------------------------------------------------- the two together, streams and graphs
def _angles(n, rot):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(rot // 2).double() / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


class _Server:
    """Sequences that grow: a prompt in chunks, then token by token, beside the same in fp64."""

    def __init__(self, seqs, per, page, hq, hk, d, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.hq, self.hk, self.d, self.page = hq, hk, d, page
        self.table = torch.randperm(seqs * per, generator=self.g).int().view(seqs, per)
        self.lens = torch.zeros(seqs, dtype=torch.int32)
        self.k = torch.zeros(seqs * per, hk, page, d, dtype=torch.int8)
        self.v = torch.zeros_like(self.k)
        self.kd, self.vd, self.td = self.k.to(DEV), self.v.to(DEV), self.table.to(DEV)
        self.cs = _angles(per * page, d)
        self.csd = self.cs.to(DEV)

    def step(self, new):
        rows = sum(new)
        self.lens += torch.tensor(new, dtype=torch.int32)
        cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int()
        q, k, v = (torch.randn(rows, h, self.d, generator=self.g, dtype=torch.float32).half() for h in (self.hq, self.hk, self.hk))
        ld, cd = self.lens.to(DEV), cu.to(DEV)
        qd = _paged().paged_kv_append_s8(k.to(DEV), v.to(DEV), self.kd, self.vd, self.td, ld, cd, 30.0, 30.0, query=q.to(DEV),
                                         alpha_q=30.0, cos_sin=self.csd)
        got = _paged().paged_attn_s8(qd, self.kd, self.vd, self.td, ld, cd, 2.0 / (900 * self.d ** 0.5), 0.03,
                                     out_dtype=torch.float16).cpu()
        self.k, self.v, qs = orc.append(k, v, self.k, self.v, self.table, self.lens, cu, 30.0, 30.0, q, 30.0, self.cs)
        assert torch.equal(qd.cpu(), qs) and torch.equal(self.kd.cpu(), self.k) and torch.equal(self.vd.cpu(), self.v)
        want, size, most = orc.attention(qs, self.k, self.v, self.table, self.lens, cu, 2.0 / (900 * self.d ** 0.5), 0.03)
        worst = orc.attention_error(got, want, size, most, int(self.lens.max()), FP16_WEIGHTS)
        print("step", new, worst, flush=True)
        assert worst <= 1.0


@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 64, 16), (4, 4, 128, 32), (6, 1, 80, 64)])
def test_prompts_in_chunks_then_tokens(hq, hk, d, page):
    s = _Server(3, 256 // page, page, hq, hk, d, hq)
    for new in ([40, 7, 1], [64, 100, 0], [1, 1, 33], [1, 1, 1], [3, 1, 2], [0, 1, 0]):
        s.step(new)


def test_the_same_inputs_give_the_same_bits_on_any_stream():
    g = torch.Generator().manual_seed(31)
    cu, lens, table, pages, rows = _batch(g, [6000, 900, 40], [1, 20, 1], 16)
    k, v = (_s8(g, pages, 2, 16, 128, spread=30).to(DEV) for _ in range(2))
    q = _s8(g, rows, 8, 128, spread=30).to(DEV)
    args = (q, k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), 2e-4, 0.02)
    first = _paged().paged_attn_s8(*args, out_dtype=torch.float16)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_paged().paged_attn_s8(*args, out_dtype=torch.float16))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)


@pytest.mark.parametrize("hq,hk,d,lens,new", [(1, 1, 128, [70000], [1]), (8, 1, 64, [9000, 2, 700], [1, 1, 1]), (4, 2, 80, [3000, 2900], [9, 1]),
                                              (32, 2, 128, [5000, 40, 6001], [1, 1, 2]), (12, 12, 64, [1025], [1]),
                                              (4, 2, 128, [4000, 70], [100, 1]), (1, 1, 64, [3000], [200]), (8, 8, 80, [1500], [33])])
def test_slices_that_meet_in_the_launch_or_behind_it(hq, hk, d, lens, new, monkeypatch):
    # the same bits with the counters, without them (a second launch), again and again, and after calls whose tables hold
    # nonsense: the counters are zero behind every call; against fp64 as well
    P = _paged()
    g = torch.Generator().manual_seed(41 + hq)
    cu, lens, table, pages, rows = _batch(g, lens, new, 16)
    k, v = (_s8(g, pages, hk, 16, d, spread=30).to(DEV) for _ in range(2))
    q = _s8(g, rows, hq, d, spread=30)
    a_qk = 2.0 / (900 * d ** 0.5)
    first = _attend(("meet", hq, hk, d), q, k, v, table, lens, cu, a_qk, 0.02, FP16_WEIGHTS, out_dtype=torch.float16).to(DEV)
    args = (q.to(DEV), k, v, table.to(DEV), lens.to(DEV), cu.to(DEV), a_qk, 0.02)
    assert len(P._counters) > 0
    for i in range(60):
        got = P.paged_attn_s8(*args, out_dtype=torch.float16)
        assert torch.equal(got, first), i
    for bad in ([0] + [rows, 0] * len(lens), [-7, 2 ** 31 - 1] * len(lens)):
        bad_cu = torch.tensor(bad[: len(lens) + 1], dtype=torch.int32, device=DEV)
        P.paged_attn_s8(args[0], k, v, args[3], torch.full_like(args[4], 2 ** 31 - 1), bad_cu, a_qk, 0.02)
        assert all(int(t.abs().max()) == 0 for t in P._counters.values())
        assert torch.equal(P.paged_attn_s8(*args, out_dtype=torch.float16), first)
    monkeypatch.setattr(P, "_arrivals", lambda *a: (None, 0))
    assert torch.equal(P.paged_attn_s8(*args, out_dtype=torch.float16), first)
    monkeypatch.setattr(P._CUDA, "_workspace", lambda *a: (None, 0, 0))     # nothing is cut
    got = P.paged_attn_s8(*args, out_dtype=torch.float16).cpu()
    want, size, most = orc.attention(q, k.cpu(), v.cpu(), table, lens, cu, a_qk, 0.02)
    assert orc.attention_error(got, want, size, most, int(lens.max()), FP16_WEIGHTS) <= 1.0


def test_recorded_steps_read_the_batch_when_they_replay():
    g = torch.Generator().manual_seed(37)
    seqs, per, page, hq, hk, d = 3, 100, 16, 8, 2, 128
    table = torch.randperm(seqs * per, generator=g).int().view(seqs, per).to(DEV)
    cs = _angles(per * page, d).to(DEV)
    lens = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device=DEV)
    rows = 4
    q, k, v = (torch.zeros(rows, h, d, dtype=torch.float16, device=DEV) for h in (hq, hk, hk))
    pools = [_s8(g, seqs * per, hk, page, d, spread=30).to(DEV) for _ in range(2)]

    def step(kc, vc):
        qs = _paged().paged_kv_append_s8(k, v, kc, vc, table, lens, cu, 30.0, 30.0, query=q, alpha_q=30.0, cos_sin=cs)
        return qs, _paged().paged_attn_s8(qs, kc, vc, table, lens, cu, 2e-4, 0.02, out_dtype=torch.float16)

    recorded = []
    for _ in range(2):          # two graphs, each with pools of its own
        kc, vc = pools[0].clone(), pools[1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(kc, vc)
        recorded.append((graph, kc, vc, out))
    for at, new in (([1, 700, 33], [1, 1, 1]), ([1590, 2, 900], [0, 1, 2]), ([5, 6, 1600], [2, 0, 1]), ([3, 1, 1], [1, 1, 1])):
        lens.copy_(torch.tensor(at, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int())
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).half())
        kc, vc = recorded[0][1].clone(), recorded[0][2].clone()
        qs, want = step(kc, vc)
        torch.cuda.synchronize()
        for graph, gk, gv, (gq, gout) in recorded:
            graph.replay()
        torch.cuda.synchronize()
        for graph, gk, gv, (gq, gout) in recorded:
            assert torch.equal(gk, kc) and torch.equal(gv, vc) and torch.equal(gq, qs) and torch.equal(gout, want)
