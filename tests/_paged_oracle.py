"""The paged cache's two operators in fp64 on the CPU, from their formulas, token by token.  Only tests use this."""
import torch


def tokens(cu_new, context_lens, rows, capacity):
    """(row, sequence, position) of every new token, with what lies outside cut off: rows at ``rows``, lengths at ``capacity``."""
    cu, lens = cu_new.tolist(), context_lens.tolist()
    for b, n in enumerate(lens):
        lo = min(max(cu[b], 0), rows)
        hi = min(max(cu[b + 1], lo), rows)
        n = min(max(n, 0), capacity)
        for i in range(hi - lo):
            yield lo + i, b, n - (hi - lo) + i


def rotate(x, cos_sin, neighbours):
    rot = cos_sin.shape[0]
    first = torch.arange(0, rot, 2) if neighbours else torch.arange(rot // 2)
    second = first + (1 if neighbours else rot // 2)
    c, s = cos_sin[: rot // 2].double(), cos_sin[rot // 2:].double()
    y = x.clone()
    y[:, first] = x[:, first] * c - x[:, second] * s
    y[:, second] = x[:, second] * c + x[:, first] * s
    return y


def to_s8(y):
    return torch.nan_to_num(y.round().clamp(-128, 127), nan=0.0).to(torch.int8)


def append(key, value, k_cache, v_cache, block_table, context_lens, cu_new, alpha_k, alpha_v, query=None, alpha_q=1.0, cos_sin=None,
           neighbours=False):
    """New caches, the int8 queries (zeros where nothing is written)."""
    k_cache, v_cache = k_cache.clone(), v_cache.clone()
    pages, _, page, _ = k_cache.shape
    f32 = lambda a: float(torch.tensor(a, dtype=torch.float32))  # noqa: E731
    q_out = None if query is None else torch.zeros(query.shape, dtype=torch.int8)
    for row, b, p in tokens(cu_new, context_lens, key.shape[0], block_table.shape[1] * page):
        if p < 0 or (cos_sin is not None and p >= cos_sin.shape[0]):
            continue
        turn = (lambda x: x) if cos_sin is None else (lambda x: rotate(x, cos_sin[p], neighbours))  # noqa: B023
        if query is not None:
            q_out[row] = to_s8(turn(query[row].double()) * f32(alpha_q))
        at = int(block_table[b, p // page])
        if 0 <= at < pages:
            k_cache[at, :, p % page] = to_s8(turn(key[row].double()) * f32(alpha_k))
            v_cache[at, :, p % page] = to_s8(value[row].double() * f32(alpha_v))
    return k_cache, v_cache, q_out


def attention(query, k_cache, v_cache, block_table, context_lens, cu_new, alpha_qk, alpha_pv):
    """(context, sum of weight times |value|, largest |score| of a row in powers of two), fp64, unrounded; zeros where a token
    sees nothing or a row belongs to nobody."""
    pages, heads, page, d = k_cache.shape
    rows, q_heads, _ = query.shape
    group = q_heads // heads
    out = torch.zeros(rows, q_heads, d, dtype=torch.float64)
    size = torch.zeros(rows, q_heads, d, dtype=torch.float64)
    most = torch.zeros(rows, q_heads, 1, dtype=torch.float64)
    alpha_qk, alpha_pv = (float(torch.tensor(a, dtype=torch.float32)) for a in (alpha_qk, alpha_pv))
    gathered = {}
    for row, b, p in tokens(cu_new, context_lens, rows, block_table.shape[1] * page):
        if p < 0:
            continue
        if b not in gathered:
            n = min(max(int(context_lens[b]), 0), block_table.shape[1] * page)
            place = torch.arange(n)
            at = block_table[b].long()[place // page]
            there = (at >= 0) & (at < pages)
            at = at.clamp(0, pages - 1)
            gathered[b] = (k_cache[at, :, place % page].double(), v_cache[at, :, place % page].double(), there)
        k, v, there = gathered[b]
        k, v, there = k[: p + 1], v[: p + 1], there[: p + 1]
        if not bool(there.any()):
            continue
        k, v = k[there].repeat_interleave(group, 1), v[there].repeat_interleave(group, 1)
        s = alpha_qk * (k * query[row].double()).sum(-1)  # [positions, q_heads]
        w = torch.softmax(s, 0)
        out[row] = alpha_pv * (w[:, :, None] * v).sum(0)
        size[row] = abs(alpha_pv) * (w[:, :, None] * v.abs()).sum(0)
        most[row] = s.abs().amax(0)[:, None] * 1.4427
    return out, size, most


def attention_error(got, want, size, most, keys, weight_error):
    """Largest error over the bound that the arithmetic allows, which a right kernel keeps at 1 or below.

    A weight 2^(x c + m): x is an exact integer; c = fp32(alpha log2 e) and its products are off by some 2^-23 of the exponent
    (twice 2^-24: the constant, the multiply-add), of which both m and x have one, so 2^-22 of it times ln 2, and the hardware's
    2^x by 2^-22 more; the weight is stored with a relative error of ``weight_error``.  The same weights are in numerator and
    denominator, so the context is off by twice that share of the sum of weight times |value|; sums of `keys` terms in fp32
    add at most their number times 2^-24, rescalings and the final quotient 2^-20.  Then one rounding: half a step."""
    share = 2 * (most * 2.0 ** -22 * 0.7 + 2.0 ** -22 + weight_error) + keys * 2.0 ** -24 + 2.0 ** -20
    if got.dtype is torch.int8:
        bound = 0.5 + share * size
        want = want.clamp(-128, 127)
    else:
        tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0
        bound = (torch.finfo(got.dtype).eps / 2) * want.abs() * (1 + 1e-3) + share * size + tiny
    off = (got.double() - want).abs()
    return float(torch.where(off == 0, 0.0, off / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
