"""The 4-bit paged cache's operators in fp64 on the CPU, from their formulas, token by token.  Only tests use this."""
import torch

from tests._paged_oracle import rotate, to_s8, tokens

# every step of the format, ascending: fp16 numbers whose low four bits are zero
STEPS = (torch.arange(0x7C00 >> 4, dtype=torch.int32) << 4).to(torch.int16).view(torch.float16).double()
MOST = 57344.0


def f32(a):
    return float(torch.tensor(a, dtype=torch.float32))


def quantise(y, groups):
    """Codes [..., d / 2] and words [..., groups] of fp64 values [..., d] that are numbers of fp32."""
    y = torch.nan_to_num(y, nan=0.0, posinf=MOST, neginf=-MOST).clamp(-MOST, MOST)
    parts = y.unflatten(-1, (groups, -1))
    low, high = parts.amin(-1).clamp(max=0.0), parts.amax(-1).clamp(min=0.0)
    at = torch.searchsorted(15 * STEPS, (high - low).contiguous())      # the first of which 15 are enough
    step = STEPS[at]
    some = torch.where(step > 0, step, 1.0)
    zero = (-low / some).round()
    u = ((parts / some[..., None]).round() + zero[..., None]).clamp(0, 15).flatten(-2).to(torch.uint8)
    half = u.shape[-1] // 2
    return u[..., :half] + 16 * u[..., half:], ((at << 4) + zero.long()).to(torch.int16)


def parts(codes, words):
    """fp64 steps, codes and zeros of every column [..., d] of codes [..., d / 2] and words [..., groups]."""
    step, zero = STEPS[((words.int() & 0x7FF0) >> 4).long().clamp(max=len(STEPS) - 1)], (words & 15).double()
    u = torch.cat([codes % 16, codes // 16], -1).double()
    return step.repeat_interleave(u.shape[-1] // words.shape[-1], -1), u, zero.repeat_interleave(u.shape[-1] // words.shape[-1], -1)


def values(codes, words):
    """fp64 values of codes [..., d / 2] and words [..., groups]."""
    step, u, zero = parts(codes, words)
    return step * (u - zero)


def append(key, value, caches, block_table, context_lens, cu_new, alpha_k=1.0, alpha_v=1.0, query=None, alpha_q=1.0, cos_sin=None,
           neighbours=False, query_dtype=torch.int8):
    """New caches (k, v, k_scale, v_scale), the queries (zeros where nothing is written)."""
    k_cache, v_cache, k_scale, v_scale = (t.clone() for t in caches)
    pages, _, page, _ = k_cache.shape
    groups = k_scale.shape[3]
    q_out = None if query is None else torch.zeros(query.shape, dtype=query_dtype)
    for row, b, p in tokens(cu_new, context_lens, key.shape[0], block_table.shape[1] * page):
        if p < 0 or (cos_sin is not None and p >= cos_sin.shape[0]):
            continue
        turn = (lambda x: x) if cos_sin is None else (lambda x: rotate(x, cos_sin[p], neighbours))  # noqa: B023
        if query is not None:
            y = turn(query[row].double()) * f32(alpha_q)
            q_out[row] = to_s8(y) if query_dtype is torch.int8 else y.float().to(query_dtype)
        at = int(block_table[b, p // page])
        if 0 <= at < pages:
            for y, codes, words in ((turn(key[row].double()) * f32(alpha_k), k_cache, k_scale), (value[row].double() * f32(alpha_v), v_cache, v_scale)):
                codes[at, :, p % page], words[at, :, p % page] = quantise(y.float().double(), groups)
    return (k_cache, v_cache, k_scale, v_scale), q_out


def read(caches, block_table, context_lens, cu, rows, dtype, alpha_k=1.0, alpha_v=1.0):
    k_cache, v_cache, k_scale, v_scale = caches
    pages, heads, page, half = k_cache.shape
    out = [torch.zeros(rows, heads, 2 * half, dtype=dtype) for _ in range(2)]
    for row, b, p in tokens(cu, context_lens, rows, block_table.shape[1] * page):
        at = int(block_table[b, p // page]) if p >= 0 else -1
        if 0 <= at < pages:
            for to, codes, words, alpha in ((out[0], k_cache, k_scale, alpha_k), (out[1], v_cache, v_scale, alpha_v)):
                y = values(codes[at, :, p % page], words[at, :, p % page]) * f32(alpha)
                to[row] = to_s8(y) if dtype is torch.int8 else y.float().to(dtype)
    return out


def attention(query, caches, block_table, context_lens, cu_new, alpha_qk, alpha_pv=1.0, window=0, sinks=0):
    """(context, what `attention_error` needs), fp64, unrounded; zeros where a token sees nothing or a row belongs to nobody."""
    k_cache, v_cache, k_scale, v_scale = caches
    pages, heads, page, half = k_cache.shape
    rows, q_heads, d = query.shape
    group = q_heads // heads
    out = torch.zeros(rows, q_heads, d, dtype=torch.float64)
    size, light = torch.zeros_like(out), torch.zeros_like(out)
    keys = torch.zeros(rows, 1, 1, dtype=torch.float64)
    most, mass = torch.zeros(rows, q_heads, 1, dtype=torch.float64), torch.zeros(rows, q_heads, 1, dtype=torch.float64)
    alpha_qk, alpha_pv = f32(alpha_qk), f32(alpha_pv)
    gathered = {}
    for row, b, p in tokens(cu_new, context_lens, rows, block_table.shape[1] * page):
        if p < 0:
            continue
        if b not in gathered:
            place = torch.arange(min(max(int(context_lens[b]), 0), block_table.shape[1] * page))
            at = block_table[b].long()[place // page]
            there = (at >= 0) & (at < pages)
            at = at.clamp(0, pages - 1)
            gathered[b] = (*(parts(codes[at, :, place % page], words[at, :, place % page])
                             for codes, words in ((k_cache, k_scale), (v_cache, v_scale))), there, place)
        k_parts, v_parts, there, place = gathered[b]
        sees = there & (place <= p)
        if window:
            sees &= (p - place < window) | (place < sinks)
        if not bool(sees.any()):
            continue
        (ks, ku, kz), (vs, vu, vz) = ((x[sees].repeat_interleave(group, 1) for x in y) for y in (k_parts, v_parts))
        k, v = ks * (ku - kz), vs * (vu - vz)
        terms = k * query[row].double()
        s = alpha_qk * terms.sum(-1)  # [positions, q_heads]
        w = torch.softmax(s, 0)
        out[row] = alpha_pv * (w[:, :, None] * v).sum(0)
        size[row] = abs(alpha_pv) * (w[:, :, None] * v.abs()).sum(0)
        light[row] = abs(alpha_pv) * ((vu - vz).abs() * vs.amax((0, 2))[:, None]).sum(0)
        most[row] = 1.4427 * s.abs().amax(0)[:, None]
        mass[row] = 1.4427 * alpha_qk * d * terms.abs().sum(-1).amax(0)[:, None]
        keys[row] = s.shape[0]
    return out, (size, light, most, mass, keys)


def attention_error(got, want, about, weight_error):
    """Largest error over the bound that the arithmetic allows, which a right kernel keeps at 1 or below.

    `about`: the sum of weight times |value|; of |value| where every step were the row's largest; the largest |score| of
    a row in powers of two; head_dim times the largest sum of |q k|, in powers of two as well; the number of keys.

    A weight 2^(x c + m): x is a sum of head_dim products, exact ones, in fp32, off by head_dim 2^-24 of the sum of their sizes; c =
    fp32(alpha log2 e) and the multiply-add are off by 2^-24 of the exponent each, and m has one too, so 2^-22 of it; both times
    ln 2; the hardware's 2^x by 2^-22 more.  The
    weight, or its product with the value's step, is stored with a relative error of ``weight_error``, or, where it is less than
    2^-14, in multiples of 2^-24: off by 2^-25, where the row's largest weight, times the next power of two to the largest step, counts
    2^7 at least.  So a key's part is off by 2^-32 of its value in units of its step, times twice the largest step, in shares of the
    largest weight, which is no more than the denominator.  Weights in numerator and denominator are off alike, so the context is
    by twice these shares.  Sums of `keys` terms in fp32 add at most their number times 2^-24, rescalings and the final quotient
    2^-20.  Then one rounding: half a step."""
    size, light, most, terms, keys = about
    share = 2 * ((most * 2.0 ** -22 + terms * 2.0 ** -24) * 0.7 + 2.0 ** -22 + weight_error) + keys * 2.0 ** -24 + 2.0 ** -20
    off_by = share * size + 2.0 ** -30 * (light + keys * size)
    if got.dtype is torch.int8:
        bound = 0.5 + off_by
        want = want.clamp(-128, 127)
    else:
        tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0
        bound = (torch.finfo(got.dtype).eps / 2) * want.abs() * (1 + 1e-3) + off_by + tiny
    off = (got.double() - want).abs()
    return float(torch.where(off == 0, 0.0, off / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
