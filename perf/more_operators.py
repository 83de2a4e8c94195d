"""The paged KV cache in 4 bits as cases that can be timed and compared: appending to it, attending over it, reading it back.

Three operators, each through ``torch_int.functional.paged_s4``:

* ``append``: ``paged_kv_append_s4``, which rotates the new tokens' keys by their positions, finds a step and a zero for each
  group of a head's values, and writes codes of 4 bits into the pages; queries are rotated (and quantised to int8) beside them.
* ``attention``: ``paged_attn_s4``, the causal attention of every sequence's new tokens over its pages, all of them or a window
  of the last ones and a few first ones.
* ``read``: ``paged_kv_read_s4``, the values of a sequence's last positions as rows of keys and values.

A batch is ``cu_new``, ``context_lens`` and ``block_table``, as for the INT8 cache; the pages of a sequence lie anywhere in the
pool.  Byte j of a row holds the code of dimension j (low four bits) and of dimension head_dim / 2 + j; each group (the whole
head, or its halves) has a 16-bit word, a step with the bits 4 to 14 of an fp16 number and a zero z in the low four:
value = step * (code - z).
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}
# query heads, key/value heads, head size: the widths of the OPT models this package serves, and shared heads
HEADS = [(12, 12, 64), (32, 32, 64), (32, 32, 80), (32, 32, 128), (40, 40, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128),
         (16, 1, 128), (20, 4, 96), (24, 8, 64)]
POSITIONS = 16384  # rows of the table of angles

_calls = {}


def _paged():
    if not _calls:
        sys.path.insert(0, os.path.join(os.getcwd(), "torch-int_amd"))
        from torch_int.functional import paged_s4
        _calls["paged"] = paged_s4
    return _calls["paged"]


def listed():
    return [
        # A chat turn on the smallest model, int8 all the way: one token, where latency counts.
        {"name": "decode_1x600_12h64", "op": "attention", "heads": 12, "kv_heads": 12, "dim": 64, "groups": 1, "page": 16, "seqs": 1,
         "low": 600, "high": 600, "new": 1, "chunks": 1, "pad": 0, "query": "int8", "out": "int8", "window": 0, "sinks": 0},
        # A served batch where every head has its own keys, one step for each head.
        {"name": "decode_28x1500_40h128", "op": "attention", "heads": 40, "kv_heads": 40, "dim": 128, "groups": 1, "page": 16, "seqs": 28,
         "low": 301, "high": 1507, "new": 1, "chunks": 0, "pad": 0, "query": "fp16", "out": "fp16", "window": 0, "sinks": 0},
        # Many users, four query heads to a key head, long chats of very different lengths, a graph's spare rows behind.
        {"name": "decode_75x7000_32h8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 2, "page": 32, "seqs": 75,
         "low": 50, "high": 7003, "new": 1, "chunks": 0, "pad": 5, "query": "bf16", "out": "bf16", "window": 0, "sinks": 0},
        # One user with a long document: one sequence, a long axis.
        {"name": "decode_1x200k_64h8", "op": "attention", "heads": 64, "kv_heads": 8, "dim": 128, "groups": 2, "page": 64, "seqs": 1,
         "low": 200011, "high": 200011, "new": 1, "chunks": 0, "pad": 0, "query": "int8", "out": "fp16", "window": 0, "sinks": 0},
        # Long chats of a model that keeps a window and its first tokens; four drafted tokens to a sequence, head size 80.
        {"name": "window_20x4_32h80", "op": "attention", "heads": 32, "kv_heads": 32, "dim": 80, "groups": 2, "page": 16, "seqs": 20,
         "low": 900, "high": 9001, "new": 4, "chunks": 20, "pad": 0, "query": "bf16", "out": "bf16", "window": 1024, "sinks": 4},
        # Three whole prompts of ragged lengths.
        {"name": "prefill_3x700_40h128", "op": "attention", "heads": 40, "kv_heads": 40, "dim": 128, "groups": 1, "page": 64, "seqs": 3,
         "low": 700, "high": 700, "new": 700, "chunks": 3, "pad": 0, "query": "fp16", "out": "fp16", "window": 0, "sinks": 0},
        # A chunk of 1536 tokens at the end of a document, beside users who decode.
        {"name": "chunk_1536_of_12k_32h8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 2, "page": 128, "seqs": 9,
         "low": 700, "high": 12013, "new": 1536, "chunks": 1, "pad": 0, "query": "bf16", "out": "bf16", "window": 0, "sinks": 0},
        # One token of the smallest model: already int8, learned positions, so nothing is rotated.
        {"name": "append_1_12h64", "op": "append", "heads": 12, "kv_heads": 12, "dim": 64, "groups": 1, "page": 16, "seqs": 1,
         "low": 600, "high": 600, "new": 1, "chunks": 1, "pad": 0, "type": "int8", "query": "none", "rot": 0, "neighbours": False},
        # One token of each of 75 users.
        {"name": "append_75_32h8", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 2, "page": 32, "seqs": 75, "low": 50,
         "high": 1003, "new": 1, "chunks": 0, "pad": 5, "type": "bf16", "query": "bf16", "rot": 128, "neighbours": False},
        # A long prompt's chunk, queries to int8.
        {"name": "append_7001_32h8", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 2, "page": 128, "seqs": 1,
         "low": 8011, "high": 8011, "new": 7001, "chunks": 1, "pad": 0, "type": "fp16", "query": "int8", "rot": 128, "neighbours": False},
        # A short sequence that moves to a worker with a cache of another kind.
        {"name": "read_1x250_12h64", "op": "read", "heads": 12, "kv_heads": 12, "dim": 64, "groups": 1, "page": 16, "seqs": 1, "low": 250,
         "high": 250, "new": 250, "chunks": 1, "pad": 0, "out": "int8"},
        # Prefixes that many prompts share, read for an attention of the caller's own.
        {"name": "read_6x5000_32h8", "op": "read", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 2, "page": 64, "seqs": 6, "low": 5003,
         "high": 6100, "new": 5003, "chunks": 6, "pad": 0, "out": "bf16"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_attention(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    kind = rng.choice(["decode", "decode", "few", "mixed", "chunk"])
    new = {"decode": 1, "few": _log_int(rng, 2, 16), "mixed": _log_int(rng, 17, 700), "chunk": _log_int(rng, 17, 1536)}[kind]
    seqs = _log_int(rng, 2 if kind == "mixed" else 1, {"decode": 80, "few": 32, "mixed": 32, "chunk": 6}[kind])
    high = _log_int(rng, max(new, 16), 200000 if kind == "decode" else 13000)
    low = max(min(new, high), int(high * rng.uniform(0.2, 1.0)))
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    query = rng.choice(["int8", "fp16", "bf16"])
    return {"op": "attention", "heads": heads, "kv_heads": kv_heads, "dim": dim, "groups": rng.choice([1, 2]),
            "page": rng.choice([16, 32, 64, 128]), "seqs": seqs, "low": low, "high": high, "new": new,
            "chunks": 1 if kind == "mixed" else 0 if kind == "decode" else seqs, "pad": rng.choice([0, 0, rng.randrange(1, 9)]),
            "query": query, "out": rng.choice(["int8", "fp16", "bf16"] if kind in ("decode", "few") else ["fp16", "bf16"]),
            "window": window, "sinks": rng.choice([0, 4, rng.randrange(1, 70)]) if window else 0}


def _draw_append(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    new = rng.choice([1, _log_int(rng, 1, 7000)])
    seqs = _log_int(rng, 1, 80 if new == 1 else max(2, 7000 // new) if new < 3500 else 1)
    high = new + _log_int(rng, 1, 2000)
    kind = rng.choice(["fp32", "fp16", "bf16", "int8"])
    rot = rng.choice([dim, dim, dim // 32 * 16, 0])
    query = rng.choice(["int8", "fp16", "bf16"]) if rot else "none"
    return {"op": "append", "heads": heads, "kv_heads": kv_heads, "dim": dim, "groups": rng.choice([1, 2]),
            "page": rng.choice([16, 32, 64, 128]), "seqs": seqs, "low": rng.randrange(new, high + 1), "high": high, "new": new,
            "chunks": seqs, "pad": rng.choice([0, 0, rng.randrange(1, 9)]), "type": kind, "query": query, "rot": rot,
            "neighbours": rng.choice([False, True])}


def _draw_read(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    new = _log_int(rng, 1, 6000)
    seqs = _log_int(rng, 1, max(1, min(64, 30000 // new)))
    high = new + rng.choice([0, _log_int(rng, 1, 2000)])
    return {"op": "read", "heads": heads, "kv_heads": kv_heads, "dim": dim, "groups": rng.choice([1, 2]),
            "page": rng.choice([16, 32, 64, 128]), "seqs": seqs, "low": rng.randrange(new, high + 1), "high": high, "new": new,
            "chunks": seqs, "pad": rng.choice([0, 0, rng.randrange(1, 9)]), "out": rng.choice(["fp32", "fp16", "bf16", "int8"])}


def _plain_cells(case):
    """Score cells that the plain form computes: every sequence padded to the longest, every row count too."""
    return case["seqs"] * case["heads"] * case["new"] * case["high"]


def _pool_values(case):
    return case["seqs"] * case["high"] * case["kv_heads"] * case["dim"]


def draw(rng):
    big = {c["name"]: c for c in listed()}
    kind = rng.choice(["attention", "attention", "attention", "append", "read"])
    if kind == "attention":
        most_bytes = work(big["decode_75x7000_32h8"])["bytes"]
        most_flops = work(big["chunk_1536_of_12k_32h8"])["flops"]
        while True:
            case = _draw_attention(rng)
            w = work(case)
            # neither the kernels nor the plain form (which pads) has more to do than in the largest listed case
            if w["bytes"] <= most_bytes and w["flops"] <= most_flops and _plain_cells(case) <= 9 * 32 * 1536 * 12013 and \
                    _pool_values(case) < 2 ** 29:
                return case
    make, name = {"append": (_draw_append, "append_7001_32h8"), "read": (_draw_read, "read_6x5000_32h8")}[kind]
    most = work(big[name])["bytes"]
    while True:
        case = make(rng)
        if work(case)["bytes"] <= most and _pool_values(case) < 2 ** 28:
            return case


def _lengths(case):
    """Context lengths and new tokens of the sequences, the same for every seed but for their order: spread from `low` to
    `high`, both of them among the lengths."""
    n, low, high = case["seqs"], case["low"], case["high"]
    lens = [high if i == 0 else low if i == 1 else low + int((high - low) * ((i * 0.6180339887) % 1.0)) for i in range(n)]
    new = [case["new"] if i < case["chunks"] else 1 for i in range(n)]
    return lens, new


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _codes(g, *shape):
    """Bytes of two codes each, of normally distributed values whose 16 steps span some 5.5 standard deviations."""
    at = (torch.arange(256, dtype=torch.float64, device=DEV) + 0.5) / 256
    quantile = (math.sqrt(2) * torch.erfinv(2 * at - 1) * 2.7 + 7.5).round().clamp(0, 15).long()
    table = (quantile[:, None] * 16 + quantile[None, :]).flatten().to(torch.uint8)
    out = torch.empty(shape, dtype=torch.uint8, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        part = flat[i:i + (1 << 26)]
        part.copy_(table[torch.randint(0, 65536, part.shape, device=DEV, generator=g)])
    return out


def _words(g, *shape):
    """Steps around 0.36 (values of standard deviation 1), zeros near the middle."""
    s = (torch.randn(*shape, device=DEV, generator=g) * 0.15).exp_().mul_(0.36).half()
    z = torch.randint(6, 10, shape, device=DEV, generator=g).to(torch.int16)
    return (s.view(torch.int16) & 0x7FF0) | z


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = torch.Generator().manual_seed(seed)
    lens, new = _lengths(case)
    order = torch.randperm(len(lens), generator=c).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    page, hq, hk, d, groups = case["page"], case["heads"], case["kv_heads"], case["dim"], case["groups"]
    per = -(-max(lens) // page)
    need = [-(-x // page) for x in lens]
    pages = sum(need) + 3
    at = torch.randperm(pages, generator=c)
    table = torch.zeros(len(lens), per, dtype=torch.int32)
    k = 0
    for b, n in enumerate(need):
        table[b, :n] = at[k:k + n].int()
        k += n
    tokens = sum(new) + case["pad"]
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    state = {"case": case, "table": table.to(DEV), "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
             "cu": torch.tensor(cu, dtype=torch.int32, device=DEV), "max_new": max(new), "rows": tokens,
             "k_cache": _codes(g, pages, hk, page, d // 2), "v_cache": _codes(g, pages, hk, page, d // 2),
             "k_scale": _words(g, pages, hk, page, groups), "v_scale": _words(g, pages, hk, page, groups)}

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def s8(*shape):  # a tensor quantised by its largest magnitude has a standard deviation of some 30 steps
        return normal(*shape).mul_(30).round_().clamp_(-127, 127).to(torch.int8)

    if case["op"] == "attention":
        kind = case["query"]
        state["query"] = s8(tokens, hq, d) if kind == "int8" else normal(tokens, hq, d).to(DTYPES[kind])
        # scores with a standard deviation of 2; a context of some 30 steps where it is int8
        state["alpha_qk"] = _f32(2.0 / ((30.0 if kind == "int8" else 1.0) * math.sqrt(d)))
        state["alpha_pv"] = _f32(100.0 if case["out"] == "int8" else 1.0)
        state["step"] = torch.full((1,), 0.0078125, dtype=torch.float16, device=DEV)
    elif case["op"] == "read":
        state["alphas"] = (_f32(31.0), _f32(29.0)) if case["out"] == "int8" else (1.0, 1.0)
    else:
        kind = DTYPES[case["type"]]
        if kind is torch.int8:
            state["query"], state["key"], state["value"] = s8(tokens, hq, d), s8(tokens, hk, d), s8(tokens, hk, d)
            state["alphas"] = (_f32(0.9), _f32(0.031), _f32(0.029))
        else:
            # keys have channels of several times the others' magnitude
            channel = torch.where(torch.arange(d, device=DEV) % 29 == 5, 4.0, 1.0)
            state["query"], state["key"], state["value"] = ((normal(tokens, h, d) * m).to(kind)
                                                            for h, m in ((hq, 1.0), (hk, channel), (hk, 1.0)))
            state["alphas"] = (_f32(31.0) if case["query"] == "int8" else 1.0, 1.0, 1.0)
        if case["query"] == "none":
            state["query"] = None
        state["cos_sin"] = None
        if case["rot"]:
            half = case["rot"] // 2
            angle = (torch.arange(POSITIONS, dtype=torch.float64, device=DEV)[:, None]
                     * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half))
            state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return state


# ---------------------------------------------------------------- plain forms
def _sequence_of(state):
    """For each row its sequence (clamped), its place among the sequence's new tokens, and whether it belongs to one."""
    row = torch.arange(state["rows"], device=DEV)
    seq = torch.searchsorted(state["cu"][1:].long(), row, right=True)
    real = seq < state["lens"].numel()
    seq = seq.clamp(max=state["lens"].numel() - 1)
    return seq, row - state["cu"].long()[seq], real


def _places(state):
    """Page and offset of every row that belongs to a sequence, and its position."""
    case, cu, lens = state["case"], state["cu"].long(), state["lens"].long()
    seq, at, real = _sequence_of(state)
    position = ((lens - (cu[1:] - cu[:-1]))[seq] + at).masked_fill(~real, 0)
    n = state["rows"] - case["pad"]  # rows behind the last sequence go nowhere
    return state["table"].long()[seq, position // case["page"]][:n], (position % case["page"])[:n], position, real


def _values(codes, words):
    """fp32 values of rows of codes [..., d / 2] and their words [..., groups]."""
    step = (words & 0x7FF0).view(torch.float16).float()
    zero = (words & 15).float()
    u = torch.cat([codes & 15, codes >> 4], -1).float()
    u = u.view(*words.shape, u.shape[-1] // words.shape[-1])
    return ((u - zero[..., None]) * step[..., None]).flatten(-2)


def _attention_plain(s):
    case, cu, lens = s["case"], s["cu"].long(), s["lens"].long()
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    group, tokens, B = case["heads"] // hk, s["rows"], lens.numel()
    span = s["table"].shape[1] * page
    pages = s["table"].long()
    k, v = (_values(codes[pages], words[pages]).transpose(1, 2).reshape(B, hk, span, d)
            for codes, words in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
    new, most = cu[1:] - cu[:-1], s["max_new"]
    i = torch.arange(most, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=tokens - 1)
    q = s["query"][rows].view(B, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B, hk, group * most, d).float()
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["alpha_qk"]).view(B, hk, group, most, span)
    last = (lens[:, None] - new[:, None] + i)[:, :, None]
    place = torch.arange(span, device=DEV)
    hidden = place > last
    if case["window"]:
        hidden |= (place <= last - case["window"]) & (place >= case["sinks"])
    x.masked_fill_(hidden[:, None, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(B, hk, group * most, span), v).view(B, hk, group, most, d).div_(total).mul_(s["alpha_pv"])
    y = y.permute(0, 3, 1, 2, 4).reshape(B, most, hk * group, d)
    seq, at, real = _sequence_of(s)
    out = y[seq, at.clamp(0, most - 1)].masked_fill_(~real[:, None, None], 0.0)
    if case["out"] == "int8":
        return out.round().clamp(-128, 127).to(torch.int8) * s["step"]
    return out.to(DTYPES[case["out"]])


def _rotate_plain(x, cos_sin, rot, neighbours):
    half = rot // 2
    c, t = cos_sin[:, None, :half], cos_sin[:, None, half:]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if neighbours else (x[..., :half], x[..., half:rot])
    p, q = a * c - b * t, b * c + a * t
    turned = torch.stack([p, q], -1).flatten(-2) if neighbours else torch.cat([p, q], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _quantise_plain(x, alpha, groups):
    """Codes and words of [rows, heads, d] in 64 bits (next to a border between two codes): the step is the smallest of its format
    of which 15 span the group's values and 0."""
    y = (x * alpha).float().nan_to_num(0.0, float("inf"), float("-inf")).clamp(-57344, 57344).double()
    y = y.view(*y.shape[:2], groups, y.shape[2] // groups)
    low, high = y.amin(-1).clamp(max=0), y.amax(-1).clamp(min=0)
    span = high - low
    bits = (((span / 15).half().view(torch.int16) & 0x7FF0) - 16).clamp(min=0)
    for _ in range(3):
        bits = torch.where(15 * bits.view(torch.float16).double() < span, bits + 16, bits)
    step = bits.view(torch.float16).double()
    some = step > 0
    by = torch.where(some, step, 1.0)
    zero = torch.where(some, -low / by, 0.0).round()
    u = ((y / by[..., None]).round() + zero[..., None]).clamp(0, 15).flatten(2).to(torch.uint8)
    half = u.shape[2] // 2
    return u[..., :half] | (u[..., half:] << 4), bits | zero.to(torch.int16)


def _append_plain(s):
    case, groups = s["case"], s["case"]["groups"]
    pages, offset, position, real = _places(s)
    n = pages.numel()
    k, v, q = s["key"].double(), s["value"].double(), None if s["query"] is None else s["query"].double()
    if case["rot"]:
        turn = s["cos_sin"][position].double()
        k = _rotate_plain(k, turn, case["rot"], case["neighbours"])
        q = None if q is None else _rotate_plain(q, turn, case["rot"], case["neighbours"])
    aq, ak, av = s["alphas"]
    out = []
    for x, alpha, codes, words in ((k, ak, s["k_cache"], s["k_scale"]), (v, av, s["v_cache"], s["v_scale"])):
        new_codes, new_words = _quantise_plain(x[:n], alpha, groups)
        codes.transpose(1, 2)[pages, offset] = new_codes
        words.transpose(1, 2)[pages, offset] = new_words
        out += [codes, words]
    if q is not None:
        q = (q * aq).masked_fill_(~real[:, None, None], 0.0)
        out.append(q.round().clamp(-128, 127).to(torch.int8) if case["query"] == "int8" else q.float().to(DTYPES[case["query"]]))
    return out


def _read_plain(s):
    case = s["case"]
    pages, offset, _, _ = _places(s)
    out = []
    for codes, words, alpha in ((s["k_cache"], s["k_scale"], s["alphas"][0]), (s["v_cache"], s["v_scale"], s["alphas"][1])):
        y = _values(codes.transpose(1, 2)[pages, offset], words.transpose(1, 2)[pages, offset])
        if case["out"] == "int8":  # in 64 bits next to a border
            y = (y.double() * alpha).round().clamp(-128, 127)
        z = torch.zeros(s["rows"], *y.shape[1:], dtype=DTYPES[case["out"]], device=DEV)
        z[:y.shape[0]] = y.to(z.dtype)
        out.append(z)
    return out


def run(state):
    case = state["case"]
    if not own:
        return {"attention": _attention_plain, "append": _append_plain, "read": _read_plain}[case["op"]](state)
    pools = (state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])
    batch = (state["table"], state["lens"], state["cu"])
    if case["op"] == "attention":
        out = _paged().paged_attn_s4(state["query"], *pools, *batch, state["alpha_qk"], state["alpha_pv"], window=case["window"],
                                     sinks=case["sinks"], out_dtype=DTYPES[case["out"]])
        return out * state["step"] if case["out"] == "int8" else out
    if case["op"] == "read":
        return list(_paged().paged_kv_read_s4(*pools, *batch, state["rows"], out_dtype=DTYPES[case["out"]], alpha_k=state["alphas"][0],
                                              alpha_v=state["alphas"][1]))
    aq, ak, av = state["alphas"]
    q = _paged().paged_kv_append_s4(state["key"], state["value"], *pools, *batch, ak, av, query=state["query"], alpha_q=aq,
                                    cos_sin=state["cos_sin"], neighbours=case["neighbours"],
                                    query_dtype=DTYPES.get(case["query"], torch.int8))
    # the caches as they are, bit for bit: codes and words that differ would stand for other values
    return [pools[0], pools[2], pools[1], pools[3]] + ([] if q is None else [q])


def _seen(length, new, window, sinks):
    """Pairs of a new token and a position it sees, and positions that any of them sees."""
    pairs = 0
    first = length - new
    if not window:
        return new * first + new * (new + 1) // 2, length
    for p in range(first, length):
        begin = max(0, p - window + 1)
        pairs += p + 1 - begin + min(sinks, begin)
    begin = max(0, first - window + 1)
    return pairs, length - begin + min(sinks, begin)


def work(case):
    lens, new = _lengths(case)
    hq, hk, d, n = case["heads"], case["kv_heads"], case["dim"], sum(new)
    row = d // 2 + 2 * case["groups"]  # bytes of a position of one head, of the keys or of the values
    tables = 4 * (2 * case["seqs"] + 1)
    if case["op"] == "attention":
        seen = [_seen(x, t, case["window"], case["sinks"]) for x, t in zip(lens, new)]
        held = sum(x for _, x in seen)
        return {"bytes": 2 * held * hk * row + n * hq * d * (SIZES[case["query"]] + SIZES[case["out"]]) + tables + 4 * held // case["page"],
                "flops": 4 * sum(p for p, _ in seen) * hq * d}
    if case["op"] == "read":
        return {"bytes": 2 * n * hk * (row + d * SIZES[case["out"]]) + tables + 4 * n // case["page"], "flops": 4 * n * hk * d}
    queries = 0 if case["query"] == "none" else n * hq * d
    size = SIZES[case["type"]]
    return {"bytes": n * 2 * hk * (d * size + row) + queries * (size + SIZES.get(case["query"], 0)) + 4 * n * case["rot"] + tables + 4 * n,
            "flops": 10 * n * 2 * hk * d + 6 * queries}


# ---------------------------------------------------------------- the definition in 64 bits
def _decode(codes, words, d):
    """fp64 values of codes [n, d / 2] and words [n, groups] of one head."""
    groups = words.shape[1]
    out = torch.empty(codes.shape[0], d, dtype=torch.float64, device=DEV)
    for j in range(groups):
        w = words[:, j].int()
        e, m, z = (w >> 10) & 31, (w >> 4) & 63, (w & 15).double()
        step = torch.where(e == 0, torch.ldexp(m.double(), torch.tensor(-20, device=DEV)), torch.ldexp((64 + m).double(), e - 21))
        dims = torch.arange(j * d // groups, (j + 1) * d // groups, device=DEV)
        byte = codes[:, dims % (d // 2)].int()
        out[:, dims] = step[:, None] * (torch.where(dims >= d // 2, byte // 16, byte % 16).double() - z[:, None])
    return out


def _exact_attention(case, s):
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["rows"], hq, d, dtype=torch.float64, device=DEV)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b in range(len(lens)):
        t, n = cu[b + 1] - cu[b], lens[b]
        places = torch.arange(n, device=DEV)
        pages, at = s["table"][b].long()[places // page], places % page
        behind = places[None, :] - torch.arange(n - t, n, device=DEV)[:, None]  # of each new token
        seen = behind <= 0
        if case["window"]:
            seen &= (behind > -case["window"]) | (places < case["sinks"])
        for h in range(hk):
            k = _decode(s["k_cache"][pages, h, at], s["k_scale"][pages, h, at], d)
            v = _decode(s["v_cache"][pages, h, at], s["v_scale"][pages, h, at], d)
            for head in range(h * (hq // hk), (h + 1) * (hq // hk)):
                score = float(s["alpha_qk"]) * (s["query"][cu[b]:cu[b + 1], head].double() @ k.T)
                w = torch.softmax(torch.where(seen, score, float("-inf")), 1)
                out[cu[b]:cu[b + 1], head] = float(s["alpha_pv"]) * (w @ v)
    if case["out"] == "int8":
        return out.round().clamp(-128, 127) * float(s["step"])
    return out


def _turned(x, position, s, case):
    y, rot = x.double(), case["rot"]
    if rot:
        first = torch.arange(0, rot, 2) if case["neighbours"] else torch.arange(rot // 2)
        second = first + 1 if case["neighbours"] else first + rot // 2
        e = s["cos_sin"][position].double()
        cos, sin = e[:, None, : rot // 2], e[:, None, rot // 2:]
        a, b = y[..., first], y[..., second]
        y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y


def _exact_append(case, s):
    page, groups, d = case["page"], case["groups"], case["dim"]
    pools = {n: s[n].clone() for n in ("k_cache", "k_scale", "v_cache", "v_scale")}
    cu, lens, alphas = s["cu"].tolist(), s["lens"].tolist(), s["alphas"]
    q_out = None
    if s["query"] is not None:
        q_out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b in range(len(lens)):
        rows = slice(cu[b], cu[b + 1])
        position = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device=DEV)
        pages, offset = s["table"][b].long()[position // page], position % page
        if q_out is not None:
            q_out[rows] = _turned(s["query"][rows], position, s, case) * float(alphas[0])
        for name, y in (("k", _turned(s["key"][rows], position, s, case) * float(alphas[1])),
                        ("v", s["value"][rows].double() * float(alphas[2]))):
            y = y.float().double().clamp(-57344.0, 57344.0)  # the value that is quantised is one of fp32
            codes = torch.zeros(*y.shape[:2], d, dtype=torch.int64, device=DEV)
            words = []
            for j in range(groups):
                part = slice(j * d // groups, (j + 1) * d // groups)
                low = torch.minimum(y[..., part].min(-1).values, torch.zeros((), dtype=torch.float64, device=DEV))
                span = torch.maximum(y[..., part].max(-1).values, torch.zeros((), dtype=torch.float64, device=DEV)) - low
                # steps are n * 2^(e - 6): n from 64 to 127, or fewer at the smallest e
                e = (torch.frexp(span / 15).exponent.long() - 1).clamp(min=-14)
                n = torch.ceil(torch.ldexp(span / 15, 6 - e))
                n = torch.where(15 * torch.ldexp(n, e - 6) < span, n + 1, n)
                step = torch.ldexp(n, e - 6)
                z = torch.where(n > 0, torch.round(-low / step.clamp(min=2.0 ** -20)), 0.0)
                twice = torch.floor(y[..., part] * 2 / step.clamp(min=2.0 ** -20)[..., None])
                tie = twice * step[..., None] == y[..., part] * 2
                up = torch.where(tie & (twice.remainder(4) == 1), (twice - 1) / 2, torch.floor((twice + 1) / 2))
                codes[..., part] = (up + z[..., None]).clamp(0, 15).long()
                words.append(step.half().view(torch.int16) + z.to(torch.int16))
            pools[name + "_cache"][pages, :, offset] = (codes[..., : d // 2] + 16 * codes[..., d // 2:]).to(torch.uint8)
            pools[name + "_scale"][pages, :, offset] = torch.stack(words, -1)
    out = [pools[n] for n in ("k_cache", "k_scale", "v_cache", "v_scale")]
    if q_out is not None:
        out.append(q_out.round().clamp(-128, 127).to(torch.int8) if case["query"] == "int8" else q_out)
    return out


def _exact_read(case, s):
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    out = [torch.zeros(s["rows"], hk, d, dtype=torch.float64, device=DEV) for _ in range(2)]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b in range(len(lens)):
        position = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device=DEV)
        pages, at = s["table"][b].long()[position // page], position % page
        for h in range(hk):
            for i, name in enumerate("kv"):
                y = _decode(s[name + "_cache"][pages, h, at], s[name + "_scale"][pages, h, at], d) * float(s["alphas"][i])
                out[i][cu[b]:cu[b + 1], h] = y.round().clamp(-128, 127) if case["out"] == "int8" else y
    return [y.to(torch.int8) for y in out] if case["out"] == "int8" else out


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "read": _exact_read}[case["op"]](case, s)
