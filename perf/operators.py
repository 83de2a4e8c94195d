"""The paged INT8 KV cache as cases that can be timed and compared: appending to it and attending over it.

Two operators, each through ``torch_int.functional.paged``:

* ``append``: ``paged_kv_append_s8``, which rotates the new tokens' keys by their positions, quantises keys and values and
  writes them into the pages of their sequences; with a rotation the queries are rotated and quantised in the same call.
* ``attention``: ``paged_attn_s8``, the causal attention of every sequence's new tokens over its pages.

A batch is ``cu_new`` (where each sequence's new tokens begin), ``context_lens`` (cached tokens, the new ones counted) and
``block_table`` (pages of each sequence); the pages of a sequence lie anywhere in the pool.  Rows behind the last sequence
(``pad``) are what a program that records graphs for a few batch sizes has.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
# query heads, key/value heads, head size: the widths of the OPT models this package serves, and shared heads
HEADS = [(12, 12, 64), (32, 32, 64), (32, 32, 80), (32, 32, 128), (40, 40, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128),
         (16, 1, 128), (24, 8, 64)]
POSITIONS = 16384  # rows of the table of angles

_calls = {}


def _paged():
    if not _calls:
        sys.path.insert(0, os.path.join(os.getcwd(), "torch-int_amd"))
        from torch_int.functional import paged
        _calls["paged"] = paged
    return _calls["paged"]


def listed():
    return [
        # A chat turn on the smallest model: one token, where latency counts.
        {"name": "decode_1x500_12h64", "op": "attention", "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "seqs": 1,
         "low": 500, "high": 500, "new": 1, "chunks": 1, "pad": 0, "out": "fp16"},
        # A served batch of users of a model whose next layer is int8: every head has its own keys.
        {"name": "decode_24x1000_32h128", "op": "attention", "heads": 32, "kv_heads": 32, "dim": 128, "page": 16, "seqs": 24,
         "low": 251, "high": 1003, "new": 1, "chunks": 0, "pad": 0, "out": "int8"},
        # Many users, four query heads to a key head, long chats of very different lengths, a graph's spare rows behind.
        {"name": "decode_61x4000_32h8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 61,
         "low": 40, "high": 4001, "new": 1, "chunks": 0, "pad": 3, "out": "bf16"},
        # Two users with long documents: few sequences, a long axis.
        {"name": "decode_2x100k_64h8", "op": "attention", "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "seqs": 2,
         "low": 90007, "high": 100003, "new": 1, "chunks": 0, "pad": 0, "out": "fp16"},
        # Drafted tokens that are checked, five to a sequence, head size 80.
        {"name": "verify_16x5_32h80", "op": "attention", "heads": 32, "kv_heads": 32, "dim": 80, "page": 16, "seqs": 16,
         "low": 333, "high": 1501, "new": 5, "chunks": 16, "pad": 0, "out": "bf16"},
        # A prompt's chunk of 512 tokens that rides along with 31 users who decode.
        {"name": "mixed_512_31_32h8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "seqs": 32,
         "low": 600, "high": 2007, "new": 512, "chunks": 1, "pad": 0, "out": "bf16"},
        # Four whole prompts at once.
        {"name": "prefill_4x512_40h128", "op": "attention", "heads": 40, "kv_heads": 40, "dim": 128, "page": 64, "seqs": 4,
         "low": 512, "high": 512, "new": 512, "chunks": 4, "pad": 0, "out": "fp16"},
        # A chunk of 2048 tokens at the end of a document.
        {"name": "chunk_2048_of_16k_32h8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "seqs": 1,
         "low": 16229, "high": 16229, "new": 2048, "chunks": 1, "pad": 0, "out": "bf16"},
        # One token of the smallest model: already int8, learned positions, so nothing is rotated.
        {"name": "append_1_12h64", "op": "append", "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "seqs": 1, "low": 500,
         "high": 500, "new": 1, "chunks": 1, "pad": 0, "type": "int8", "rot": 0, "neighbours": False},
        # One token of each of 61 users.
        {"name": "append_61_32h8", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "seqs": 61, "low": 40,
         "high": 999, "new": 1, "chunks": 0, "pad": 3, "type": "bf16", "rot": 128, "neighbours": False},
        # A batch of ragged prompts of an fp32 stream, a quarter of the head rotated, pairs of neighbours.
        {"name": "append_4x509_32h128", "op": "append", "heads": 32, "kv_heads": 32, "dim": 128, "page": 16, "seqs": 4,
         "low": 509, "high": 640, "new": 509, "chunks": 4, "pad": 0, "type": "fp32", "rot": 32, "neighbours": True},
        # A long prompt's chunk.
        {"name": "append_8192_32h8", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "seqs": 1, "low": 9001,
         "high": 9001, "new": 8192, "chunks": 1, "pad": 0, "type": "fp16", "rot": 128, "neighbours": False},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_attention(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    kind = rng.choice(["decode", "decode", "few", "mixed", "chunk"])
    new = {"decode": 1, "few": _log_int(rng, 2, 16), "mixed": _log_int(rng, 17, 700), "chunk": _log_int(rng, 17, 2048)}[kind]
    seqs = _log_int(rng, 2 if kind == "mixed" else 1, {"decode": 64, "few": 32, "mixed": 32, "chunk": 6}[kind])
    high = _log_int(rng, max(new, 16), 100000 if kind == "decode" else 16000)
    low = max(min(new, high), int(high * rng.uniform(0.2, 1.0)))
    return {"op": "attention", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
            "seqs": seqs, "low": low, "high": high, "new": new, "chunks": 1 if kind == "mixed" else 0 if kind == "decode" else seqs,
            "pad": rng.choice([0, 0, rng.randrange(1, 9)]), "out": rng.choice(["int8", "fp16", "bf16"] if kind in ("decode", "few")
                                                                             else ["fp16", "bf16"])}


def _draw_append(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    new = rng.choice([1, _log_int(rng, 1, 8192)])
    seqs = _log_int(rng, 1, 64 if new == 1 else max(2, 8192 // new) if new < 4096 else 1)
    high = new + _log_int(rng, 1, 2000)
    kind = rng.choice(["fp32", "fp16", "bf16", "int8"])
    rot = 0 if kind == "int8" else rng.choice([dim, dim, dim // 32 * 16, 0])
    return {"op": "append", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "seqs": seqs,
            "low": rng.randrange(new, high + 1), "high": high, "new": new, "chunks": seqs, "pad": rng.choice([0, 0, rng.randrange(1, 9)]),
            "type": kind, "rot": rot, "neighbours": rng.choice([False, True])}


def _plain_cells(case):
    """Score cells that the plain form computes: every sequence padded to the longest."""
    return case["seqs"] * case["heads"] * case["new"] * case["high"]


def draw(rng):
    if rng.random() < 0.35:
        while True:
            case = _draw_append(rng)
            most = work(next(c for c in listed() if c["name"] == "append_4x509_32h128"))["bytes"]
            if case["seqs"] * case["high"] * case["kv_heads"] * case["dim"] < 2 ** 28 and work(case)["bytes"] <= most:
                return case
    big = {c["name"]: c for c in listed()}
    most_bytes = work(big["decode_2x100k_64h8"])["bytes"]
    most_flops = work(big["chunk_2048_of_16k_32h8"])["flops"]
    while True:
        case = _draw_attention(rng)
        w = work(case)
        # neither the kernels nor the plain form (which pads) has more to do than in the largest listed case
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and _plain_cells(case) <= 32 * 2048 * 16229 and \
                case["seqs"] * case["high"] * case["kv_heads"] * case["dim"] < 2 ** 28:
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


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = torch.Generator().manual_seed(seed)
    lens, new = _lengths(case)
    order = torch.randperm(len(lens), generator=c).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    page, hq, hk, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
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

    def s8(*shape):  # a tensor quantised by its largest magnitude has a standard deviation of some 30 steps
        return torch.randn(*shape, device=DEV, generator=g).mul_(30).round_().clamp_(-127, 127).to(torch.int8)

    state = {"case": case, "table": table.to(DEV), "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
             "cu": torch.tensor(cu, dtype=torch.int32, device=DEV), "max_new": max(new),
             "k_cache": s8(pages, hk, page, d), "v_cache": s8(pages, hk, page, d)}
    if case["op"] == "attention":
        state["query"] = s8(tokens, hq, d)
        # scores with a standard deviation of 2; a context of some 30 steps where it is int8
        state["alpha_qk"] = _f32(2.0 / (900.0 * math.sqrt(d)))
        state["alpha_pv"] = _f32({"int8": 6.0, "fp16": 0.02, "bf16": 0.02}[case["out"]])
        state["step"] = torch.full((1,), 0.0078125, dtype=torch.float16, device=DEV)
        return state
    kind = DTYPES[case["type"]]
    if kind is torch.int8:
        state["query"], state["key"], state["value"] = None, s8(tokens, hk, d), s8(tokens, hk, d)
        state["alphas"] = (1.0, 1.0, 1.0)
    else:
        state["query"], state["key"], state["value"] = (torch.randn(tokens, h, d, device=DEV, generator=g).to(kind)
                                                        for h in (hq, hk, hk))
        state["alphas"] = (_f32(31.0), _f32(29.0), _f32(33.0))
    state["cos_sin"] = None
    if case["rot"]:
        half = case["rot"] // 2
        angle = (torch.arange(POSITIONS, dtype=torch.float64, device=DEV)[:, None]
                 * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half))
        state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    else:
        state["query"] = None
    return state


# ---------------------------------------------------------------- plain forms
def _sequence_of(state, tokens):
    """For each row its sequence (clamped), its place among the sequence's new tokens, and whether it belongs to one."""
    row = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(state["cu"][1:].long(), row, right=True)
    real = seq < state["lens"].numel()
    seq = seq.clamp(max=state["lens"].numel() - 1)
    return seq, row - state["cu"].long()[seq], real


def _attention_plain(s):
    case, cu, lens = s["case"], s["cu"].long(), s["lens"].long()
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    group, tokens, B = case["heads"] // hk, s["query"].shape[0], lens.numel()
    span = s["table"].shape[1] * page
    k = s["k_cache"][s["table"].long()].transpose(1, 2).reshape(B, hk, span, d).float()
    v = s["v_cache"][s["table"].long()].transpose(1, 2).reshape(B, hk, span, d).float()
    new, most = cu[1:] - cu[:-1], s["max_new"]
    i = torch.arange(most, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=tokens - 1)
    q = s["query"][rows].view(B, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B, hk, group * most, d).float()
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["alpha_qk"]).view(B, hk, group, most, span)
    last = lens[:, None] - new[:, None] + i
    x.masked_fill_(torch.arange(span, device=DEV) > last[:, None, None, :, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(B, hk, group * most, span), v).view(B, hk, group, most, d).div_(total).mul_(s["alpha_pv"])
    y = y.permute(0, 3, 1, 2, 4).reshape(B, most, hk * group, d)
    seq, at, real = _sequence_of(s, tokens)
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


def _append_plain(s):
    case = s["case"]
    tokens, page = s["key"].shape[0], case["page"]
    seq, at, real = _sequence_of(s, tokens)
    cu, lens = s["cu"].long(), s["lens"].long()
    position = (lens - (cu[1:] - cu[:-1]))[seq] + at
    position = position.masked_fill(~real, 0)
    k, v, q = s["key"].double(), s["value"].double(), None if s["query"] is None else s["query"].double()  # next to a border
    if case["rot"]:
        turn = s["cos_sin"][position].double()
        k, q = (_rotate_plain(x, turn, case["rot"], case["neighbours"]) for x in (k, q))

    def s8(x, alpha):
        return (x * alpha).round().clamp(-128, 127).to(torch.int8)

    aq, ak, av = s["alphas"]
    n = tokens - case["pad"]  # rows behind the last sequence go nowhere
    pages, offset = s["table"].long()[seq, position // page][:n], (position % page)[:n]
    s["k_cache"].transpose(1, 2)[pages, offset] = s8(k[:n], ak)
    s["v_cache"].transpose(1, 2)[pages, offset] = s8(v[:n], av)
    out = [s["k_cache"], s["v_cache"]]
    if q is not None:
        out.append(s8(q, aq).masked_fill_(~real[:, None, None], 0))
    return out


def run(state):
    case = state["case"]
    if case["op"] == "attention":
        if own:
            out = _paged().paged_attn_s8(state["query"], state["k_cache"], state["v_cache"], state["table"], state["lens"],
                                         state["cu"], state["alpha_qk"], state["alpha_pv"], out_dtype=DTYPES[case["out"]])
            return out * state["step"] if case["out"] == "int8" else out
        return _attention_plain(state)
    if own:
        aq, ak, av = state["alphas"]
        q = _paged().paged_kv_append_s8(state["key"], state["value"], state["k_cache"], state["v_cache"], state["table"],
                                        state["lens"], state["cu"], ak, av, query=state["query"], alpha_q=aq,
                                        cos_sin=state["cos_sin"], neighbours=case["neighbours"])
        return [state["k_cache"], state["v_cache"]] + ([] if q is None else [q])
    return _append_plain(state)


def work(case):
    lens, new = _lengths(case)
    hq, hk, d, n = case["heads"], case["kv_heads"], case["dim"], sum(new)
    tables = 4 * (sum(-(-x // case["page"]) for x in lens) + 2 * case["seqs"] + 1)
    if case["op"] == "attention":
        size = {"int8": 1, "fp16": 2, "bf16": 2}[case["out"]]
        seen = sum(t * (x - t) + t * (t + 1) // 2 for x, t in zip(lens, new))
        return {"bytes": 2 * sum(lens) * hk * d + n * hq * d * (1 + size) + tables, "flops": 4 * seen * hq * d}
    size = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}[case["type"]]
    elements = n * (2 * hk + (hq if case["rot"] else 0)) * d
    tables = 4 * (n + 2 * case["seqs"] + 1)
    return {"bytes": elements * (size + 1) + 4 * n * case["rot"] + tables, "flops": 6 * elements}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_attention(case, s):
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["query"].shape[0], hq, d, dtype=torch.float64, device=DEV)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b in range(len(lens)):
        t, n = cu[b + 1] - cu[b], lens[b]
        places = torch.arange(n, device=DEV)
        pages = s["table"][b].long()[places // page]
        for h in range(hk):
            k = s["k_cache"][pages, h, places % page].double()
            v = s["v_cache"][pages, h, places % page].double()
            for g in range(hq // hk):
                head = h * (hq // hk) + g
                score = float(s["alpha_qk"]) * (s["query"][cu[b]:cu[b + 1], head].double() @ k.T)
                if t > 1:
                    score += torch.full((t, n), float("-inf"), dtype=torch.float64, device=DEV).triu_(n - t + 1)
                out[cu[b]:cu[b + 1], head] = float(s["alpha_pv"]) * (torch.softmax(score, 1) @ v)
    if case["out"] == "int8":
        return out.round().clamp(-128, 127) * float(s["step"])
    return out


def _exact_append(case, s):
    page, rot = case["page"], case["rot"]
    k_cache, v_cache = s["k_cache"].clone(), s["v_cache"].clone()
    cu, lens, alphas = s["cu"].tolist(), s["lens"].tolist(), s["alphas"]
    q_out = None if s["query"] is None else torch.zeros(s["query"].shape, dtype=torch.int8, device=DEV)
    for b in range(len(lens)):
        rows = slice(cu[b], cu[b + 1])
        position = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device=DEV)
        pages, offset = s["table"][b].long()[position // page], position % page
        done = []
        for x, alpha, turned in ((s["query"], alphas[0], True), (s["key"], alphas[1], True), (s["value"], alphas[2], False)):
            if x is None:
                done.append(None)
                continue
            y = x[rows].double()
            if turned and rot:
                first = torch.arange(0, rot, 2) if case["neighbours"] else torch.arange(rot // 2)
                second = first + 1 if case["neighbours"] else first + rot // 2
                z = torch.view_as_complex(torch.stack([y[..., first], y[..., second]], -1).contiguous())
                e = s["cos_sin"][position].double()
                z = z * torch.complex(e[:, : rot // 2], e[:, rot // 2:])[:, None]
                y[..., first], y[..., second] = z.real, z.imag
            done.append((y * float(alpha)).round().clamp(-128, 127).to(torch.int8))
        k_cache[pages, :, offset], v_cache[pages, :, offset] = done[1], done[2]
        if q_out is not None:
            q_out[rows] = done[0]
    return [k_cache, v_cache] + ([] if q_out is None else [q_out])


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(case, s) if case["op"] == "attention" else _exact_append(case, s)
