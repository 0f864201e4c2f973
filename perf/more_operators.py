"""A key/value cache in pages and in 4 bits, operator by operator, and the log probabilities by which a user judges what a model gives its tokens: keys and
values that a step appends, attention over the pages, and log probability, entropy, rank and best alternatives of given tokens.

The cache of a layer: codes uint8 [pages, key/value heads, P, D / 2], two to a byte, the even column in the low half, and one word int16 [pages, heads, P] for each
row: its scale s, a float32 of five significant bits (exponent in the upper eight bits of the word, mantissa in the four below), and its zero point z in
the lowest four bits. A code c stands for (c - z) s. A table [requests, W] says which pages hold a request's tokens; a slot is page * P + row.

* append: keys and queries are rotated (neox pairs), and by a Hadamard matrix / sqrt(D) behind that where `hadamard` says so. Of a row's values, which
  count as +-2^126 beyond that: hi = max(largest, 0), lo = min(smallest, 0) of the finite ones, s = (hi - lo) / 15 rounded to five significant bits (halves up), at
  least 2^-60, z = rint(-lo / s), c = rint(x / s) + z, both between 0 and 15. Behind it the rows are read back in 16 bits, as a program does that moves pages.
* attend: softmax attention of every token over its request's keys up to its own position.
* logprob: of each row of logits / temperature: the given token's log probability and rank (1: no logit is larger), the entropy, and the `top` largest log
  probabilities with their tokens, equal ones by the lower token.

A case is a dict of plain values; `kind` says which of the three it is.
"""
import math

import torch

own = False
F16, F32, F64, I16, I32, I64, U8 = torch.float16, torch.float32, torch.float64, torch.int16, torch.int32, torch.int64, torch.uint8
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FLOOR, MOST = 2.0 ** -60, 2.0 ** 126


def listed():
    return [
        # one draft token of each of the four sequences of an interactive server
        {"name": "append_draft_4", "kind": "append", "seqs": 4, "per": 1, "context": 900, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "hadamard": True},
        # 64 sequences with four tokens each, in front of their verification
        {"name": "append_verify_256", "kind": "append", "seqs": 64, "per": 4, "context": 1000, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "hadamard": True},
        # prompt portions of three sequences, keys as they are
        {"name": "append_prompt_4200", "kind": "append", "seqs": 3, "per": 1400, "context": 701, "heads": 40, "kv": 8, "dim": 128, "page": 32, "type": "bf16", "hadamard": False},
        # attention of one draft token of each of four sequences
        {"name": "attend_draft_4", "kind": "attend", "seqs": 4, "per": 1, "context": 900, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "decoding": 0},
        # 64 sequences verify three draft tokens each, over unequal contexts
        {"name": "attend_verify_256", "kind": "attend", "seqs": 64, "per": 4, "context": 4000, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "decoding": 0},
        # one token after a very long context
        {"name": "attend_long_131071", "kind": "attend", "seqs": 1, "per": 1, "context": 131071, "heads": 64, "kv": 8, "dim": 128, "page": 128, "type": "bf16", "decoding": 0},
        # a prompt portion in the middle of a prompt
        {"name": "attend_prompt_2000", "kind": "attend", "seqs": 1, "per": 2000, "context": 1000, "heads": 32, "kv": 8, "dim": 128, "page": 32, "type": "f16", "decoding": 0},
        # the token that each of four sequences has emitted, without alternatives
        {"name": "logprob_4", "kind": "logprob", "rows": 4, "vocab": 128256, "top": 0, "type": "f16", "temperature": 1.0},
        # all places of a verification by 64 sequences, with the five best tokens
        {"name": "logprob_verify_256", "kind": "logprob", "rows": 256, "vocab": 128256, "top": 5, "type": "f16", "temperature": 0.8},
        # a text of 1000 tokens is scored, over a vocabulary of odd size, with twenty alternatives
        {"name": "logprob_text_1000", "kind": "logprob", "rows": 1000, "vocab": 151643, "top": 20, "type": "f32", "temperature": 1.0},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "append", "attend", "attend", "attend", "logprob", "logprob"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (40, 8, 128), (16, 16, 128), (8, 1, 128), (16, 4, 64), (4, 2, 64), (12, 4, 128)])
    kind_of = rng.choice(["f16", "f16", "bf16"])
    if kind == "append":
        if rng.random() < 0.6:
            seqs, per = log(1, 64), rng.randint(1, 6)
        else:
            seqs, per = rng.randint(1, 4), log(16, 4200 * 56 * 128 // ((heads + 2 * kv) * dim) // 4)
            per = min(per, 1200)
        return {"kind": kind, "seqs": seqs, "per": per, "context": log(1, 1000), "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind_of,
                "hadamard": rng.random() < 0.6}
    if kind == "attend":
        if rng.random() < 0.7:
            seqs, per = log(1, 100), rng.choice([1, 1, 2, 4, 5])
            most = 64 * 4000 * 8 * 128 // (kv * dim * seqs)
            context = log(1, max(1, min(131071, most)))
            return {"kind": kind, "seqs": seqs, "per": per, "context": context, "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind_of, "decoding": 0}
        seqs = rng.randint(1, 3)
        per = log(17, min(2000, 2000 * 32 * 128 // (heads * dim * seqs)))
        context = rng.choice([0, 1, rng.randint(2, 1000)])
        return {"kind": kind, "seqs": seqs, "per": per, "context": context, "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind_of, "decoding": rng.choice([0, 0, 1])}
    vocab, kind_of = rng.choice([1024, 32000, 32001, 128256, 151643, 152064]), rng.choice(["f16", "f16", "bf16", "f32"])
    return {"kind": kind, "rows": log(1, min(1000, 1000 * 151643 // vocab)), "vocab": vocab, "top": rng.choice([0, 1, 2, 5, 20, 32]), "type": kind_of,
            "temperature": rng.choice([1.0, 0.7, 1.5])}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + part)


def _spread(most, n, seed):
    """Lengths from half of `most` up to it, in an order of the seed's."""
    g = torch.Generator().manual_seed(seed * 31 + 5)
    if n == 1:
        return torch.tensor([most])
    return torch.linspace(most - most // 2, most, n).round().to(I64)[torch.randperm(n, generator=g)]


def _pages(lens, page, seed, extra=3):
    """A table for requests that hold `lens` tokens each; the pages lie anywhere among all of them."""
    need = (lens + page - 1) // page
    total, width = int(need.sum()), max(1, int(need.max()))
    g = torch.Generator().manual_seed(seed * 31 + 6)
    order = torch.randperm(total + extra, generator=g)
    at = torch.arange(width)[None] + (need.cumsum(0) - need)[:, None]
    table = torch.where(torch.arange(width)[None] < need[:, None], order[at.clamp(max=total + extra - 1)], 0)
    return table.to(I32), total + extra


def _appended(case, seed):
    """Positions, slots and the slots of all rows that the requests hold in the touched pages."""
    page, per = case["page"], case["per"]
    first = _spread(case["context"], case["seqs"], seed)
    table, pages = _pages(first + per, page, seed)
    pos = first[:, None] + torch.arange(per)[None]
    slots = table.to(I64).gather(1, pos // page) * page + pos % page
    begin = first // page * page
    most = int((first + per - begin).max())
    row = begin[:, None] + torch.arange(most)[None]
    there = row < (first + per)[:, None]
    rows = (table.to(I64).gather(1, (row // page).clamp(max=table.shape[1] - 1)) * page + row % page)[there]
    return pos.reshape(-1), slots.reshape(-1), rows, pages


def _cos_sin(rows, dim, dtype):
    inv = 1.0 / (500000.0 ** (torch.arange(0, dim, 2, dtype=F32) / dim))
    angle = torch.outer(torch.arange(rows, dtype=F32), inv)
    return torch.cat((angle.cos(), angle.sin()), -1).to(dtype).cuda()


def _pool(g, pages, kv, page, dim):
    """Pages as rows of normal numbers leave them: codes around a zero point near the middle, scales of a third, more or less."""
    middle = 6 + torch.randint(0, 4, (pages, kv, page), generator=g, device="cuda")
    codes = torch.randn(pages, kv, page, dim, generator=g, device="cuda").mul_(3).add_(middle[..., None]).round_().clamp_(0, 15).to(U8)
    # (16 .. 31) / 16 times 2^-2: 0.25 to 0.48
    word = (125 << 8) + (torch.randint(0, 16, (pages, kv, page), generator=g, device="cuda") << 4) + middle
    return codes[..., 0::2] | codes[..., 1::2] << 4, word.to(I16)


def _append_inputs(case, seed):
    pos, slots, rows, pages = _appended(case, seed)
    g, dtype = _gen(seed, 1), TYPES[case["type"]]
    tokens, width = pos.numel(), (case["heads"] + 2 * case["kv"]) * case["dim"]
    qkv = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    k, kp = _pool(g, pages, case["kv"], case["page"], case["dim"])
    v, vp = _pool(g, pages, case["kv"], case["page"], case["dim"])
    return qkv, _cos_sin(int(pos.max()) + 1, case["dim"], dtype), pos.to(I32).cuda(), slots.to(I32).cuda(), rows.to(I32).cuda(), k, v, kp, vp


def _attend_lens(case, seed):
    first = _spread(case["context"], case["seqs"], seed)
    count = torch.full((case["seqs"],), case["per"])
    if case["decoding"]:
        first = torch.cat([first, _spread(case["context"] + 40, case["decoding"], seed + 1)])
        count = torch.cat([count, torch.ones(case["decoding"], dtype=I64)])
    return first, count


def _attend_inputs(case, seed):
    first, count = _attend_lens(case, seed)
    table, pages = _pages(first + count, case["page"], seed)
    g = _gen(seed, 1)
    q = (1.5 * torch.randn(int(count.sum()), case["heads"], case["dim"], generator=g, device="cuda")).to(TYPES[case["type"]])
    k, kp = _pool(g, pages, case["kv"], case["page"], case["dim"])
    v, vp = _pool(g, pages, case["kv"], case["page"], case["dim"])
    start = torch.cat([torch.zeros(1, dtype=I64), count.cumsum(0)]).to(I32).cuda()
    return q, k, v, kp, vp, table.cuda(), start, (first + count).to(I32).cuda()


def _logprob_inputs(case, seed):
    g = _gen(seed, 1)
    logits = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda").mul_(3).to(TYPES[case["type"]])
    # tokens that a model emits: the largest of a few at random, and sometimes any
    some = torch.randint(0, case["vocab"], (case["rows"], 50), generator=g, device="cuda")
    return logits, some.gather(1, logits.gather(1, some).argmax(1, keepdim=True))[:, 0]


def prepare(case, seed):
    kind = case["kind"]
    cuda = {"device": "cuda"}
    if kind == "append":
        qkv, cos_sin, pos, slots, rows, k, v, kp, vp = _append_inputs(case, seed)
        shape = (rows.numel(), case["kv"], case["dim"])
        return {"kind": kind, "qkv": qkv, "cos_sin": cos_sin, "positions": pos, "slots": slots, "rows": rows, "k": k, "v": v, "kp": kp, "vp": vp, "heads": case["heads"],
                "hadamard": case["hadamard"], "q": torch.empty(pos.numel(), case["heads"], case["dim"], dtype=qkv.dtype, **cuda),
                "k_rows": torch.empty(shape, dtype=qkv.dtype, **cuda), "v_rows": torch.empty(shape, dtype=qkv.dtype, **cuda)}
    if kind == "attend":
        q, k, v, kp, vp, table, start, lens = _attend_inputs(case, seed)
        return {"kind": kind, "q": q, "k": k, "v": v, "kp": kp, "vp": vp, "table": table, "q_start": start, "kv_len": lens, "scale": case["dim"] ** -0.5,
                "most": max(case["per"], 1), "out": torch.empty_like(q), "work": None}
    logits, tokens = _logprob_inputs(case, seed)
    n, top = case["rows"], case["top"]
    return {"kind": kind, "logits": logits, "tokens": tokens, "temperature": case["temperature"], "top": top, "logprobs": torch.empty(n, dtype=F32, **cuda),
            "entropy": torch.empty(n, dtype=F32, **cuda), "ranks": torch.empty(n, dtype=I64, **cuda), "top_logprobs": torch.empty(n, top, dtype=F32, **cuda),
            "top_tokens": torch.empty(n, top, dtype=I64, **cuda)}


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------
def _plain_turned(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_butterflies(x, step):
    """Sums and differences of the values `step` apart, and then of those twice as far."""
    if step == x.shape[-1]:
        return x * x.shape[-1] ** -0.5
    a, b = x.unflatten(-1, (-1, 2, step)).unbind(-2)
    return _plain_butterflies(torch.stack((a + b, a - b), -2).flatten(-3), 2 * step)


def _plain_scale(word):
    return ((word.to(I32) & 0xfff0) << 15).view(F32), (word.to(I32) & 15).float()


def _plain_values(codes, word):
    scale, zero = _plain_scale(word)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (both.float() - zero[..., None]) * scale[..., None]


def _plain_write(x, slots, codes, words):
    """Rows x [T, G, D] into their slots, which are all there."""
    page = codes.shape[2]
    x = x.clamp(-MOST, MOST)
    hi, lo = x.amax(-1).clamp(min=0), x.amin(-1).clamp(max=0)
    bits = (((hi - lo) / 15).clamp(min=FLOOR).view(I32) + (1 << 18)) >> 19
    scale = (bits << 19).view(F32)
    zero = (-lo / scale).round().clamp(0, 15)
    code = ((x / scale[..., None]).round() + zero[..., None]).clamp(0, 15).to(U8)
    codes[slots // page, :, slots % page] = code[..., 0::2] | code[..., 1::2] << 4
    words[slots // page, :, slots % page] = (bits << 4 | zero.to(I32)).to(I16)


def _plain_append(s):
    heads, kv, dim = s["heads"], s["k"].shape[1], s["k"].shape[3] * 2
    t = s["positions"].numel()
    qkv = s["qkv"].float().reshape(t, heads + 2 * kv, dim)
    cos, sin = s["cos_sin"][s["positions"].long()].float()[:, None].chunk(2, -1)
    turned = _plain_turned(qkv[:, : heads + kv], cos, sin)
    if s["hadamard"]:
        turned = _plain_butterflies(turned, 1)
    slots, rows, page = s["slots"].long(), s["rows"].long(), s["k"].shape[2]
    _plain_write(turned[:, heads:], slots, s["k"], s["kp"])
    _plain_write(qkv[:, heads + kv:], slots, s["v"], s["vp"])
    back = [_plain_values(c[rows // page, :, rows % page], w[rows // page, :, rows % page]).to(s["qkv"].dtype) for c, w in ((s["k"], s["kp"]), (s["v"], s["vp"]))]
    return [turned[:, :heads].to(s["qkv"].dtype), *back, s["kp"], s["vp"]]


def _plain_attend(s):
    q, table = s["q"], s["table"].long()
    t, heads, dim = q.shape
    n, kv = table.shape[0], s["k"].shape[1]
    start, lens = s["q_start"].long(), s["kv_len"].long()
    token = torch.arange(t, device=q.device)
    req = torch.searchsorted(start[1:], token, right=True)
    nth = token - start[req]
    pos = lens[req] - (start[1:] - start[:-1])[req] + nth
    keys, values = (_plain_values(c, w)[table].permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim) for c, w in ((s["k"], s["kp"]), (s["v"], s["vp"])))
    # every request's tokens in rows of their own, as many as the longest has
    most, rep = s["most"], heads // kv
    rows = torch.zeros(n, most, heads, dim, device=q.device)
    rows[req, nth] = q.float()
    at = torch.full((n, most), -1, device=q.device)
    at[req, nth] = pos
    rows = rows.reshape(n, most, kv, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, most * rep, dim)
    score = torch.matmul(rows, keys.transpose(2, 3)) * s["scale"]
    hidden = torch.arange(keys.shape[2], device=q.device)[None, None] > at.repeat_interleave(rep, 1)[:, :, None]
    score = score.masked_fill_(hidden[:, None], -math.inf)
    weight = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, kv, most, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, most, heads, dim)
    return out[req, nth].to(q.dtype)


def _plain_logprob(s):
    logits, tokens = s["logits"], s["tokens"]
    # (sums over a vocabulary in 64 bits)
    z = logits.double() / s["temperature"]
    z = z - z.amax(-1, keepdim=True)
    weight = z.exp()
    total = weight.sum(-1)
    lse = total.log()
    entropy = lse - (weight * z).sum(-1) / total
    del weight
    at = tokens[:, None]
    logprob = z.gather(1, at)[:, 0] - lse
    rank = (logits > logits.gather(1, at)).sum(-1) + 1
    # (the order of equal ones is kept: the lower token first)
    best = logits.sort(dim=-1, descending=True, stable=True).indices[:, : s["top"]]
    return [logprob.float(), entropy.float(), rank, (z.gather(1, best) - lse[:, None]).float(), best]


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logprob": _plain_logprob}[kind](s)
    from qspec_b200 import ops
    if kind == "append":
        ops.kv4_append(s["qkv"], s["cos_sin"], s["positions"], s["slots"], s["k"], s["v"], s["kp"], s["vp"], s["q"], hadamard=s["hadamard"])
        ops.kv4_read(s["k"], s["v"], s["kp"], s["vp"], s["rows"], s["k_rows"], s["v_rows"])
        return [s["q"], s["k_rows"], s["v_rows"], s["kp"], s["vp"]]
    if kind == "attend":
        if s["work"] is None:  # kept from call to call, as a model keeps it from layer to layer
            s["work"] = ops.kv4_attention_workspace(s["q"].device)
        return ops.kv4_attention(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["q_start"], s["kv_len"], s["out"], s["scale"], s["work"], max_tokens=s["most"])
    top = (s["top_logprobs"], s["top_tokens"]) if s["top"] else (None, None)
    ops.token_logprobs(s["logits"], s["tokens"], s["logprobs"], s["entropy"], s["ranks"], *top, temperature=s["temperature"])
    return [s["logprobs"], s["entropy"], s["ranks"], s["top_logprobs"], s["top_tokens"]]


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "logprob":
        n, size = case["rows"], {"f16": 2, "bf16": 2, "f32": 4}[case["type"]]
        return {"bytes": n * (case["vocab"] * size + 24 + case["top"] * 12), "flops": n * case["vocab"] * 6}
    row = case["kv"] * (case["dim"] // 2 + 2) * 2  # a token's codes and words, keys and values
    if kind == "append":
        first = _spread(case["context"], case["seqs"], 0)
        rows = int((first % case["page"]).sum()) + case["seqs"] * case["per"]
        tokens = case["seqs"] * case["per"]
        qkv = (case["heads"] * 2 + case["kv"] * 2) * case["dim"] * 2
        stages = int(math.log2(case["dim"])) + 1 if case["hadamard"] else 0
        return {"bytes": tokens * (qkv + row + case["dim"] * 2 + 8) + rows * (row + case["kv"] * case["dim"] * 4 + 4),
                "flops": tokens * case["dim"] * ((case["heads"] + case["kv"]) * (3 + stages) + case["kv"] * 2 * 4)}
    first, count = _attend_lens(case, 0)
    pairs = int((count * first + count * (count + 1) // 2).sum())
    keys, tokens = int((first + count).sum()), int(count.sum())
    return {"bytes": keys * row + keys // case["page"] * 4 + tokens * case["heads"] * case["dim"] * 4, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------------------
def _exact_rows(codes, word):
    """What the words and codes of rows [n, D / 2] stand for."""
    w = word.to(I64) % 65536
    scale = torch.ldexp(1 + (w // 16 % 16).to(F64) / 16, w // 256 - 127)
    c = codes.to(I64)
    both = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=F64, device=codes.device)
    both[..., ::2], both[..., 1::2] = (c % 16).to(F64), (c // 16).to(F64)
    return (both - (w % 16).to(F64)[..., None]) * scale[..., None]


def _exact_quantised(x):
    hi, lo = torch.relu(x.amax(-1)), -torch.relu(-x.amin(-1))
    mantissa, exponent = torch.frexp(torch.maximum((hi - lo) / 15, torch.tensor(FLOOR, dtype=F64, device=x.device)))
    scale = torch.ldexp(torch.floor(mantissa * 32 + 0.5), exponent - 5)
    zero = torch.round(-lo / scale).clamp(0, 15)
    return ((torch.round(x / scale[..., None]) + zero[..., None]).clamp(0, 15) - zero[..., None]) * scale[..., None]


def _exact_append(case, seed):
    qkv, cos_sin, pos, slots, rows, k, v, kp, vp = _append_inputs(case, seed)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    z = qkv.to(F64).view(-1, heads + 2 * kv, 2, dim // 2)
    table = cos_sin.to(F64)[pos.long()].view(-1, 1, 2, dim // 2)
    turned = torch.complex(z[:, :, 0], z[:, :, 1]) * torch.complex(table[:, :, 0], table[:, :, 1])
    turned = torch.stack([turned.real, turned.imag], 2).reshape(-1, heads + 2 * kv, dim)
    if case["hadamard"]:
        i = torch.arange(dim, device="cuda")
        both, signs = i[:, None] & i[None], torch.zeros(dim, dim, dtype=I64, device="cuda")
        for bit in range(7):
            signs += both >> bit & 1
        turned = turned @ ((1 - 2 * (signs % 2)).to(F64) / math.sqrt(dim))
    sides = []
    for x, codes, words in ((turned[:, heads: heads + kv], k, kp), (z.reshape(-1, heads + 2 * kv, dim)[:, heads + kv:], v, vp)):
        at = rows.long()
        values = _exact_rows(codes[at // page, :, at % page], words[at // page, :, at % page])
        where = torch.full((codes.shape[0] * page,), -1, device="cuda")
        where[at] = torch.arange(at.numel(), device="cuda")
        values[where[slots.long()]] = _exact_quantised(x)
        sides.append(values)
    return [turned[:, :heads].contiguous(), *sides, None, None]


def _exact_attend(case, seed):
    q, k, v, kp, vp, table, start, lens = _attend_inputs(case, seed)
    rep = case["heads"] // case["kv"]
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    for b, (lo, hi, n) in enumerate(zip(start[:-1].tolist(), start[1:].tolist(), lens.tolist())):
        own_pages = table[b, : -(-n // case["page"])].long()
        for g in range(case["kv"]):
            keys, values = (_exact_rows(c[own_pages, g], w[own_pages, g]).reshape(-1, case["dim"])[:n] for c, w in ((k, kp), (v, vp)))
            for h in range(g * rep, (g + 1) * rep):
                z = q[lo:hi, h].to(F64) @ keys.T * case["dim"] ** -0.5
                late = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
                out[lo:hi, h] = torch.softmax(z.masked_fill(late, -math.inf), 1) @ values
    return out


def _exact_logprob(case, seed):
    logits, tokens = _logprob_inputs(case, seed)
    n, top = case["rows"], case["top"]
    out = [torch.empty(n, dtype=F64, device="cuda"), torch.empty(n, dtype=F64, device="cuda"), None, torch.empty(n, top, dtype=F64, device="cuda"), None]
    for lo in range(0, n, 64):
        at = slice(lo, min(lo + 64, n))
        p = torch.log_softmax(logits[at].to(F64) / case["temperature"], -1)
        out[0][at] = p[torch.arange(p.shape[0], device="cuda"), tokens[at]]
        out[1][at] = -torch.special.xlogy(p.exp(), p.exp()).sum(-1)
        out[3][at] = torch.topk(p, top, -1).values
    return out


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "logprob": _exact_logprob}[case["kind"]](case, seed)
