"""A speculative step over a key/value cache that lies in pages and in 8 bits, operator by operator: pages and slots for the step's tokens, the
keys and values that the step appends, attention over the pages, and the verification of drafted tokens with random numbers.

The cache of a layer: codes int8 [pages, key/value heads, P, D] and scales float32 [pages, heads], one for each page and head; a code c stands
for c * scale. A table [requests, W] says which pages hold a request's tokens; a slot is page * P + row.

* plan: `lengths` tokens are held, `counts` come with the step (negative: the request has ended). Ended requests give their pages back, behind
  the free ones; the others take the pages that they need from the end of that list, in the order of the requests. A request whose pages do not
  fit any more (everything that was asked for so far, its own included, is more than there is) gets none, and its tokens no slots.
* append: keys and queries are rotated; a page's scale is the largest of |x| / 127 of its rows, of what it was before (unless the page begins
  in this step) and 2^-60; the older rows of a page whose scale grows are put on the new one. Behind it the rows of the pages that the step
  touched are read back in 16 bits, as a program does that moves pages.
* attend: softmax attention of every token over its request's keys up to its own position.
* verify: draft i is taken if u_i q(d_i) < p(d_i) and all before it were; then one token from max(p - q, 0) at the first place that was refused (from
  p where all were taken, or where nothing is left): the first whose running sum is above u * total.

A case is a dict of plain values; `kind` says which of the four it is.
"""
import math

import torch

own = False
F16, F32, F64, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
FLOOR = 2.0 ** -60


def listed():
    return [
        # the page plan of one step of a server with 64 sequences that verify three draft tokens each; five requests have ended
        {"name": "plan_step_64", "kind": "plan", "requests": 64, "per": 4, "context": 1000, "page": 64, "ended": 5, "prompts": 0, "portion": 0, "scarce": False},
        # a step of a large server: prompts beside decoding requests, small pages, long contexts, more asked for than there is
        {"name": "plan_mixed_1000", "kind": "plan", "requests": 1000, "per": 2, "context": 32000, "page": 16, "ended": 37, "prompts": 30, "portion": 2001, "scarce": True},
        # one draft token of each of the four sequences of an interactive server. The smallest call.
        {"name": "append_draft_4", "kind": "append", "seqs": 4, "per": 1, "context": 900, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16"},
        # 64 sequences with four tokens each, in front of their verification
        {"name": "append_verify_256", "kind": "append", "seqs": 64, "per": 4, "context": 1000, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16"},
        # prompt portions of three sequences
        {"name": "append_prompt_4200", "kind": "append", "seqs": 3, "per": 1400, "context": 700, "heads": 40, "kv": 8, "dim": 128, "page": 32, "type": "bf16"},
        # attention of one draft token of each of four sequences
        {"name": "attend_draft_4", "kind": "attend", "seqs": 4, "per": 1, "context": 900, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "decoding": 0},
        # 64 sequences verify three draft tokens each, over unequal contexts
        {"name": "attend_verify_256", "kind": "attend", "seqs": 64, "per": 4, "context": 4000, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "f16", "decoding": 0},
        # one token after a very long context
        {"name": "attend_long_131071", "kind": "attend", "seqs": 1, "per": 1, "context": 131071, "heads": 64, "kv": 8, "dim": 128, "page": 128, "type": "bf16", "decoding": 0},
        # a prompt portion in the middle of a prompt
        {"name": "attend_prompt_2000", "kind": "attend", "seqs": 1, "per": 2000, "context": 1000, "heads": 32, "kv": 8, "dim": 128, "page": 32, "type": "f16", "decoding": 0},
        # four sequences, three draft tokens each
        {"name": "verify_4", "kind": "verify", "seqs": 4, "drafts": 3, "vocab": 128256, "agree": 0.8, "ragged": False},
        # 64 sequences
        {"name": "verify_64", "kind": "verify", "seqs": 64, "drafts": 3, "vocab": 128256, "agree": 0.8, "ragged": False},
        # many sequences with up to five draft tokens, not all of them the same number
        {"name": "verify_190_ragged", "kind": "verify", "seqs": 190, "drafts": 5, "vocab": 152064, "agree": 0.5, "ragged": True},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "verify", "verify"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (40, 8, 128), (16, 16, 128), (8, 1, 128), (16, 4, 64), (4, 2, 64), (12, 4, 128)])
    kind_of = rng.choice(["f16", "f16", "bf16"])
    if kind == "plan":
        requests = log(1, 1000)
        return {"kind": kind, "requests": requests, "per": rng.randint(1, 6), "context": log(1, 32000), "page": page, "ended": rng.randint(0, requests // 8),
                "prompts": min(requests // 4, rng.randint(0, 20)), "portion": log(2, 2000), "scarce": rng.random() < 0.3}
    if kind == "append":
        if rng.random() < 0.6:
            seqs, per = log(1, 64), rng.randint(1, 6)
        else:
            seqs, per = rng.randint(1, 4), log(16, 4200 * 56 * 128 // ((heads + 2 * kv) * dim) // 4)
            per = min(per, 1200)
        return {"kind": kind, "seqs": seqs, "per": per, "context": log(1, 1000), "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind_of}
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
    return {"kind": kind, "seqs": log(1, 100), "drafts": rng.choice([0, 1, 2, 3, 3, 4, 5, 8]), "vocab": rng.choice([1024, 32000, 32001, 128256, 151643, 152064]),
            "agree": rng.choice([0.3, 0.5, 0.8, 0.95]), "ragged": rng.random() < 0.4}


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


def _plan_inputs(case, seed):
    n, page = case["requests"], case["page"]
    g = torch.Generator().manual_seed(seed * 31 + 7)
    # who asks for what is the case's, in which order they come is the seed's
    mix = torch.Generator().manual_seed(11)
    lens = (torch.rand(n, generator=mix) * case["context"] + 1).to(I64)
    lens[: case["prompts"]] //= 4
    counts = torch.full((n,), case["per"], dtype=I64)
    counts[: case["prompts"]] = case["portion"]
    counts[case["prompts"]: case["prompts"] + case["ended"]] = -1
    counts[n - n // 16:] = 0  # requests that wait
    held = (lens + page - 1) // page
    held = held + (torch.rand(n, generator=mix) < 0.1)  # a page more, where a draft that was refused had begun one
    shuffled = torch.randperm(n, generator=g)
    lens, counts, held = lens[shuffled], counts[shuffled], held[shuffled]
    width = int(((lens + counts.clamp(min=0) + page - 1) // page).max().clamp(min=int(held.max())))
    need = (((lens + counts.clamp(min=0) + page - 1) // page) - held).clamp(min=0) * (counts > 0)
    back = int((held * (counts < 0)).sum())
    free = max(0, int(need.sum()) * 2 // 3 - back) if case["scarce"] else int(need.sum()) + 40
    order = torch.randperm(int(held.sum()) + free, generator=g)
    at = torch.arange(width)[None] + (held.cumsum(0) - held)[:, None]
    table = torch.where(torch.arange(width)[None] < held[:, None], order[free:][at.clamp(max=int(held.sum()) - 1)], 0)
    stack = torch.zeros(order.numel(), dtype=I64)
    stack[:free] = order[:free]
    state = torch.cat([held, torch.tensor([free])])
    tokens = n * case["per"] + case["prompts"] * case["portion"]
    return [t.to(I32).cuda() for t in (lens, counts, table, stack, state)], tokens


def _appended(case, seed):
    """Positions, slots and the slots of all rows of the touched pages."""
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
    codes = (torch.randn(pages, kv, page, dim, generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
    scales = 2.0 ** (torch.rand(pages, kv, generator=g, device="cuda") - 0.5) / 32
    return codes, scales


def _append_inputs(case, seed):
    pos, slots, rows, pages = _appended(case, seed)
    g, dtype = _gen(seed, 1), TYPES[case["type"]]
    tokens, width = pos.numel(), (case["heads"] + 2 * case["kv"]) * case["dim"]
    qkv = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    k, ks = _pool(g, pages, case["kv"], case["page"], case["dim"])
    v, vs = _pool(g, pages, case["kv"], case["page"], case["dim"])
    return qkv, _cos_sin(int(pos.max()) + 1, case["dim"], dtype), pos.to(I32).cuda(), slots.to(I32).cuda(), rows.to(I32).cuda(), k, v, ks, vs


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
    k, ks = _pool(g, pages, case["kv"], case["page"], case["dim"])
    v, vs = _pool(g, pages, case["kv"], case["page"], case["dim"])
    start = torch.cat([torch.zeros(1, dtype=I64), count.cumsum(0)]).to(I32).cuda()
    return q, k, v, ks, vs, table.cuda(), start, (first + count).to(I32).cuda()


def _verify_inputs(case, seed):
    b, k, n = case["seqs"], case["drafts"], case["vocab"]
    g = _gen(seed, 1)
    target = torch.softmax(torch.randn(b, k + 1, n, generator=g, device="cuda").mul_(2.5), -1)
    if k:
        # a draft model that gives tokens other probabilities than the target, the more the less they agree
        noise = torch.randn(b, k, n, generator=g, device="cuda").mul_(2.5 * (1 - case["agree"]))
        draft = torch.softmax(target[:, :k].log().add_(noise), -1)
        del noise
        drafted = torch.multinomial(draft.reshape(b * k, n), 1, generator=g).reshape(b, k)
    else:
        draft, drafted = torch.empty(b, 0, n, device="cuda"), torch.empty(b, 0, dtype=I64, device="cuda")
    uniform = torch.rand(b, k + 1, generator=g, device="cuda")
    counts = torch.randint(0, k + 1, (b,), generator=g, device="cuda").to(I32) if case["ragged"] else None
    return drafted, draft, target, uniform, counts


def prepare(case, seed):
    kind = case["kind"]
    cuda = {"device": "cuda"}
    if kind == "plan":
        (lens, counts, table, stack, state), tokens = _plan_inputs(case, seed)
        n = case["requests"]
        i32 = {"dtype": I32, "device": "cuda"}
        return {"kind": kind, "lengths": lens, "counts": counts, "table": table, "free": stack, "state": state, "page": case["page"],
                "q_start": torch.empty(n + 1, **i32), "kv_len": torch.empty(n, **i32), "positions": torch.empty(tokens, **i32), "seq_ids": torch.empty(tokens, **i32),
                "slots": torch.empty(tokens, **i32), "state_out": torch.empty(n + 2, **i32)}
    if kind == "append":
        qkv, cos_sin, pos, slots, rows, k, v, ks, vs = _append_inputs(case, seed)
        shape = (rows.numel(), case["kv"], case["dim"])
        return {"kind": kind, "qkv": qkv, "cos_sin": cos_sin, "positions": pos, "slots": slots, "rows": rows, "k": k, "v": v, "ks": ks, "vs": vs, "heads": case["heads"],
                "q": torch.empty(pos.numel(), case["heads"], case["dim"], dtype=qkv.dtype, **cuda),
                "k_rows": torch.empty(shape, dtype=qkv.dtype, **cuda), "v_rows": torch.empty(shape, dtype=qkv.dtype, **cuda)}
    if kind == "attend":
        q, k, v, ks, vs, table, start, lens = _attend_inputs(case, seed)
        return {"kind": kind, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table, "q_start": start, "kv_len": lens, "scale": case["dim"] ** -0.5,
                "most": max(case["per"], 1), "out": torch.empty_like(q), "work": None}
    drafted, draft, target, uniform, counts = _verify_inputs(case, seed)
    return {"kind": kind, "drafted": drafted, "draft": draft, "target": target, "uniform": uniform, "counts": counts,
            "tokens": torch.empty(case["seqs"], case["drafts"] + 1, dtype=I64, **cuda), "emitted": torch.empty(case["seqs"], dtype=I64, **cuda)}


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------
def _plain_plan(s):
    lens, counts, table, stack, page = s["lengths"].long(), s["counts"].long(), s["table"], s["free"], s["page"]
    n, width = table.shape
    held, free = s["state"][:n].long(), s["state"][n].long()
    ends, new = counts < 0, counts.clamp(min=0)
    wanted = (lens + new + page - 1) // page
    fits = wanted <= width
    need = torch.where((counts > 0) & fits, (wanted - held).clamp(min=0), 0)
    back = torch.where(ends, held, 0)
    have = free + back.sum()
    asked = need.cumsum(0)
    granted = ~ends & ((need == 0) | (asked <= have)) & ((counts == 0) | fits)
    # the list of free pages with what has come back behind it
    col = torch.arange(width, device=table.device)
    back_at = torch.where(ends[:, None] & (col[None] < held[:, None]), free + (back.cumsum(0) - back)[:, None] + col[None], stack.numel())
    whole = torch.zeros(stack.numel() + 1, dtype=I64, device=table.device)
    whole[: stack.numel()] = stack
    whole = whole.scatter(0, back_at.reshape(-1), table.reshape(-1).long())
    # pages are taken from its end
    takes = granted & (need > 0)
    nth = (asked - need)[:, None] + col[None] - held[:, None]
    new_page = takes[:, None] & (col[None] >= held[:, None]) & (col[None] < wanted[:, None])
    table.copy_(torch.where(new_page, whole[(have - 1 - nth).clamp(0, stack.numel())], table.long()))
    taken = (need * takes).sum()
    left = have - taken
    idx = torch.arange(stack.numel(), device=table.device)
    stack.copy_(torch.where((idx >= free) & (idx < left), whole[:-1], stack.long()))
    held_out = torch.where(ends, 0, torch.where(takes, wanted, held))
    refused = (~granted & ~ends).sum()
    start = torch.cat([torch.zeros(1, dtype=I64, device=table.device), new.cumsum(0)])
    token = torch.arange(s["slots"].numel(), device=table.device)
    req = torch.searchsorted(start[1:], token, right=True)
    inside = req < n
    req = req.clamp(max=n - 1)
    there = inside & granted[req]
    pos = torch.where(there, lens[req] + token - start[req], -1)
    slot = torch.where(there, table[req, (pos.clamp(min=0) // page)].long() * page + pos % page, -1)
    kv_len = torch.where(granted, lens + new, 0)
    out = [start, kv_len, pos, torch.where(inside, req, -1), slot, torch.cat([held_out, left[None], refused[None]])]
    return [t.to(I32) for t in out] + [table, stack]


def _largest(x):
    """The largest finite |x| of each row."""
    x = x.abs()
    return torch.where(x < math.inf, x, 0.0).amax(-1)


def _codes(x, scale):
    return torch.where(x == x, (x * (1.0 / scale)).round().clamp(-127, 127), 0.0)


def _plain_rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_write(x, slots, codes, scales):
    """Rows x [T, G, D] into the pages of their slots, which all are there."""
    page = codes.shape[2]
    at, row = slots // page, slots % page
    largest = torch.zeros_like(scales).index_reduce_(0, at, _largest(x), "amax")
    begun = torch.zeros(scales.shape[0], device=x.device).index_fill_(0, at, 1.0)
    fresh = torch.zeros(scales.shape[0] + 1, device=x.device).index_fill_(0, torch.where(row == 0, at, scales.shape[0]), 1.0)[:-1]
    before = torch.where(fresh[:, None] > 0, 0.0, scales)
    after = torch.maximum(torch.maximum(largest * (1.0 / 127.0), before), torch.tensor(FLOOR, device=x.device))
    codes[at] = (codes[at].float() * (before / after)[at][:, :, None, None]).round().to(torch.int8)
    codes[at, :, row] = _codes(x, after[at][:, :, None]).to(torch.int8)
    scales.copy_(torch.where(begun[:, None] > 0, after, scales))


def _plain_append(s):
    heads, kv, dim = s["heads"], s["k"].shape[1], s["k"].shape[3]
    t = s["positions"].numel()
    qkv = s["qkv"].float().reshape(t, heads + 2 * kv, dim)
    cos, sin = s["cos_sin"][s["positions"].long()].float()[:, None].chunk(2, -1)
    turned = _plain_rotated(qkv[:, : heads + kv], cos, sin)
    slots, rows, page = s["slots"].long(), s["rows"].long(), s["k"].shape[2]
    _plain_write(turned[:, heads:], slots, s["k"], s["ks"])
    _plain_write(qkv[:, heads + kv:], slots, s["v"], s["vs"])
    back = [(c[rows // page, :, rows % page].float() * sc[rows // page][:, :, None]).to(s["qkv"].dtype) for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
    return [turned[:, :heads].to(s["qkv"].dtype), *back, s["ks"], s["vs"]]


def _plain_attend(s):
    q, table, page = s["q"], s["table"].long(), s["k"].shape[2]
    t, heads, dim = q.shape
    n, kv = table.shape[0], s["k"].shape[1]
    start, lens = s["q_start"].long(), s["kv_len"].long()
    token = torch.arange(t, device=q.device)
    req = torch.searchsorted(start[1:], token, right=True)
    nth = token - start[req]
    pos = lens[req] - (start[1:] - start[:-1])[req] + nth
    keys, values = ((c[table].float() * sc[table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim) for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])))
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


def _plain_verify(s):
    target, draft, drafted, uniform = s["target"], s["draft"], s["drafted"], s["uniform"]
    b, k = drafted.shape
    place = torch.arange(k, device=target.device)
    at = drafted[:, :, None]
    taken = uniform[:, :k].double() * draft.gather(2, at)[..., 0].double() < target[:, :k].gather(2, at)[..., 0].double()
    many = s["counts"].long() if s["counts"] is not None else torch.full((b,), k, device=target.device)
    taken = taken & (place[None] < many[:, None])
    accepted = taken.long().cumprod(1).sum(1)
    req = torch.arange(b, device=target.device)
    p = target[req, accepted].double()
    rest = p
    if k:
        rest = torch.where((accepted < many)[:, None], (p - draft[req, accepted.clamp(max=k - 1)].double()).clamp(min=0), p)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(1)
    last = (upto <= uniform[:, k].double()[:, None] * upto[:, -1:]).sum(1)
    every = torch.cat([place, place.new_full((1,), k)])
    tokens = torch.cat([drafted, drafted.new_zeros(b, 1)], 1)
    tokens = torch.where(every[None] < accepted[:, None], tokens, torch.where(every[None] == accepted[:, None], last[:, None], -1))
    return tokens, accepted + 1


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "verify": _plain_verify}[kind](s)
    from qspec_b200 import ops
    if kind == "plan":
        ops.page_plan(s["lengths"], s["counts"], s["table"], s["free"], s["state"], s["page"], s["q_start"], s["kv_len"], s["positions"], s["seq_ids"], s["slots"], s["state_out"])
        return [s["q_start"], s["kv_len"], s["positions"], s["seq_ids"], s["slots"], s["state_out"], s["table"], s["free"]]
    if kind == "append":
        ops.kv8_append(s["qkv"], s["cos_sin"], s["positions"], s["slots"], s["k"], s["v"], s["ks"], s["vs"], s["q"])
        ops.kv8_read(s["k"], s["v"], s["ks"], s["vs"], s["rows"], s["k_rows"], s["v_rows"])
        return [s["q"], s["k_rows"], s["v_rows"], s["ks"], s["vs"]]
    if kind == "attend":
        if s["work"] is None:  # kept from call to call, as a model keeps it from layer to layer
            s["work"] = ops.kv8_attention_workspace(s["q"].device)
        return ops.kv8_attention(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["q_start"], s["kv_len"], s["out"], s["scale"], s["work"], max_tokens=s["most"])
    ops.verify_drafts(s["drafted"] if s["drafted"].numel() else None, s["draft"] if s["draft"].numel() else None, s["target"], s["uniform"], s["tokens"], s["emitted"],
                      draft_counts=s["counts"])
    return s["tokens"], s["emitted"]


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "plan":
        tokens = case["requests"] * case["per"] + case["prompts"] * case["portion"]
        pages = tokens // case["page"] + case["requests"]  # entries of the table that are read or written
        return {"bytes": case["requests"] * 4 * 6 + tokens * 12 + pages * 4, "flops": 0}
    if kind == "append":
        first = _spread(case["context"], case["seqs"], 0)
        rows = int((first % case["page"]).sum()) + case["seqs"] * case["per"]
        tokens, row = case["seqs"] * case["per"], case["kv"] * case["dim"] * 2
        qkv = (case["heads"] * 2 + case["kv"] * 2) * case["dim"] * 2
        return {"bytes": tokens * (qkv + row + case["dim"] * 2 + 8) + rows * (row + 2 * row + 4) + rows // case["page"] * case["kv"] * 16,
                "flops": tokens * (case["heads"] + 2 * case["kv"]) * case["dim"] * 4}
    if kind == "attend":
        first, count = _attend_lens(case, 0)
        pairs = int((count * first + count * (count + 1) // 2).sum())
        keys, tokens, row = int((first + count).sum()), int(count.sum()), case["kv"] * case["dim"] * 2
        return {"bytes": keys * row + keys // case["page"] * (case["kv"] * 8 + 4) + tokens * case["heads"] * case["dim"] * 4,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    b, k, n = case["seqs"], case["drafts"], case["vocab"]
    # a sequence whose drafts are all taken needs the target's row alone; of the drafts about this share is taken
    share = {0.3: 0.38, 0.5: 0.53, 0.8: 0.8, 0.95: 0.95}[case["agree"]]
    all_taken = share ** k if not case["ragged"] else sum(share ** i for i in range(k + 1)) / (k + 1)
    return {"bytes": int(b * n * 4 * (2 - all_taken)) + b * (k + 1) * 24, "flops": int(b * n * 3)}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------------------
def _exact_page(code, scale, x, first):
    """One page's rows code [G, P, D] at `scale` [G] once x [n, G, D] stands from row `first` on: values, scale."""
    largest = torch.nan_to_num(x, 0.0, 0.0, 0.0).abs().amax((0, 2)) / 127
    old = scale if first else torch.zeros_like(scale)
    new = torch.stack([largest, old, torch.full_like(old, FLOOR)]).amax(0)
    rows = [torch.round(code[:, :first] * (old / new)[:, None, None])] if first else []
    rows.append(torch.nan_to_num(torch.round(x.transpose(0, 1) / new[:, None, None]), 0.0, 127.0, -127.0).clamp(-127, 127))
    return torch.cat(rows, 1) * new[:, None, None], new


def _exact_append(case, seed):
    qkv, cos_sin, pos, slots, rows, k, v, ks, vs = _append_inputs(case, seed)
    heads, kv, dim, page, per = case["heads"], case["kv"], case["dim"], case["page"], case["per"]
    z = qkv.to(F64).view(-1, heads + 2 * kv, 2, dim // 2)
    table = cos_sin.to(F64)[pos.long()].view(-1, 1, 2, dim // 2)
    turn = torch.complex(table[:, :, 0], table[:, :, 1])
    turned = torch.complex(z[:, :, 0], z[:, :, 1]) * turn
    turned = torch.stack([turned.real, turned.imag], 2).reshape(-1, heads + 2 * kv, dim)
    sides = []
    for x, codes, scales in ((turned[:, heads: heads + kv], k, ks), (z.reshape(-1, heads + 2 * kv, dim)[:, heads + kv:], v, vs)):
        scales, back = scales.to(F64), []
        for b in range(case["seqs"]):
            at = slots[b * per: (b + 1) * per].tolist()
            i = 0
            while i < per:
                first, n = at[i] % page, min(per - i, page - at[i] % page)
                values, new = _exact_page(codes[at[i] // page].to(F64), scales[at[i] // page], x[b * per + i: b * per + i + n], first)
                scales[at[i] // page] = new
                back.append(values.transpose(0, 1))
                i += n
        sides.append((torch.cat(back), scales))
    return [turned[:, :heads].contiguous(), sides[0][0], sides[1][0], sides[0][1], sides[1][1]]


def _exact_attend(case, seed):
    q, k, v, ks, vs, table, start, lens = _attend_inputs(case, seed)
    page, rep = case["page"], case["heads"] // case["kv"]
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    for b, (lo, hi, n) in enumerate(zip(start[:-1].tolist(), start[1:].tolist(), lens.tolist())):
        if hi == lo:
            continue
        own_pages = table[b, : -(-n // page)].long()
        for g in range(case["kv"]):
            keys, values = ((c[own_pages, g].to(F64) * sc[own_pages, g].to(F64)[:, None, None]).reshape(-1, case["dim"])[:n] for c, sc in ((k, ks), (v, vs)))
            for h in range(g * rep, (g + 1) * rep):
                z = q[lo:hi, h].to(F64) @ keys.T * case["dim"] ** -0.5
                late = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
                out[lo:hi, h] = torch.softmax(z.masked_fill(late, -math.inf), 1) @ values
    return out


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    return None  # whole numbers
