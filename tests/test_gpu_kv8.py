"""The paged 8-bit cache on the GPU: page plan, writer and reader, attention -- against loops and 64-bit sums."""
import math

import pytest
import torch

from qspec_b200 import _lib, ops

pytestmark = pytest.mark.gpu
I32, F32, F64 = torch.int32, torch.float32, torch.float64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.as_tensor(x, dtype=I32).cuda()


# ---- the page plan ------------------------------------------------------------------------------------------------------------------
def plan_by_hand(lengths, counts, table, free, held, n_free, P, T):
    """The plan of a step, request by request."""
    B, W = len(lengths), len(table[0])
    stack = list(free[:n_free])
    for b in range(B):
        if counts[b] < 0:
            stack += table[b][:held[b]]
    have, asked, start = len(stack), 0, 0
    table, held_out, taken = [list(r) for r in table], [], 0
    q_start, kv_len, pos, seq, slots, refused = [], [], [], [], [], 0
    for b in range(B):
        c = max(counts[b], 0)
        q_start.append(min(start, T))
        wants = -(-(lengths[b] + c) // P)
        room = c == 0 or (wants <= W and start + c <= T)
        need = max(wants - held[b], 0) if c and wants <= W else 0
        asked += need
        granted = counts[b] >= 0 and room and (need == 0 or asked <= have)
        if granted:
            for i in range(need):
                table[b][held[b] + i] = stack[have - 1 - taken]
                taken += 1
        refused += counts[b] >= 0 and not granted
        held_out.append(0 if counts[b] < 0 else held[b] + (need if granted else 0))
        kv_len.append(lengths[b] + c if granted else 0)
        for i in range(c):
            if start + i < T:
                p = lengths[b] + i
                pos.append(p if granted else -1)
                seq.append(b)
                slots.append(table[b][p // P] * P + p % P if granted else -1)
        start += c
    q_start.append(min(start, T))
    pad = T - len(pos)
    left = have - taken
    free = list(free)
    for i in range(n_free, left):
        free[i] = stack[i]
    return q_start, kv_len, pos + [-1] * pad, seq + [-1] * pad, slots + [-1] * pad, held_out + [left, refused], table, free


def run_plan(lengths, counts, table, free, held, n_free, P, T):
    B = len(lengths)
    state = i32(list(held) + [n_free])
    t, f = i32(table), i32(free)
    out = [torch.full((n,), -7, dtype=I32, device="cuda") for n in (B + 1, B, T, T, T, B + 2)]
    kept = state.clone()
    ops.page_plan(i32(lengths), i32(counts), t, f, state, P, out[0], out[1], out[2], out[3], out[4], out[5])
    assert torch.equal(state, kept)
    return [o.tolist() for o in out] + [t.tolist(), f.tolist()]


def random_plan(B, P, seed, scarce, W=40, extra_T=3, most=5):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    lengths = [r(0, (W - 2) * P) for _ in range(B)]
    counts = [[-1, 0, 1, r(1, most), r(1, 2 * P)][r(0, 4)] for _ in range(B)]
    held = [min(-(-n // P) + r(0, 1), W) for n in lengths]
    pages = torch.randperm(sum(held) + B + 3 + r(0, 2 * B), generator=g).tolist()
    table, at = [], 0
    for b in range(B):
        table.append(pages[at:at + held[b]] + [0] * (W - held[b]))
        at += held[b]
    n_free = min(B // 3 if scarce else len(pages) - at, len(pages) - at)
    free = pages[at:at + n_free] + [0] * (len(pages) - n_free)
    return lengths, counts, table, free, held, n_free, P, sum(max(c, 0) for c in counts) + extra_T


@pytest.mark.parametrize("B,P,scarce", [(1, 16, False), (2, 64, True), (31, 32, False), (33, 128, True), (64, 64, True), (500, 16, True), (1025, 16, False), (4096, 32, True)])
def test_page_plan_is_the_plan_made_by_hand(B, P, scarce):
    for seed in range(3):
        case = random_plan(B, P, seed, scarce)
        assert run_plan(*case) == list(plan_by_hand(*case))


def test_page_plan_again_gives_the_same_and_steps_follow_each_other():
    lengths, counts, table, free, held, n_free, P, T = random_plan(40, 16, 5, False)
    first = run_plan(lengths, counts, table, free, held, n_free, P, T)
    again = run_plan(lengths, counts, first[6], first[7], held, n_free, P, T)
    assert first == again                                     # what a plan writes does not belong to the state it came from
    for step in range(6):                                     # every page is in one place, step after step
        q_start, kv_len, pos, seq, slots, state, table, free = run_plan(lengths, counts, table, free, held, n_free, P, T)
        held, n_free = state[:-2], state[-2]
        at = [p for b in range(len(held)) for p in table[b][:held[b]]] + free[:n_free]
        assert len(set(at)) == len(at) and set(at) <= set(range(len(free))) and state[-1] == 0
        assert all(s == table[b][p // P] * P + p % P for p, b, s in zip(pos, seq, slots) if p >= 0)
        lengths = [k if c >= 0 else 0 for k, c in zip(kv_len, counts)]
        counts = [(3 * b + step) % 4 - (1 if (b + step) % 7 == 0 else 0) if n < 30 * P else -1 for b, n in enumerate(lengths)]
        T = sum(max(c, 0) for c in counts) + 2


def test_page_plan_refuses_what_does_not_fit():
    # the row of the table, the step's tokens, the free pages -- and the next requests are served where they can be
    case = ([60, 5, 0, 8], [10, 3, 4, 0], [[0, 1, 2, 3], [4, 0, 0, 0], [0] * 4, [5, 0, 0, 0]], [6, 7, 8, 9, 0, 0, 0, 0, 0, 0], [4, 1, 0, 1], 4, 16, 40)
    got = run_plan(*case)
    assert got == list(plan_by_hand(*case)) and got[5][-1] == 1 and got[1] == [0, 8, 4, 8]
    case = case[:-1] + (14,)                                  # the third request's tokens do not fit into the step
    got = run_plan(*case)
    assert got == list(plan_by_hand(*case)) and got[5][-1] == 2 and got[0] == [0, 10, 13, 14, 14]
    case = ([15, 0], [1, 40], [[0, 0, 0], [0, 0, 0]], [1, 2, 3], [1, 0], 2, 16, 41)
    got = run_plan(*case)
    assert got == list(plan_by_hand(*case)) and got[5] == [1, 0, 2, 1]


# ---- the writer and the reader ------------------------------------------------------------------------------------------------------
def rotated(x, cs, dtype):
    a, b = x.chunk(2, -1)
    cos, sin = cs[:, None].to(dtype).chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def write_by_hand(x, slots, codes, scales, dtype=F32):
    """Rows x [T, G, D] into a copy of codes / scales, one run of a page after the other, in `dtype`."""
    codes, scales, P = codes.clone(), scales.clone(), codes.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % P:
            n += 1
        page, first = slots[t] // P, slots[t] % P
        rows = x[t:t + n].to(dtype)
        amax = torch.where(rows.abs() < math.inf, rows.abs(), 0.0).amax((0, 2))
        before = scales[page].to(dtype) if first else torch.zeros_like(amax)
        after = torch.maximum(torch.maximum(amax * torch.tensor(1.0 / 127.0, dtype=dtype, device=x.device), before), torch.tensor(2.0 ** -60, dtype=dtype, device=x.device))
        if first:
            codes[page, :, :first] = (codes[page, :, :first].to(dtype) * (before / after)[:, None, None]).round().to(torch.int8)
        q = (rows * after.reciprocal()[None, :, None]).round().clamp(-127, 127)
        codes[page, :, first:first + n] = torch.where(rows == rows, q, 0.0).to(torch.int8).transpose(0, 1)
        scales[page] = after.to(scales.dtype)
        t += n
    return codes, scales


def make_append(seed, runs, H, G, D, P, dtype, pages=40, spoil=False):
    """runs: (first position, tokens) of each request; pages are handed out at random."""
    g = gen(seed)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    pos, slots = [], []
    for first, n in runs:
        table = [order.pop() for _ in range(-(-(first + n) // P) - first // P)]
        for p in range(first, first + n):
            pos.append(p)
            slots.append(table[p // P - first // P] * P + p % P)
    T = len(pos)
    qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device="cuda").to(dtype)
    if spoil:
        qkv.view(-1)[::997] = math.inf
        qkv.view(-1)[5::1499] = -math.inf
        qkv.view(-1)[7::1201] = math.nan
    angle = torch.rand(max(pos) + 1, D // 2, generator=g, device="cuda") * 6.28
    cs = torch.cat((angle.cos(), angle.sin()), -1).to(dtype)
    codes = [torch.randint(-127, 128, (pages, G, P, D), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
    scales = [2.0 ** (torch.rand(pages, G, generator=g, device="cuda") * 4 - 7.5) for _ in range(2)]
    return qkv, cs, pos, slots, codes, scales


RUNS = {"one": [(0, 1)], "decode": [(5, 1), (63, 1), (64, 1), (200, 1)], "verify": [(62, 4), (15, 5), (0, 3), (31, 4), (127, 2)], "prompts": [(0, 300), (100, 70), (17, 1), (48, 16)]}


@pytest.mark.parametrize("D,P,H,G,dtype", [(128, 64, 8, 2, torch.float16), (128, 16, 4, 4, torch.bfloat16), (64, 32, 5, 1, torch.float16), (64, 128, 6, 3, torch.bfloat16)])
@pytest.mark.parametrize("runs", list(RUNS))
@pytest.mark.parametrize("spoil", [False, True])
def test_append_gives_the_codes_of_its_formulas(runs, D, P, H, G, dtype, spoil):
    check_append(RUNS[runs], D, P, H, G, dtype, spoil)


@pytest.mark.parametrize("D,P,H,G,dtype", [(128, 64, 8, 2, torch.float16), (128, 16, 4, 4, torch.bfloat16), (64, 32, 5, 1, torch.float16), (64, 128, 6, 3, torch.bfloat16),
                                           (128, 128, 10, 2, torch.float16)])
@pytest.mark.parametrize("runs", [[(0, 513)], [(100, 500), (0, 1), (130, 63), (7, 1), (8, 1), (77, 300), (63, 2)]])
def test_append_of_long_steps(runs, D, P, H, G, dtype):
    check_append(runs, D, P, H, G, dtype, False, 90)


@pytest.mark.parametrize("D,P,H,G,dtype", [(128, 64, 8, 2, torch.float16), (64, 16, 6, 3, torch.bfloat16), (128, 16, 1, 1, torch.float16), (64, 32, 37, 1, torch.float16)])
@pytest.mark.parametrize("runs", [[(60 + i, 1) for i in range(70)], [(i * 7, 1 + i % 11) for i in range(30)], [(3, 8), (64, 9), (1, 7), (0, 40), (5, 1), (6, 1), (16, 17), (8, 8)] * 4,
                                  [(i, 1) for i in range(1030)], [(i % 50, 2 + 17 * (i % 2)) for i in range(60)]])
@pytest.mark.parametrize("spoil", [False, True])
def test_append_of_runs_of_every_length_next_to_each_other(runs, D, P, H, G, dtype, spoil):
    check_append(runs, D, P, H, G, dtype, spoil, 1100)


def check_append(runs, D, P, H, G, dtype, spoil, pages=40):
    qkv, cs, pos, slots, codes, scales = make_append(3, runs, H, G, D, P, dtype, pages=pages, spoil=spoil)
    T = len(pos)
    x = qkv.float().view(T, H + 2 * G, D)
    turned = rotated(x[:, :H + G], cs[torch.tensor(pos, device="cuda")].float(), F32)
    want = [write_by_hand(y, slots, c, s) for y, c, s in ((turned[:, H:], codes[0], scales[0]), (x[:, H + G:], codes[1], scales[1]))]
    k, v, ks, vs = codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone()
    q = torch.empty(T, H, D, dtype=dtype, device="cuda")
    kept = qkv.clone()
    ops.kv8_append(qkv, cs, i32(pos), i32(slots), k, v, ks, vs, q)
    assert torch.equal(qkv.nan_to_num(), kept.nan_to_num())
    torch.testing.assert_close(q, turned[:, :H].to(dtype), rtol=0, atol=0, equal_nan=True)
    # float32 formulas, each operation rounded: the same bits (rows behind a page's last are no one's)
    assert torch.equal(ks, want[0][1]) and torch.equal(vs, want[1][1])
    assert torch.equal(k, want[0][0]) and torch.equal(v, want[1][0])
    # the reader: code times scale, rounded once; none for slots outside
    asked = slots + [-1, pages * P]
    ko, vo = (torch.empty(len(asked), G, D, dtype=dtype, device="cuda") for _ in range(2))
    ops.kv8_read(k, v, ks, vs, i32(asked), ko, vo)
    at = torch.tensor(slots, device="cuda")
    for got, c, s in ((ko, k, ks), (vo, v, vs)):
        assert torch.equal(got[:T], (c[at // P, :, at % P].float() * s[at // P][:, :, None]).to(dtype)) and not got[T:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_the_cache_holds_is_near_what_was_written(dtype):
    """Against 64 bits: a code is off by half a step of the scale it was made with (and the rounding of x / scale: 127 * 2^-22 of a step at most), and by
    half a step more each time that the page's scale has grown since."""
    H, G, D, P, n = 2, 2, 128, 32, 75
    g = gen(8)
    qkv = (torch.randn(n, (H + 2 * G) * D, generator=g, device="cuda") * torch.linspace(0.2, 3, n, device="cuda")[:, None]).to(dtype)
    angle = torch.rand(n, D // 2, generator=g, device="cuda")
    cs = torch.cat((angle.cos(), angle.sin()), -1).to(dtype)
    k, v = (torch.zeros(4, G, P, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(4, G, device="cuda") for _ in range(2))
    grown = torch.zeros(4, G, 2, device="cuda")
    begin = 0
    while begin < n:                                          # 1, 2, 3, 1, 2, .. tokens at a time
        m = min(begin % 3 + 1, n - begin)
        was = torch.stack([ks, vs], -1)
        pos = torch.arange(begin, begin + m)
        ops.kv8_append(qkv[begin:begin + m], cs, i32(pos), i32(pos), k, v, ks, vs, None)
        grown += (torch.stack([ks, vs], -1) > was).float()
        begin += m
    x = qkv.to(F64).view(n, H + 2 * G, D)
    want = [rotated(x[:, H:H + G], cs.to(F64), F64), x[:, H + G:]]
    for i, (c, s) in enumerate(((k, ks), (v, vs))):
        at = torch.arange(n, device="cuda")
        got = c[at // P, :, at % P].to(F64) * s[at // P][:, :, None].to(F64)
        step = s[at // P][:, :, None].to(F64)
        often = grown[at // P][:, :, i, None].to(F64)
        # (rotation in float32: three roundings of values up to |a| + |b| <= 2 * 127 steps)
        assert ((got - want[i]).abs() <= step * (0.5 * often + 127 * 2.0 ** -22 + 4 * 127 * 3 * 2.0 ** -24)).all()


def test_append_skips_tokens_without_a_place_and_leaves_the_rest():
    H, G, D, P = 4, 2, 128, 32
    qkv, cs, pos, slots, codes, scales = make_append(4, [(10, 4), (40, 3)], H, G, D, P, torch.float16)
    pos2, slots2 = list(pos), list(slots)
    slots2[3] = -1                                            # no slot (the last of its run: a page's tokens are neighbours, in consecutive rows)
    pos2[4] = len(cs)                                         # a position that the table of angles does not have
    slots2[6] = 40 * P                                        # a slot behind the cache
    k, v, ks, vs = codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone()
    q = torch.full((7, H, D), 9.0, dtype=torch.float16, device="cuda")
    ops.kv8_append(qkv, cs, i32(pos2), i32(slots2), k, v, ks, vs, q)
    assert (q[4] == 9).all() and not (q[3] == 9).all()        # (queries go by their position alone)
    gone = [s if i not in (3, 4, 6) else -1 for i, s in enumerate(slots)]
    x = qkv.float().view(7, H + 2 * G, D)
    want = write_by_hand(x[:, H + G:], gone, codes[1], scales[1])
    assert torch.equal(v, want[0]) and torch.equal(vs, want[1])


def test_append_of_strided_rows_and_an_empty_step():
    H, G, D, P = 4, 2, 64, 16
    qkv, cs, pos, slots, codes, scales = make_append(6, [(3, 20)], H, G, D, P, torch.float16)
    outs = []
    for rows in (qkv, torch.cat([qkv, qkv], 1)[:, :qkv.shape[1]]):
        c = [x.clone() for x in (*codes, *scales)]
        q = torch.empty(20, 2 * H, D, dtype=torch.float16, device="cuda")[:, :H]
        ops.kv8_append(rows, cs, i32(pos), i32(slots), *c, q)
        outs.append((*c, q.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    c = [x.clone() for x in (*codes, *scales)]
    ops.kv8_append(qkv[:0], cs, i32([]), i32([]), *c, None)
    assert all(torch.equal(a, b) for a, b in zip(c, (*codes, *scales)))


# ---- attention ----------------------------------------------------------------------------------------------------------------------
def make_attention(seed, lens, counts, H, G, D, P, dtype, spread=1.0, q_scale=1.5):
    """Requests that hold `lens` tokens, `counts` of them new; random pages, garbage in the rows and pages behind them."""
    g = gen(seed)
    need = [-(-n // P) for n in lens]
    order = torch.randperm(sum(need) + 4, generator=torch.Generator().manual_seed(seed)).tolist()
    W = max(need + [1]) + 1
    table = [[order.pop() for _ in range(n)] + [-5] * (W - n) for n in need]
    pages = sum(need) + 4
    k, v = ((torch.randn(pages, G, P, D, generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
    ks, vs = (2.0 ** (spread * (torch.rand(pages, G, generator=g, device="cuda") * 2 - 1)) / 40 for _ in range(2))
    q = (q_scale * torch.randn(sum(counts), H, D, generator=g, device="cuda")).to(dtype)
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    return q, k, v, ks, vs, i32(table), i32(start), i32(lens)


def attention_in_64_bits(q, k, v, ks, vs, table, start, lens, scale):
    """(result, bound): how far float32 scores, float16 weights and the result's rounding may take it.
    Weights are rounded to float16: 2^-11 relative, or 2^-25 absolute where the largest weight * value scale of a row is 1 (below float16's
    normal range). A score is a sum of D exact products in float32 (at most 2^-23 of the sum of their sizes for each addition in the tensor cores,
    which cut), times factors (3 roundings), and enters the exponential, whose own error and that of log2 of the scale are below 2^-20; sums of
    values and weights in float32 add 2^-23 a key at most. Codes c of keys enter the products as c + 128, and the 128 is taken out by where a sum begins:
    D / 8 products of 16 terms, no partial sum of which is above 255 sum |q| (in units of the key's scale), each term cut at 2^-24 of that."""
    T, H, D = q.shape
    P, G = k.shape[2], k.shape[1]
    rep = H // G
    out, bound = torch.zeros(T, H, D, dtype=F64, device="cuda"), torch.zeros(T, H, D, dtype=F64, device="cuda")
    for b, n in enumerate(lens.tolist()):
        lo, hi = int(start[b]), int(start[b + 1])
        if hi == lo or n == 0:
            continue
        at = table[b, :-(-n // P)].long()
        for g in range(G):
            kk, vv = (c[at, g].to(F64).reshape(-1, D)[:n] for c in (k, v))
            fk, fv = (s[at, g].to(F64).repeat_interleave(P)[:n] for s in (ks, vs))
            kk, vv = kk * fk[:, None], vv * fv[:, None]
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
            for h in range(g * rep, (g + 1) * rep):
                x = q[lo:hi, h].to(F64)
                s = (x @ kk.T * scale).masked_fill(hidden, -math.inf)
                some = ~hidden.all(1)
                w = torch.exp(s - s.amax(1, keepdim=True).nan_to_num(neginf=0.0))
                total = w.sum(1, keepdim=True)
                o = w @ vv / total.clamp(min=1e-300)
                size = w @ vv.abs() / total.clamp(min=1e-300)
                carried = x.abs().sum(1, keepdim=True) * 255 * fk[None] * (D // 8 * 17 * 2.0 ** -24)
                ds = (((x.abs() @ kk.abs().T) * ((D + 4) * 2.0 ** -23) + carried) * scale + 2.0 ** -20).masked_fill(hidden, 0.0).amax(1, keepdim=True)
                top = (w * fv[None]).amax(1, keepdim=True)
                small = n * 2.0 ** -25 * 127 * top / total.clamp(min=1e-300)
                out[lo:hi, h] = torch.where(some[:, None], o, 0.0)
                bound[lo:hi, h] = size * (2.0 ** -11 + 2 * ds + n * 2.0 ** -23) + small
    return out, bound + (out.abs() + bound) * (torch.finfo(q.dtype).eps / 2) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)


def check_attention(case, D, max_tokens=None, workspace=None):
    q, k, v, ks, vs, table, start, lens = case
    scale = D ** -0.5
    out = torch.full_like(q, 3.0)
    work = ops.kv8_attention_workspace("cuda") if workspace is None else workspace
    for _ in range(2):                                        # the workspace is left as the next call needs it
        ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, scale, work, max_tokens=max_tokens)
    want, bound = attention_in_64_bits(q, k, v, ks, vs, table, start, lens, scale)
    rows = int(start[-1])
    off = (out[:rows].to(F64) - want[:rows]).abs()
    assert torch.isfinite(out[:rows]).all()
    assert (off <= bound[:rows]).all(), float((off / bound[:rows].clamp(min=1e-30)).max())
    assert (out[rows:] == 3.0).all()
    return out


@pytest.mark.parametrize("H,G,D,dtype", [(32, 8, 128, torch.float16), (8, 8, 128, torch.bfloat16), (40, 8, 128, torch.float16), (16, 2, 64, torch.bfloat16), (7, 1, 64, torch.float16)])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_attention_of_decoding_requests(H, G, D, dtype, P):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000]
    check_attention(make_attention(1, lens, [1] * len(lens), H, G, D, P, dtype), D, max_tokens=1)


@pytest.mark.parametrize("H,G,D,P,dtype", [(32, 8, 128, 64, torch.float16), (64, 8, 128, 16, torch.bfloat16), (40, 8, 128, 32, torch.bfloat16), (16, 16, 64, 128, torch.float16)])
def test_attention_of_several_tokens_a_request(H, G, D, P, dtype):
    lens = [4, 5, 64, 66, 700, 333, 129, 3]
    counts = [4, 3, 4, 5, 1, 0, 2, 3]
    check_attention(make_attention(2, lens, counts, H, G, D, P, dtype), D, max_tokens=5)


@pytest.mark.parametrize("lens,counts", [([3000], [1]), ([20000, 3], [2, 1]), ([70] * 300, [1] * 300), ([1] * 64, [1] * 64)])
def test_attention_over_stretches_of_every_kind(lens, counts):
    check_attention(make_attention(3, lens, counts, 8, 2, 128, 64, torch.float16), 128)


@pytest.mark.parametrize("H,G,D,P,dtype", [(32, 8, 128, 64, torch.float16), (8, 1, 128, 16, torch.bfloat16), (12, 4, 128, 128, torch.float16), (4, 2, 64, 32, torch.bfloat16),
                                           (40, 8, 128, 32, torch.bfloat16)])
@pytest.mark.parametrize("lens,counts", [([17], [17]), ([200], [200]), ([130, 400, 65, 300], [130, 100, 1, 300]), ([257, 9, 1000], [33, 4, 129])])
def test_attention_of_prompts(H, G, D, P, dtype, lens, counts):
    check_attention(make_attention(4, lens, counts, H, G, D, P, dtype), D)


def test_attention_rows_that_see_nothing_and_rows_of_no_request():
    q, k, v, ks, vs, table, start, lens = make_attention(5, [0, 40, 0, 300], [2, 1, 40, 3], 8, 2, 128, 32, torch.float16)
    q = torch.cat([q, q[:9]])                                 # rows behind the last request
    out = check_attention((q, k, v, ks, vs, table, start, lens), 128)
    assert not out[:2].any() and not out[3:43].any() and out[2].any()


@pytest.mark.parametrize("counts", [[1, 4, 2], [150, 4, 60]])
def test_attention_with_scales_far_apart(counts):
    """Pages whose scales differ by 2^20: the weights' common factor takes the value scale in, and no page loses its part of the sum."""
    q, k, v, ks, vs, table, start, lens = make_attention(6, [500, 200, 900], counts, 8, 2, 128, 16, torch.bfloat16, spread=0.5)
    vs.mul_(2.0 ** torch.randint(-20, 1, vs.shape, device="cuda", generator=gen(2)))
    vs[::7] = 2.0 ** -60
    check_attention((q, k, v, ks, vs, table, start, lens), 128)


@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e30])
def test_attention_of_queries_of_any_size(q_scale):
    case = make_attention(7, [100, 70], [2, 30], 4, 2, 128, 32, torch.bfloat16, q_scale=q_scale)
    if q_scale > 1:                                           # one key takes all: its value, rounded
        q, k, v, ks, vs, table, start, lens = case
        out = torch.empty_like(q)
        ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
        want, _ = attention_in_64_bits(q, k, v, ks, vs, table, start, lens, 128 ** -0.5)
        torch.testing.assert_close(out.to(F64), want, rtol=2.0 ** -8 + 2.0 ** -10, atol=1e-30)
    else:
        check_attention(case, 128)


@pytest.mark.parametrize("counts", [[1, 2, 1], [40, 2, 70]])
def test_attention_shows_what_is_broken_and_only_there(counts):
    """A query that is not a number, and a table entry outside the cache, make the rows that have to do with them NaN, and no others."""
    q, k, v, ks, vs, table, start, lens = make_attention(8, [90, 200, 150], counts, 8, 2, 128, 64, torch.float16)
    clean = check_attention((q, k, v, ks, vs, table, start, lens), 128)
    q2 = q.clone()
    q2[0, 3, 5] = math.nan
    table2 = table.clone()
    table2[2, 1] = 10 ** 6
    out = torch.empty_like(q)
    ops.kv8_attention(q2, k, v, ks, vs, table2, start, lens, out, 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 3] = True
    first = int(lens[2]) - counts[2]
    for i in range(counts[2]):
        bad[int(start[2]) + i] = first + i >= 64
    assert out.isnan().all(2).equal(bad) and out.isnan().any(2).equal(bad)
    assert torch.equal(out[~bad], clean[~bad])


def test_attention_of_strided_queries_and_outputs():
    q, k, v, ks, vs, table, start, lens = make_attention(9, [90, 200, 300], [1, 2, 40], 8, 2, 128, 64, torch.float16)
    want = check_attention((q, k, v, ks, vs, table, start, lens), 128)
    wide = torch.randn(43, 12, 160, device="cuda").half()
    wide[:, 2:10, 16:144] = q
    out = torch.full((43, 9, 136), 5.0, dtype=torch.float16, device="cuda")
    ops.kv8_attention(wide[:, 2:10, 16:144], k, v, ks, vs, table, start, lens, out[:, 1:, :128], 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
    assert torch.equal(out[:, 1:, :128], want) and (out[:, 0] == 5).all() and (out[:, :, 128:] == 5).all()


def test_attention_is_the_same_every_time_and_in_a_graph():
    case = make_attention(10, [5000, 333, 64, 1800], [4, 4, 1, 2], 32, 8, 128, 64, torch.float16)
    q, k, v, ks, vs, table, start, lens = case
    work = ops.kv8_attention_workspace("cuda")
    want = check_attention(case, 128, workspace=work)
    out = torch.empty_like(q)
    ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, 128 ** -0.5, work)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, 128 ** -0.5, work)
    for _ in range(20):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    lens.copy_(i32([4000, 500, 60, 65]))                      # other lengths, the same graph
    graph.replay()
    want, bound = attention_in_64_bits(q, k, v, ks, vs, table.clamp(min=0), start, lens, 128 ** -0.5)
    keep = torch.ones(len(q), dtype=torch.bool, device="cuda")
    keep[4:8] = False                                         # (the second request has no pages for 500 tokens)
    assert ((out.to(F64) - want).abs() <= bound)[keep].all()


def test_two_streams_with_a_workspace_each():
    cases = [make_attention(s, [9000, 700], [1, 2], 16, 4, 128, 64, torch.float16) for s in (11, 12)]
    want = [check_attention(c, 128) for c in cases]
    streams, works = [torch.cuda.Stream() for _ in cases], [ops.kv8_attention_workspace("cuda") for _ in cases]
    outs = [torch.empty_like(c[0]) for c in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, w, o in zip(cases, streams, works, outs):
            with torch.cuda.stream(s):
                ops.kv8_attention(*c, o, 128 ** -0.5, w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


# ---- refusals that need tensors on the GPU -------------------------------------------------------------------------------------------
def test_wrong_shapes_types_and_overlaps_are_refused():
    z = lambda *s, dtype=I32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    args = [z(2), z(2), z(2, 4), z(8), z(3), 16, z(3), z(2), z(5), z(5), z(5), z(4)]
    for i, bad in ((0, z(2, 1)), (1, z(3)), (4, z(2)), (6, z(2)), (9, z(4)), (11, z(3)), (2, z(4, 2).t()), (0, z(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            ops.page_plan(*[bad if j == i else a for j, a in enumerate(args)])
    both = z(6)
    with pytest.raises(ValueError, match="must not lie over"):
        ops.page_plan(*[both[:3] if j == 4 else both[2:] if j == 11 else a for j, a in enumerate(args)])
    cache = [z(3, 2, 16, 64, dtype=torch.int8), z(3, 2, 16, 64, dtype=torch.int8), z(3, 2, dtype=F32), z(3, 2, dtype=F32)]
    half = lambda *s: z(*s, dtype=torch.float16)  # noqa: E731
    app = [half(3, 8 * 64), half(9, 64), z(3), z(3), *cache, half(3, 4, 64)]
    for i, bad in ((0, half(3, 4 * 64)), (0, half(3, 8 * 64 + 1)), (1, z(9, 64, dtype=F32)), (1, half(9, 32)), (2, z(4)), (3, z(3, dtype=torch.int64)), (5, cache[0][:2]),
                   (6, z(3, dtype=F32)), (8, half(3, 3, 64)), (8, half(4, 3, 64).transpose(0, 1)), (4, cache[0].view(torch.uint8))):
        with pytest.raises(ValueError):
            ops.kv8_append(*[bad if j == i else a for j, a in enumerate(app)])
    att = [half(3, 4, 64), *cache, z(2, 4), z(3), z(2), half(3, 4, 64), 0.1, ops.kv8_attention_workspace("cuda")]
    for i, bad in ((0, z(3, 4, 64, dtype=F32)), (0, half(3, 4, 32)), (5, z(8)), (6, z(2)), (7, z(3)), (8, half(3, 4, 64).bfloat16()), (8, half(2, 4, 64)), (9, 0.0), (9, math.nan),
                   (10, z(9, dtype=F32)), (0, half(3, 5, 64)), (10, z(100, dtype=torch.uint8))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv8_attention(*[bad if j == i else a for j, a in enumerate(att)])
    with pytest.raises(ValueError):
        ops.kv8_read(*cache, z(3), half(3, 2, 64), half(2, 2, 64))


@pytest.mark.parametrize("counts", [[1, 2], [1, 90]])
def test_attention_of_tiny_queries_over_tiny_scales(counts):
    """Factors of scores below float32's normal range must not turn a hidden key's minus infinity into no number."""
    q, k, v, ks, vs, table, start, lens = make_attention(13, [70, 200], counts, 4, 2, 128, 32, torch.bfloat16, q_scale=1e-30)
    ks.fill_(2.0 ** -60)
    check_attention((q, k, v, ks, vs, table, start, lens), 128)


GIVE_UP = r"""
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from test_gpu_kv8 import make_attention, attention_in_64_bits
from qspec_b200 import _lib, ops
lib = _lib.load()
for D, dtype in ((128, torch.float16), (64, torch.bfloat16)):
    q, k, v, ks, vs, table, start, lens = make_attention(3, [500, 900, 40], [130, 300, 1], 8, 2, D, 32, dtype)
    work = ops.kv8_attention_workspace("cuda")
    good = ops.kv8_attention(q, k, v, ks, vs, table, start, lens, torch.empty_like(q), D ** -0.5, work)
    for roles in (1, 2, 4, 8, 15, 17, 18, 20, 24, 31):
        before, out = ops.attn_tile_timeouts(), torch.zeros_like(q)
        _lib.check(lib.qspec_debug_kv8_attention_give_up(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(),
                                                         start.data_ptr(), lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), len(q), 3, table.shape[1], 8, 2, D, k.shape[0],
                                                         32, 300, D ** -0.5, int(dtype == torch.bfloat16), work.data_ptr(), work.numel(), roles,
                                                         torch.cuda.current_stream().cuda_stream), "give up")
        assert ops.attn_tile_timeouts() > before, roles
        assert out[:430].isnan().all() and torch.equal(out[430:], good[430:]), roles   # the request with few rows is the other form's
        again = ops.kv8_attention(q, k, v, ks, vs, table, start, lens, torch.empty_like(q), D ** -0.5, work)
        assert torch.equal(again, good) and ops.attn_tile_timeouts() > before
print("ok")
"""


def test_a_wait_that_is_given_up_shows_and_leaves_nothing_behind():
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", GIVE_UP.format(root=os.path.dirname(tests), tests=tests)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


# ---- the prompt form at sizes at which a call would not choose it ---------------------------------------------------------------------
def prompt_form(q, k, v, ks, vs, table, start, lens, out, scale, work, max_tokens=None, pairs=False):
    lib, T, H, D = _lib.load(), q.shape[0], q.shape[1], q.shape[2]
    _lib.check(lib.qspec_debug_kv8_attention_give_up(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(),
                                                     start.data_ptr(), lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), T, len(lens), table.shape[1], H, k.shape[1], D,
                                                     k.shape[0], k.shape[2], T if max_tokens is None else max_tokens, scale, int(q.dtype == torch.bfloat16), work.data_ptr(),
                                                     work.numel(), 16 * pairs, torch.cuda.current_stream().cuda_stream), "kv8_attention")
    return out


FORCED = ([(test_attention_of_prompts, h + (lens, counts)) for h in ((32, 8, 128, 64, torch.float16), (8, 1, 128, 16, torch.bfloat16), (12, 4, 128, 128, torch.float16),
                                                                     (4, 2, 64, 32, torch.bfloat16), (40, 8, 128, 32, torch.bfloat16), (128, 1, 64, 64, torch.float16))
           for lens, counts in (([17], [17]), ([200], [200]), ([130, 400, 65, 300], [130, 100, 1, 300]), ([257, 9, 1000], [33, 4, 129]))]
          + [(test_attention_rows_that_see_nothing_and_rows_of_no_request, ()), (test_attention_with_scales_far_apart, ([150, 4, 60],)),
             (test_attention_of_queries_of_any_size, (0.0,)), (test_attention_of_queries_of_any_size, (1e-30,)), (test_attention_of_queries_of_any_size, (1e30,)),
             (test_attention_shows_what_is_broken_and_only_there, ([40, 2, 70],)), (test_attention_of_strided_queries_and_outputs, ()),
             (test_attention_of_tiny_queries_over_tiny_scales, ([1, 90],))])


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("at", range(len(FORCED)))
def test_prompt_form_of_small_calls(monkeypatch, at, pairs):
    monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=pairs, **kw))
    test, args = FORCED[at]
    test(*args)


# ---- which form a request goes to -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,counts", [([400, 2000, 130], [300, 20, 70]),       # long: its way through its keys is longer than the others', so not the prompt form
                                         ([9000, 64, 900, 5000], [65, 64, 512, 16]), ([300] * 40 + [7] * 200, [20] * 40 + [1] * 200)])
@pytest.mark.parametrize("H,G", [(32, 8), (10, 2), (5, 5)])
def test_attention_of_requests_that_take_different_forms(H, G, lens, counts):
    check_attention(make_attention(14, lens, counts, H, G, 128, 64, torch.float16), 128)


def test_the_form_is_the_rules_and_both_kernels_agree_on_it():
    """Rows of the prompt form and of the other one differ in their last bits: which form a request took shows in its rows."""
    lens, counts, H, G = [900, 9000, 300, 1200, 40], [200, 30, 1, 500, 24], 32, 8
    case = make_attention(15, lens, counts, H, G, 128, 64, torch.float16)
    out = check_attention(case, 128)
    work = ops.kv8_attention_workspace("cuda")
    forced = prompt_form(*case, torch.empty_like(out), 128 ** -0.5, work, pairs=sum(counts) * H > 160 * torch.cuda.get_device_properties(0).multi_processor_count)
    share = torch.cuda.get_device_properties(0).multi_processor_count // 4 * 128
    rows = [n * H // G for n in counts]
    total = sum(r * G * -(-n // 128) for r, n in zip(rows, lens) if r >= 65)
    picks = [r >= 65 and -(-n // 128) * share <= total for r, n in zip(rows, lens)]
    assert picks == [True, False, False, True, True]
    for b, pick in enumerate(picks):
        at = slice(sum(counts[:b]), sum(counts[:b + 1]))
        assert counts[b] == 1 or torch.equal(out[at], forced[at]) == pick


# ---- other calls that the documentation allows ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("pairs", [None, False, True])
@pytest.mark.parametrize("H,G", [(8, 2), (6, 2), (16, 1)])
def test_attention_of_requests_with_more_tokens_than_keys(H, G, pairs, monkeypatch):
    """The first tokens stand in front of the first key and see nothing, whole tiles of them, or of one of two tiles."""
    if pairs is not None:
        monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=pairs, **kw))
    lens, counts = [32, 40, 3, 1, 300], [64, 130, 70, 200, 310]
    case = make_attention(16, lens, counts, H, G, 128, 32, torch.float16)
    out = check_attention(case, 128)
    for at, keys, n in zip(case[6].tolist(), lens, counts):
        assert not out[at:at + n - keys].any() and out[at + n - keys].any()


@pytest.mark.parametrize("lens,counts", [([3000, 70], [2, 4]), ([400, 300], [300, 290])])
def test_attention_over_its_own_queries(lens, counts):
    case = make_attention(17, lens, counts, 32, 8, 128, 64, torch.float16)
    want = check_attention(case, 128)
    q = case[0].clone()
    ops.kv8_attention(q, *case[1:], q, 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
    assert torch.equal(q, want)


def test_append_turns_queries_in_place():
    H, G, D, P = 6, 2, 128, 16
    qkv, cs, pos, slots, codes, scales = make_append(5, [(0, 40), (30, 1), (5, 5)], H, G, D, P, torch.float16)
    results = []
    for inplace in (False, True):
        rows, k, v, ks, vs = qkv.clone(), codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone()
        q = rows[:, :H * D].unflatten(1, (H, D)) if inplace else torch.empty(len(pos), H, D, dtype=torch.float16, device="cuda")
        ops.kv8_append(rows, cs, i32(pos), i32(slots), k, v, ks, vs, q)
        assert torch.equal(rows[:, H * D:], qkv[:, H * D:])
        results.append((q.clone(), k, v, ks, vs))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_page_plan_refuses_results_over_its_other_tensors():
    z = lambda *s: torch.zeros(*s, dtype=I32, device="cuda")  # noqa: E731
    args = [z(3), z(3), z(3, 4), z(12), z(4), 16, z(4), z(3), z(5), z(5), z(5), z(5)]
    ops.page_plan(*args)
    for out, over in ((7, 1), (7, 0), (8, 9), (6, 4), (10, 3), (11, 4)):
        both = z(20)
        bad = list(args)
        bad[out], bad[over] = both[:args[out].numel()], both[1:1 + args[over].numel()]
        with pytest.raises(ValueError, match="must not lie over"):
            ops.page_plan(*bad)


# ---- a long context's many small weights ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ratio,gap", [(1, 25.05), (64, 19.1), (64, 24.0), (16, 21.1)])
def test_attention_loses_no_keys_of_a_long_context(ratio, gap, dtype, form):
    """Values that are all 1, whatever their weights: so is the result. The first key's score is above all others' by log2 = gap, and its page may have a value scale that
    is `ratio` times the others'. Off by the result's rounding; 2^-11 for a weight that is a normal float16; ratio * 2^-34 for each key whose weight is not (2^-25,
    the largest being 2^9 or more, with the value scale in it); and float32 sums: 2^-23 for every key that one accumulator takes, half of that for the denominator (the
    tensor cores cut each term of a product at the last place of the largest, which is the sum so far: terms 2^-25 of it, as in the first case, are gone one by one, not by
    sixteens). In the prompt form that is n keys, in the other a quarter: there so many requests (of the same pages) that each is one CTA's, of four warps."""
    n, G, H, D, P = 131000, 2, 8, 128, 64
    B, T = (256, 1) if form == "rows" else (1, 20) if form == "prompt" else (1, 50)
    pages = -(-n // P)
    k, v = torch.zeros(pages, G, P, D, dtype=torch.int8, device="cuda"), torch.full((pages, G, P, D), 64, dtype=torch.int8, device="cuda")
    ks, vs = torch.full((pages, G), gap / 127 / math.log2(math.e), device="cuda"), torch.full((pages, G), 1 / 64, device="cuda")
    v[0], vs[0] = 64 // ratio, ratio / 64
    k[0, :, 0, 0] = 127
    q = torch.zeros(B * T, H, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    case = (q, k, v, ks, vs, torch.arange(pages, dtype=I32, device="cuda").repeat(B, 1), i32(range(0, B * T + 1, T)), i32([n] * B))
    work, out = ops.kv8_attention_workspace("cuda"), torch.empty_like(q)
    if form == "rows":
        ops.kv8_attention(*case, out, 1.0, work, max_tokens=1)
    else:
        prompt_form(*case, out, 1.0, work, pairs=form == "pairs")
    chain = n / (4 if form == "rows" else 1)
    bound = torch.finfo(dtype).eps / 2 + 2.0 ** -11 + n * ratio * 2.0 ** -34 + chain * 1.5 * 2.0 ** -23
    assert (out.double() - 1).abs().max() <= bound, (float((out.double() - 1).abs().max()), bound)


def test_attention_of_scores_far_from_zero():
    """Exponents of 2^20 to 2^26, where a reference's own rounding is large: weights stay finite, and one key, or several that are alike, take all."""
    for form in ("rows", "prompt", "pairs"):
        n, G, D, P, T = 700, 2, 128, 32, 2 if form == "rows" else 40
        pages = -(-n // P)
        for log2 in (18, 20, 21.9, 22.1, 23, 23.9, 24.1, 25, 26):
            for sign in (1.0, -1.0):
                g = gen(int(log2 * 10))
                k = torch.zeros(pages, G, P, D, dtype=torch.int8, device="cuda")
                k[..., 0] = 100                                   # all scores alike, and far from zero
                v = (torch.randn(pages, G, P, D, generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8)
                ks, vs = torch.full((pages, G), 2.0 ** log2 / 100, device="cuda"), torch.full((pages, G), 1 / 64, device="cuda")
                q = torch.zeros(T, 8, D, dtype=torch.float16, device="cuda")
                q[:, :, 0] = sign
                case = (q, k, v, ks, vs, torch.arange(pages, dtype=I32, device="cuda")[None], i32([0, T]), i32([n]))
                work, out = ops.kv8_attention_workspace("cuda"), torch.empty_like(q)
                if form == "rows":
                    ops.kv8_attention(*case, out, 1.0, work, max_tokens=T)
                else:
                    prompt_form(*case, out, 1.0, work, pairs=form == "pairs")
                rows = v.double().permute(1, 0, 2, 3).reshape(G, -1, D) / 64
                want = torch.stack([rows[:, :n - T + 1 + t].mean(1) for t in range(T)]).repeat_interleave(4, 1)
                # equal weights: each off by 2^-11, sums by n / 16 * 2^-23, the result by its own rounding
                size = rows.abs().mean(1).amax()
                assert ((out.double() - want).abs() <= size * (2.0 ** -11 + 2.0 ** -11 + n / 16 * 2.0 ** -23) + want.abs() * 2.0 ** -11 + 2.0 ** -24).all(), (form, log2, sign)


@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
@pytest.mark.parametrize("log2", [-112, 100, 121])
def test_attention_of_queries_and_scales_that_make_up_for_each_other(log2, form, monkeypatch):
    """Tiny queries over keys of a huge scale, and the other way round: the factors of the scores meet before they leave float32."""
    if form != "rows":
        monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=form == "pairs", **kw))
    counts = [1, 3] if form == "rows" else [60, 40]
    q, k, v, ks, vs, table, start, lens = make_attention(18, [200, 333], counts, 8, 2, 128, 32, torch.bfloat16, q_scale=1.5 * 2.0 ** log2)
    ks.mul_(2.0 ** -min(log2, 93))                            # (scales below 2^-100 count as that)
    check_attention((q, k, v, ks, vs, table, start, lens), 128)


@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_rows_in_front_of_a_page_of_a_huge_scale(dtype, form, monkeypatch):
    """Scores of the last page leave float32. The rows that do not see it are what they are without it, within the bound of either of the two ways in which exponents are taken
    (one for all rows of a warp: those that see the page decide, so that the others' last bits may move)."""
    if form != "rows":
        monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=form == "pairs", **kw))
    q, k, v, ks, vs, table, start, lens = make_attention(19, [200, 333], [60, 40], 8, 2, 128, 32, dtype, q_scale=1.5 * 2.0 ** (10 if dtype == torch.float16 else 30))
    ks.mul_(2.0 ** (-10 if dtype == torch.float16 else -30))
    check_attention((q, k, v, ks, vs, table, start, lens), 128)
    want, bound = attention_in_64_bits(q, k, v, ks, vs, table, start, lens, 128 ** -0.5)
    ks[int(table[0, 6])] = ks[int(table[1, 10])] = 2.0 ** 120   # positions 192 and 320 on
    out = torch.empty_like(q)
    ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
    for rows in (slice(0, 52), slice(60, 87)):
        assert ((out[rows].to(F64) - want[rows]).abs() <= bound[rows]).all()


@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("runs", [[(3, 6), (40, 2)], [(16, 16), (0, 1), (5, 60)], [(10, 118), (250, 130), (7, 9)], [(i, 1 + i % 13) for i in range(60)]])
def test_append_leaves_out_tokens_without_a_position_in_the_middle_of_a_page(runs, P):
    """A page's tokens are one run whatever positions they have: one scale, of those that are written, from the first of these on."""
    H, G, D = 4, 2, 128
    qkv, cs, pos, slots, codes, scales = make_append(9, runs, H, G, D, P, torch.float16, pages=400)
    T = len(pos)
    left_out = torch.rand(T, generator=torch.Generator().manual_seed(T)) < 0.4
    left_out[:2] = True                                       # the first of a run among them
    given = [len(cs) + i % 5 if o and i % 2 else -1 - i % 3 if o else p for i, (p, o) in enumerate(zip(pos, left_out.tolist()))]
    x = qkv.float().view(T, H + 2 * G, D)
    turned = rotated(x[:, :H + G], cs[torch.tensor(pos, device="cuda")].float(), F32)
    k, v, ks, vs = codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone()
    q = torch.full((T, H, D), 9.0, dtype=torch.float16, device="cuda")
    ops.kv8_append(qkv, cs, i32(given), i32(slots), k, v, ks, vs, q)
    out = left_out.cuda()
    assert (q[out] == 9).all() and torch.equal(q[~out], turned[:, :H].half()[~out])
    for y, c, s, got_c, got_s in ((turned[:, H:], codes[0].clone(), scales[0].clone(), k, ks), (x[:, H + G:], codes[1].clone(), scales[1].clone(), v, vs)):
        begin = 0
        while begin < T:
            n = 1
            while begin + n < T and slots[begin + n] == slots[begin] + n and slots[begin + n] % P:
                n += 1
            some = [t for t in range(begin, begin + n) if not left_out[t]]
            begin += n
            if not some:
                continue
            page, row = slots[some[0]] // P, [slots[t] % P for t in some]
            before = s[page] if row[0] else torch.zeros_like(s[page])
            after = torch.maximum(torch.maximum(y[some].abs().amax((0, 2)) * torch.tensor(1.0 / 127.0, device="cuda"), before), torch.tensor(2.0 ** -60, device="cuda"))
            c[page, :, :row[0]] = (c[page, :, :row[0]].float() * (before / after)[:, None, None]).round().to(torch.int8)
            c[page][:, row] = (y[some] * after.reciprocal()[None, :, None]).round().clamp(-127, 127).to(torch.int8).transpose(0, 1)
            s[page] = after
        assert torch.equal(got_s, s) and torch.equal(got_c, c)


@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("side", ["keys", "values"])
def test_attention_shows_a_scale_that_is_no_number_and_only_where_it_is_seen(side, value, form, monkeypatch):
    if form != "rows":
        monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=form == "pairs", **kw))
    q, k, v, ks, vs, table, start, lens = make_attention(20, [200, 333], [60, 40], 8, 2, 128, 32, torch.float16)
    clean = check_attention((q, k, v, ks, vs, table, start, lens), 128)
    for page in (int(table[0, 5]), int(table[1, 9])):         # positions 160 .. 191 and 288 .. 319 of one head
        (ks if side == "keys" else vs)[page, 1] = value
    out = torch.empty_like(q)
    ops.kv8_attention(q, k, v, ks, vs, table, start, lens, out, 128 ** -0.5, ops.kv8_attention_workspace("cuda"))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[20:60, 4:] = True                                     # tokens at 140 .. 199
    bad[60:, 4:] = True                                       # tokens at 293 .. 332
    assert out.isnan().all(2).equal(bad) and out.isnan().any(2).equal(bad)
    assert torch.equal(out[~bad], clean[~bad])


def test_page_plan_gives_no_slot_in_what_is_no_page():
    """Entries of the table and of the list of free pages outside the cache: 2^26 pages of 64 tokens on is where a slot's number would begin again."""
    table = [[1 << 26, 3], [-1, 0], [2, 0], [0, 0]]
    free = [(1 << 26) + 1, 8, -7, 1, 5, 0, 0, 0]
    lengths, counts, held = [64, 10, 60, 0], [2, 1, 8, 1], [2, 1, 1, 0]
    got = run_plan(lengths, counts, table, free, held, 3, 64, 12)
    assert got[2] == [64, 65, 10, 60, 61, 62, 63, 64, 65, 66, 67, 0]
    assert got[4] == [3 * 64, 3 * 64 + 1, -1] + [2 * 64 + r for r in (60, 61, 62, 63)] + [-1] * 5
    lengths[0] = 10                                           # the page behind the cache
    assert run_plan(lengths, counts, table, free, held, 3, 64, 12)[4][:2] == [-1, -1]


@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
def test_attention_walks_no_further_than_the_table(form, monkeypatch):
    """Lengths beyond the table's pages, up to the largest number there is: the rows that see such keys are NaN, soon; others are what they are."""
    if form != "rows":
        monkeypatch.setattr(ops, "kv8_attention", lambda *args, **kw: prompt_form(*args, pairs=form == "pairs", **kw))
    q, k, v, ks, vs, table, start, lens = make_attention(21, [200, 256, 100], [40, 20, 40], 8, 2, 128, 32, torch.float16)
    clean = check_attention((q, k, v, ks, vs, table, start, lens), 128)
    work = ops.kv8_attention_workspace("cuda")
    short = table[:, :4].contiguous()                         # 128 keys
    for large in (129, 300, 10 ** 6, 2 ** 31 - 1):
        far = i32([large, 256, 100])
        out = ops.kv8_attention(q, k, v, ks, vs, short, start, far, torch.zeros_like(q), 128 ** -0.5, work)
        first = large - 40
        bad = [first + i >= 128 for i in range(40)] + [True] * 20 + [False] * 40
        bad = torch.tensor(bad, device="cuda")
        assert out[bad].isnan().all() and not out[~bad].isnan().any()
        assert torch.equal(out[60:], clean[60:])
