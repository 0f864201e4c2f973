"""The paged 4-bit cache on the GPU: writer and reader, attention -- against loops and 64-bit sums."""
import math

import pytest
import torch

from qspec_b200 import _lib, ops

pytestmark = pytest.mark.gpu
I16, I32, F32, F64, U8 = torch.int16, torch.int32, torch.float32, torch.float64, torch.uint8
FORMS = ["rows", "prompt", "pairs"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.as_tensor(x, dtype=I32).cuda()


# ---- the writer and the reader ------------------------------------------------------------------------------------------------------
def rotated(x, cs, dtype):
    a, b = x.chunk(2, -1)
    cos, sin = cs[:, None].to(dtype).chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def hadamard(x):
    """x H / sqrt(D): butterflies of strides 1, 2 .. D / 2 (the order in which they round)."""
    D, s = x.shape[-1], 1
    while s < D:
        a, b = x.unflatten(-1, (-1, 2, s)).unbind(-2)
        x = torch.stack((a + b, a - b), -2).flatten(-3)
        s *= 2
    return x * D ** -0.5


def scales(words):
    """(scale, zero point) of words."""
    w = words.to(I32) & 0xffff
    return ((w & 0xfff0) << 15).view(F32), (w & 15).float()


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def values(codes, words):
    s, z = scales(words)
    return (unpack(codes).double() - z.double()[..., None]) * s.double()[..., None]


def quantised(x):
    """Codes and words of rows x [.., D] in float32: the formulas, with what is not finite taken as they say."""
    finite = x.abs() < math.inf
    y = x.nan_to_num(0.0, math.inf, -math.inf).clamp(-2.0 ** 126, 2.0 ** 126)
    hi = torch.where(finite, y, 0.0).amax(-1).clamp(min=0)
    lo = torch.where(finite, y, 0.0).amin(-1).clamp(max=0)
    bits = (((hi - lo) / 15).clamp(min=2.0 ** -60).view(I32) + (1 << 18)) >> 19
    s = (bits << 19).view(F32)
    z = (-lo / s).round().clamp(0, 15)
    c = ((y / s[..., None]).round() + z[..., None]).clamp(0, 15).to(U8)
    return c[..., 0::2] | c[..., 1::2] << 4, (bits << 4 | z.to(I32)).to(I16)


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
        qkv[0] = 0.0
        qkv[-1, H * D:] = 2.0
        qkv[T // 2] = -qkv[T // 2].abs()
    angle = torch.rand(max(pos) + 1, D // 2, generator=g, device="cuda") * 6.28
    cs = torch.cat((angle.cos(), angle.sin()), -1).to(dtype)
    codes = [torch.randint(0, 256, (pages, G, P, D // 2), generator=g, device="cuda").to(U8) for _ in range(2)]
    words = [torch.randint(120 << 8, 130 << 8, (pages, G, P), generator=g, device="cuda").to(I16) for _ in range(2)]
    return qkv, cs, pos, slots, codes, words


RUNS = {"one": [(0, 1)], "decode": [(5, 1), (63, 1), (64, 1), (200, 1)], "verify": [(62, 4), (15, 5), (0, 3), (31, 4), (127, 2)], "prompts": [(0, 300), (100, 70), (17, 1), (48, 16)],
        "long": [(0, 1300)]}
SHAPES = [(128, 64, 8, 2, torch.float16), (128, 16, 4, 4, torch.bfloat16), (64, 32, 5, 1, torch.float16), (64, 128, 6, 3, torch.bfloat16), (128, 32, 37, 1, torch.bfloat16)]


@pytest.mark.parametrize("D,P,H,G,dtype", SHAPES)
@pytest.mark.parametrize("runs", list(RUNS))
@pytest.mark.parametrize("spoil", [False, True])
@pytest.mark.parametrize("turn", [False, True])
def test_append_gives_the_codes_of_its_formulas(runs, D, P, H, G, dtype, spoil, turn):
    qkv, cs, pos, slots, codes, words = make_append(3, RUNS[runs], H, G, D, P, dtype, pages=100, spoil=spoil)
    T = len(pos)
    x = qkv.float().view(T, H + 2 * G, D)
    turned = rotated(x[:, :H + G], cs[torch.tensor(pos, device="cuda")].float(), F32)
    if turn:
        turned = hadamard(turned)
    k, v, kw, vw = codes[0].clone(), codes[1].clone(), words[0].clone(), words[1].clone()
    q = torch.empty(T, H, D, dtype=dtype, device="cuda")
    kept = qkv.clone()
    ops.kv4_append(qkv, cs, i32(pos), i32(slots), k, v, kw, vw, q, hadamard=turn)
    assert torch.equal(qkv.nan_to_num(), kept.nan_to_num())
    torch.testing.assert_close(q, turned[:, :H].to(dtype), rtol=0, atol=0, equal_nan=True)
    # float32 formulas, each operation rounded: the same bits, and no other row touched
    at = torch.tensor(slots, device="cuda")
    for y, c, w, got_c, got_w in ((turned[:, H:], codes[0], words[0], k, kw), (x[:, H + G:], codes[1], words[1], v, vw)):
        c[at // P, :, at % P], w[at // P, :, at % P] = quantised(y)
        assert torch.equal(got_w, w) and torch.equal(got_c, c)
    # the reader: (code - zero point) times scale, rounded once; none for slots outside
    asked = slots + [-1, 100 * P]
    ko, vo = (torch.empty(len(asked), G, D, dtype=dtype, device="cuda") for _ in range(2))
    ops.kv4_read(k, v, kw, vw, i32(asked), ko, vo)
    for got, c, w in ((ko, k, kw), (vo, v, vw)):
        assert torch.equal(got[:T], values(c[at // P, :, at % P], w[at // P, :, at % P]).to(dtype)) and not got[T:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shift", [0.0, 3.0, -50.0])
def test_what_the_cache_holds_is_near_what_was_written(dtype, shift):
    """Against 64 bits. r = (hi - lo) / 15, and s is r (1 + d) with |d| <= 2^-5 (five significant bits). The zero point is off by half a step at most, a code by half a step, and
    where a value lies outside of the codes' range by up to (15 |d| + 1/2 + 1/2) steps beyond the last code's own half: in all 1.5 s at most there; inside of it half a step. What a
    float32 quotient of up to 16 adds is 2^-20 of a step, what the rotation and the Hadamard sums do (10 roundings of at most 12 standard deviations' sum, sqrt(128) / 128
    of it behind the factor) below 2^-15 of the largest value."""
    H, G, D, P, n = 2, 3, 128, 32, 75
    qkv = (torch.randn(n, (H + 2 * G) * D, generator=gen(8), device="cuda") * torch.linspace(0.2, 3, n, device="cuda")[:, None] + shift).to(dtype)
    angle = torch.rand(n, D // 2, generator=gen(9), device="cuda")
    cs = torch.cat((angle.cos(), angle.sin()), -1).to(dtype)
    k, v = (torch.zeros(4, G, P, D // 2, dtype=U8, device="cuda") for _ in range(2))
    kw, vw = (torch.zeros(4, G, P, dtype=I16, device="cuda") for _ in range(2))
    pos = i32(range(n))
    ops.kv4_append(qkv, cs, pos, pos, k, v, kw, vw, None, hadamard=True)
    x = qkv.to(F64).view(n, H + 2 * G, D)
    want = [hadamard(rotated(x[:, H:H + G], cs.to(F64), F64)), x[:, H + G:]]
    at = pos.long()
    for y, c, w in zip(want, (k, v), (kw, vw)):
        got = values(c[at // P, :, at % P], w[at // P, :, at % P])
        s = scales(w[at // P, :, at % P])[0].double()[..., None]
        r = ((y.amax(-1).clamp(min=0) - y.amin(-1).clamp(max=0)) / 15)[..., None]
        assert ((s / r - 1).abs() <= 2.0 ** -5 + 2.0 ** -14).all()
        code = unpack(c[at // P, :, at % P])
        inside = (code > 0) & (code < 15)
        slack = y.abs().amax(-1, keepdim=True) * 2.0 ** -15
        assert ((got - y).abs() <= s * torch.where(inside, 0.5 + 2.0 ** -20, 1.5) + slack).all()
        assert (got[y == 0] == 0).all()                       # zero is a code


def test_queries_and_keys_keep_their_products():
    """The Hadamard matrix over its square root is orthogonal: scores of turned queries and turned keys are those of the ones that were not. (All are written as queries, in
    float16: each value off by 2^-11 of itself, a product by 2^-10 of the sizes' sum, and float32's part in it below 2^-18.)"""
    H, G, D, P, n = 6, 1, 128, 64, 33
    qkv, cs, pos, slots, codes, words = make_append(5, [(7, n)], H, G, D, P, torch.float16)
    got = []
    for turn in (False, True):
        q = torch.empty(n, H, D, dtype=torch.float16, device="cuda")
        ops.kv4_append(qkv, cs, i32(pos), i32(slots), *codes, *words, q, hadamard=turn)
        got.append(q.double())
    products = [torch.einsum("thd,sgd->thsg", x[:, :4], x[:, 4:]) for x in got]
    size = sum(torch.einsum("thd,sgd->thsg", x[:, :4].abs(), x[:, 4:].abs()) for x in got)
    assert ((products[0] - products[1]).abs() <= size * (2.0 ** -10 + 2.0 ** -18)).all()


def test_append_skips_tokens_without_a_slot_or_a_position():
    H, G, D, P = 4, 2, 128, 32
    qkv, cs, pos, slots, codes, words = make_append(4, [(10, 4), (40, 3)], H, G, D, P, torch.float16)
    pos2, slots2 = list(pos), list(slots)
    slots2[2] = -1
    pos2[4], pos2[5] = len(cs), -1                            # positions that the table of angles does not have
    slots2[6] = 40 * P                                        # a slot behind the cache
    k, v, kw, vw = codes[0].clone(), codes[1].clone(), words[0].clone(), words[1].clone()
    q = torch.full((7, H, D), 9.0, dtype=torch.float16, device="cuda")
    ops.kv4_append(qkv, cs, i32(pos2), i32(slots2), k, v, kw, vw, q)
    assert (q[4:6] == 9).all() and not (q[2] == 9).all() and not (q[6] == 9).all()   # (queries go by their position alone)
    at = torch.tensor([slots[i] for i in (0, 1, 3)], device="cuda")
    c, w = codes[1], words[1]
    c[at // P, :, at % P], w[at // P, :, at % P] = quantised(qkv.float().view(7, H + 2 * G, D)[[0, 1, 3], H + G:])
    assert torch.equal(v, c) and torch.equal(vw, w)


def test_append_of_strided_rows_in_place_and_an_empty_step():
    H, G, D, P = 4, 2, 64, 16
    qkv, cs, pos, slots, codes, words = make_append(6, [(3, 20)], H, G, D, P, torch.float16)
    outs = []
    for way in range(3):
        c = [x.clone() for x in (*codes, *words)]
        rows = torch.cat([qkv, qkv], 1)[:, :qkv.shape[1]] if way == 1 else qkv.clone()
        q = rows[:, :H * D].unflatten(1, (H, D)) if way == 2 else torch.empty(20, 2 * H, D, dtype=torch.float16, device="cuda")[:, :H]
        ops.kv4_append(rows, cs, i32(pos), i32(slots), *c, q, hadamard=True)
        assert torch.equal(rows[:, H * D:], qkv[:, H * D:])
        outs.append((*c, q.clone()))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))
    c = [x.clone() for x in (*codes, *words)]
    ops.kv4_append(qkv[:0], cs, i32([]), i32([]), *c, None)
    assert all(torch.equal(a, b) for a, b in zip(c, (*codes, *words)))


# ---- attention ----------------------------------------------------------------------------------------------------------------------
def make_attention(seed, lens, counts, H, G, D, P, dtype, q_scale=1.5, spread=1.0):
    """Requests that hold `lens` tokens, `counts` of them new; random pages, garbage in the rows and pages behind them."""
    g = gen(seed)
    need = [-(-n // P) for n in lens]
    order = torch.randperm(sum(need) + 4, generator=torch.Generator().manual_seed(seed)).tolist()
    W = max(need + [1]) + 1
    table = [[order.pop() for _ in range(n)] + [-5] * (W - n) for n in need]
    pages = sum(need) + 4
    k, v = (torch.randint(0, 256, (pages, G, P, D // 2), generator=g, device="cuda").to(U8) for _ in range(2))
    kw, vw = (words_of(2.0 ** (spread * (torch.rand(pages, G, P, generator=g, device="cuda") * 2 - 1)) / 5, torch.randint(0, 16, (pages, G, P), generator=g, device="cuda"))
              for _ in range(2))
    for t, n in zip(table, lens):                             # words of rows behind the last: anything
        if n % P:
            kw[t[n // P], :, n % P:] = torch.randint(-2 ** 15, 2 ** 15, (G, P - n % P), generator=g, device="cuda").to(I16)
            vw[t[n // P], :, n % P:] = 0xff03 - 65536               # (an infinite scale)
    q = (q_scale * torch.randn(sum(counts), H, D, generator=g, device="cuda")).to(dtype)
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    return q, k, v, kw, vw, i32(table), i32(start), i32(lens)


def words_of(scale, zero):
    return ((scale.view(I32) >> 19) << 4 | zero.to(I32)).to(I16)


def attention_in_64_bits(q, k, v, kw, vw, table, start, lens, scale):
    """(result, bound): how far float32 scores, float16 weights and the result's rounding may take it.
    Weights are rounded to float16: 2^-11 relative, or 2^-25 absolute where the largest weight * value scale of a row is 1 (below float16's
    normal range). A score is a sum of D exact products in float32 (at most 2^-23 of the sum of their sizes for each addition in the tensor cores,
    which cut), times factors (4 roundings), and enters the exponential, whose own error and that of log2 of the scale are below 2^-20; sums of
    values and weights in float32 add 2^-23 a key at most. Codes of keys enter the products without their zero point, which is taken out behind them:
    D / 16 products of 16 terms and as many of the row's sum, no partial sum of which is above 15 sum |q| (in units of the key's scale), each term cut at 2^-24 of that."""
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
            kk, vv = (values(c[at, g], w[at, g]).reshape(-1, D)[:n] for c, w in ((k, kw), (v, vw)))
            fk, fv = (scales(w[at, g])[0].double().reshape(-1)[:n] for w in (kw, vw))
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
            for h in range(g * rep, (g + 1) * rep):
                x = q[lo:hi, h].to(F64)
                s = (x @ kk.T * scale).masked_fill(hidden, -math.inf)
                some = ~hidden.all(1)
                w = torch.exp(s - s.amax(1, keepdim=True).nan_to_num(neginf=0.0))
                total = w.sum(1, keepdim=True)
                o = w @ vv / total.clamp(min=1e-300)
                size = w @ vv.abs() / total.clamp(min=1e-300)
                carried = x.abs().sum(1, keepdim=True) * 15 * fk[None] * (2 * D // 16 * 17 * 2.0 ** -24)
                ds = (((x.abs() @ kk.abs().T) * ((D + 5) * 2.0 ** -23) + carried) * scale + 2.0 ** -20).masked_fill(hidden, 0.0).amax(1, keepdim=True)
                top = (w * fv[None]).amax(1, keepdim=True)
                small = n * 2.0 ** -25 * 15 * top / total.clamp(min=1e-300)
                out[lo:hi, h] = torch.where(some[:, None], o, 0.0)
                bound[lo:hi, h] = size * (2.0 ** -11 + 2 * ds + n * 2.0 ** -23) + small
    return out, bound + (out.abs() + bound) * (torch.finfo(q.dtype).eps / 2) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)


def attend(form, q, k, v, kw, vw, table, start, lens, out, scale, work, max_tokens=None, roles=0):
    """rows: the call as it is; prompt, pairs: every request with rows enough goes to the prompt form, with one or two tiles of rows a CTA."""
    if form == "rows":
        return ops.kv4_attention(q, k, v, kw, vw, table, start, lens, out, scale, work, max_tokens=max_tokens)
    lib, T, H, D = _lib.load(), q.shape[0], q.shape[1], q.shape[2]
    _lib.check(lib.qspec_debug_kv4_attention_give_up(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), kw.data_ptr(), vw.data_ptr(), table.data_ptr(),
                                                     start.data_ptr(), lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), T, len(lens), table.shape[1], H, k.shape[1], D,
                                                     k.shape[0], k.shape[2], T if max_tokens is None else max_tokens, scale, int(q.dtype == torch.bfloat16), work.data_ptr(),
                                                     work.numel(), 16 * (form == "pairs") + roles, torch.cuda.current_stream().cuda_stream), "kv4_attention")
    return out


def check_attention(case, D, max_tokens=None, workspace=None, form="rows"):
    q, k, v, kw, vw, table, start, lens = case
    scale = D ** -0.5
    out = torch.full_like(q, 3.0)
    work = ops.kv4_attention_workspace("cuda") if workspace is None else workspace
    for _ in range(2):                                        # the workspace is left as the next call needs it
        attend(form, q, k, v, kw, vw, table, start, lens, out, scale, work, max_tokens=max_tokens)
    want, bound = attention_in_64_bits(q, k, v, kw, vw, table, start, lens, scale)
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
                                           (40, 8, 128, 32, torch.bfloat16), (128, 1, 64, 64, torch.float16)])
@pytest.mark.parametrize("lens,counts", [([17], [17]), ([200], [200]), ([130, 400, 65, 300], [130, 100, 1, 300]), ([257, 9, 1000], [33, 4, 129])])
@pytest.mark.parametrize("form", FORMS)
def test_attention_of_prompts(H, G, D, P, dtype, lens, counts, form):
    check_attention(make_attention(4, lens, counts, H, G, D, P, dtype), D, form=form)


@pytest.mark.parametrize("form", FORMS)
def test_attention_rows_that_see_nothing_and_rows_of_no_request(form):
    q, *rest = make_attention(5, [0, 40, 0, 300], [2, 1, 40, 3], 8, 2, 128, 32, torch.float16)
    out = check_attention((torch.cat([q, q[:9]]), *rest), 128, form=form)   # (nine rows behind the last request)
    assert not out[:2].any() and not out[3:43].any() and out[2].any()


@pytest.mark.parametrize("form,counts", [("rows", [1, 4, 2])] + [(f, [150, 4, 60]) for f in FORMS])
def test_attention_with_scales_far_apart(form, counts):
    """Rows whose value scales differ by 2^20: the weights' common factor takes the scale in, and no row loses its part of the sum."""
    q, k, v, kw, vw, table, start, lens = make_attention(6, [500, 200, 900], counts, 8, 2, 128, 16, torch.bfloat16)
    vw.sub_((torch.randint(0, 21, vw.shape, device="cuda", generator=gen(2)) << 8).to(I16))   # (of the exponent)
    check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e30])
def test_attention_of_queries_of_any_size(q_scale, form):
    case = make_attention(7, [100, 70], [2, 30], 4, 2, 128, 32, torch.bfloat16, q_scale=q_scale)
    if q_scale > 1:                                           # one key takes all: its value, rounded
        out = torch.empty_like(case[0])
        attend(form, *case, out, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
        want, _ = attention_in_64_bits(*case, 128 ** -0.5)
        torch.testing.assert_close(out.to(F64), want, rtol=2.0 ** -8 + 2.0 ** -10, atol=1e-30)
    else:
        check_attention(case, 128, form=form)


def test_attention_of_rows_of_very_different_sizes():
    """Rows of a tile whose queries differ by 2^60: each keeps its own digits."""
    q, *rest = make_attention(7, [300, 70], [2, 3], 8, 2, 128, 32, torch.bfloat16)
    q.mul_(2.0 ** torch.randint(-60, 1, q.shape[:2], device="cuda", generator=gen(1))[..., None].float())
    check_attention((q, *rest), 128)


@pytest.mark.parametrize("form,counts", [("rows", [1, 2, 1])] + [(f, [40, 2, 70]) for f in FORMS])
def test_attention_shows_what_is_broken_and_only_there(form, counts):
    """A query that is not a number, and a table entry outside the cache, make the rows that have to do with them NaN, and no others."""
    q, k, v, kw, vw, table, start, lens = make_attention(8, [90, 200, 150], counts, 8, 2, 128, 64, torch.float16)
    clean = check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)
    q2 = q.clone()
    q2[0, 3, 5] = math.nan
    table2 = table.clone()
    table2[2, 1] = 10 ** 6
    out = torch.empty_like(q)
    attend(form, q2, k, v, kw, vw, table2, start, lens, out, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 3] = True
    first = int(lens[2]) - counts[2]
    for i in range(counts[2]):
        bad[int(start[2]) + i] = first + i >= 64
    assert out.isnan().all(2).equal(bad) and out.isnan().any(2).equal(bad)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("word", [0xff03 - 65536, 0xffa3 - 65536])   # an infinite scale, and one that is no number
@pytest.mark.parametrize("side", ["keys", "values"])
def test_attention_shows_a_scale_that_is_no_number_and_only_where_it_is_seen(side, word, form):
    q, k, v, kw, vw, table, start, lens = make_attention(20, [200, 333], [60, 40], 8, 2, 128, 32, torch.float16)
    clean = check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)
    for page in (int(table[0, 5]), int(table[1, 9])):         # positions 165 and 293 of one head
        (kw if side == "keys" else vw)[page, 1, 5] = word
    out = torch.empty_like(q)
    attend(form, q, k, v, kw, vw, table, start, lens, out, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[25:60, 4:] = True                                     # tokens at 140 .. 199
    bad[60:, 4:] = True                                       # tokens at 293 .. 332
    assert out.isnan().all(2).equal(bad) and out.isnan().any(2).equal(bad)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("form", FORMS)
def test_attention_of_strided_queries_and_outputs(form):
    q, *rest = make_attention(9, [90, 200, 300], [1, 2, 40], 8, 2, 128, 64, torch.float16)
    want = check_attention((q, *rest), 128, form=form)
    wide = torch.randn(43, 12, 160, device="cuda").half()
    wide[:, 2:10, 16:144] = q
    out = torch.full((43, 9, 136), 5.0, dtype=torch.float16, device="cuda")
    attend(form, wide[:, 2:10, 16:144], *rest, out[:, 1:, :128], 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    assert torch.equal(out[:, 1:, :128], want) and (out[:, 0] == 5).all() and (out[:, :, 128:] == 5).all()


def test_attention_is_the_same_every_time_and_in_a_graph():
    case = make_attention(10, [5000, 333, 64, 1800], [4, 4, 1, 2], 32, 8, 128, 64, torch.float16)
    q, k, v, kw, vw, table, start, lens = case
    work = ops.kv4_attention_workspace("cuda")
    want = check_attention(case, 128, workspace=work)
    out = torch.empty_like(q)
    ops.kv4_attention(*case, out, 128 ** -0.5, work)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv4_attention(*case, out, 128 ** -0.5, work)
    for _ in range(20):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    lens.copy_(i32([4000, 300, 60, 65]))                      # other lengths, the same graph
    graph.replay()
    want, bound = attention_in_64_bits(q, k, v, kw, vw, table.clamp(min=0), start, lens, 128 ** -0.5)
    assert ((out.to(F64) - want).abs() <= bound).all()


def test_two_streams_with_a_workspace_each():
    cases = [make_attention(s, [9000, 700], [1, 2], 16, 4, 128, 64, torch.float16) for s in (11, 12)]
    want = [check_attention(c, 128) for c in cases]
    streams, works = [torch.cuda.Stream() for _ in cases], [ops.kv4_attention_workspace("cuda") for _ in cases]
    outs = [torch.empty_like(c[0]) for c in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, w, o in zip(cases, streams, works, outs):
            with torch.cuda.stream(s):
                ops.kv4_attention(*c, o, 128 ** -0.5, w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("H,G", [(8, 2), (6, 2), (16, 1)])
def test_attention_of_requests_with_more_tokens_than_keys(H, G, form):
    """The first tokens stand in front of the first key and see nothing, whole tiles of them, or of one of two tiles."""
    lens, counts = [32, 40, 3, 1, 300], [64, 130, 70, 200, 310]
    case = make_attention(16, lens, counts, H, G, 128, 32, torch.float16)
    out = check_attention(case, 128, form=form)
    for at, keys, n in zip(case[6].tolist(), lens, counts):
        assert not out[at:at + n - keys].any() and out[at + n - keys].any()


@pytest.mark.parametrize("lens,counts", [([3000, 70], [2, 4]), ([400, 300], [300, 290])])
def test_attention_over_its_own_queries(lens, counts):
    case = make_attention(17, lens, counts, 32, 8, 128, 64, torch.float16)
    want = check_attention(case, 128)
    q = case[0].clone()
    ops.kv4_attention(q, *case[1:], q, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    assert torch.equal(q, want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ratio,gap", [(1, 25.05), (8, 22.1), (8, 24.0), (4, 23.1)])
def test_attention_loses_no_keys_of_a_long_context(ratio, gap, dtype, form):
    """Values that are all 1, whatever their weights: so is the result. The first key's score is above all others' by log2 = gap, and its row may have a value scale that
    is `ratio` times the others' (and another code). Off by the result's rounding; 2^-11 for a weight that is a normal float16; ratio * 2^-34 for each key whose weight is not (2^-25,
    the largest being 2^9 or more, with the value scale in it); and float32 sums: 2^-23 for every key that one accumulator takes, half of that for the denominator. In the prompt form
    that is n keys, in the other a quarter: there so many requests (of the same pages) that each is one CTA's, of four warps."""
    n, G, H, D, P = 131000, 2, 8, 128, 64
    B, T = (256, 1) if form == "rows" else (1, 20) if form == "prompt" else (1, 50)
    pages = -(-n // P)
    k, v = torch.zeros(pages, G, P, D // 2, dtype=U8, device="cuda"), torch.full((pages, G, P, D // 2), 0x99, dtype=U8, device="cuda")
    ones = torch.ones(pages, G, P, device="cuda")
    kw, vw = words_of(ones, torch.zeros_like(ones)), words_of(ones / 8, torch.ones_like(ones))   # (9 - 1) / 8
    v[0, :, 0], vw[0, :, 0] = 0xee, int(words_of(torch.tensor(ratio / 8), torch.tensor(14 - 8 // ratio)))   # 8 / ratio * ratio / 8
    k[0, :, 0, 0] = 1
    q = torch.zeros(B * T, H, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    case = (q, k, v, kw, vw, torch.arange(pages, dtype=I32, device="cuda").repeat(B, 1), i32(range(0, B * T + 1, T)), i32([n] * B))
    out = torch.empty_like(q)
    attend(form, *case, out, gap / math.log2(math.e), ops.kv4_attention_workspace("cuda"), max_tokens=T)
    chain = n / (4 if form == "rows" else 1)
    bound = torch.finfo(dtype).eps / 2 + 2.0 ** -11 + n * ratio * 2.0 ** -34 + chain * 1.5 * 2.0 ** -23
    assert (out.double() - 1).abs().max() <= bound, (float((out.double() - 1).abs().max()), bound)


@pytest.mark.parametrize("form", FORMS)
def test_attention_of_scores_far_from_zero(form):
    """Exponents of 2^20 to 2^26, where a reference's own rounding is large: weights stay finite, and one key, or several that are alike, take all."""
    n, G, D, P, T = 700, 2, 128, 32, 2 if form == "rows" else 40
    pages = -(-n // P)
    for log2 in (18, 20, 21.9, 22.1, 23, 23.9, 24.1, 25, 26):
        for sign in (1.0, -1.0):
            g = gen(int(log2 * 10))
            k = torch.zeros(pages, G, P, D // 2, dtype=U8, device="cuda")
            k[..., 0] = 10                                        # all scores alike, and far from zero
            v = torch.randint(0, 256, (pages, G, P, D // 2), generator=g, device="cuda").to(U8)
            ones = torch.ones(pages, G, P, device="cuda")
            kw, vw = words_of(ones * 2.0 ** log2 / 10, 0 * ones), words_of(ones / 4, 0 * ones + 8)
            q = torch.zeros(T, 8, D, dtype=torch.float16, device="cuda")
            q[:, :, 0] = sign
            case = (q, k, v, kw, vw, torch.arange(pages, dtype=I32, device="cuda")[None], i32([0, T]), i32([n]))
            out = torch.empty_like(q)
            attend(form, *case, out, 1.0, ops.kv4_attention_workspace("cuda"), max_tokens=T)
            rows = values(v, vw).permute(1, 0, 2, 3).reshape(G, -1, D)
            want = torch.stack([rows[:, :n - T + 1 + t].mean(1) for t in range(T)]).repeat_interleave(4, 1)
            # equal weights: each off by 2^-11, sums by n / 16 * 2^-23, the result by its own rounding
            size = rows.abs().mean(1).amax()
            assert ((out.double() - want).abs() <= size * (2.0 ** -11 + 2.0 ** -11 + n / 16 * 2.0 ** -23) + want.abs() * 2.0 ** -11 + 2.0 ** -24).all(), (log2, sign)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("log2", [-112, 100, 120])
def test_attention_of_queries_and_scales_that_make_up_for_each_other(log2, form):
    """Tiny queries over keys of a huge scale, and the other way round: the factors of the scores meet before they leave float32."""
    counts = [1, 3] if form == "rows" else [60, 40]
    q, k, v, kw, vw, table, start, lens = make_attention(18, [200, 333], counts, 8, 2, 128, 32, torch.bfloat16, q_scale=1.5 * 2.0 ** log2)
    kw.copy_(((kw.to(I32) & 0xffff) - (min(log2, 93) << 8)).to(I16))   # (of the exponent; scales below 2^-100 count as that)
    check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)


@pytest.mark.parametrize("form", FORMS)
def test_attention_walks_no_further_than_the_table(form):
    """Lengths beyond the table's pages, up to the largest number there is: the rows that see such keys are NaN, soon; others are what they are."""
    q, k, v, kw, vw, table, start, lens = make_attention(21, [200, 256, 100], [40, 20, 40], 8, 2, 128, 32, torch.float16)
    clean = check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)
    work = ops.kv4_attention_workspace("cuda")
    short = table[:, :4].contiguous()                         # 128 keys
    for large in (129, 300, 10 ** 6, 2 ** 31 - 1):
        far = i32([large, 256, 100])
        out = attend(form, q, k, v, kw, vw, short, start, far, torch.zeros_like(q), 128 ** -0.5, work)
        first = large - 40
        bad = torch.tensor([first + i >= 128 for i in range(40)] + [True] * 20 + [False] * 40, device="cuda")
        assert out[bad].isnan().all() and not out[~bad].isnan().any()
        assert torch.equal(out[60:], clean[60:])


GIVE_UP = r"""
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from test_gpu_kv4 import make_attention, attend
from qspec_b200 import ops
for D, dtype in ((128, torch.float16), (64, torch.bfloat16)):
    case = make_attention(3, [500, 900, 40], [130, 300, 1], 8, 2, D, 32, dtype)
    q, work = case[0], ops.kv4_attention_workspace("cuda")
    good = ops.kv4_attention(*case, torch.empty_like(q), D ** -0.5, work)
    for form in ("prompt", "pairs"):
        for roles in (1, 2, 4, 8, 15):
            before = ops.attn_tile_timeouts()
            out = attend(form, *case, torch.zeros_like(q), D ** -0.5, work, 300, roles)
            assert ops.attn_tile_timeouts() > before, roles
            assert out[:430].isnan().all() and torch.equal(out[430:], good[430:]), roles   # the request with few rows is the other form's
            again = ops.kv4_attention(*case, torch.empty_like(q), D ** -0.5, work)
            assert torch.equal(again, good)
print("ok")
"""


def test_a_wait_that_is_given_up_shows_and_leaves_nothing_behind():
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", GIVE_UP.format(root=os.path.dirname(tests), tests=tests)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


@pytest.mark.parametrize("lens,counts", [([400, 2000, 130], [300, 20, 70]),       # long: its way through its keys is longer than the others', so not the prompt form
                                         ([9000, 64, 900, 5000], [65, 64, 512, 16]), ([300] * 40 + [7] * 200, [20] * 40 + [1] * 200)])
@pytest.mark.parametrize("H,G", [(32, 8), (10, 2), (5, 5)])
def test_attention_of_requests_that_take_different_forms(H, G, lens, counts):
    check_attention(make_attention(14, lens, counts, H, G, 128, 64, torch.float16), 128)


def test_the_form_is_the_rules_and_both_kernels_agree_on_it():
    """Rows of the prompt form and of the other one differ in their last bits: which form a request took shows in its rows."""
    lens, counts, H, G = [900, 9000, 300, 1200, 40], [200, 30, 1, 500, 24], 32, 8
    case = make_attention(15, lens, counts, H, G, 128, 64, torch.float16)
    out, sms = check_attention(case, 128), torch.cuda.get_device_properties(0).multi_processor_count
    forced = attend("pairs" if sum(counts) * H > 160 * sms else "prompt", *case, torch.empty_like(out), 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    rows = [n * H // G for n in counts]
    total = sum(r * G * -(-n // 128) for r, n in zip(rows, lens) if r >= 65)
    picks = [r >= 65 and -(-n // 128) * (sms // 4 * 128) <= total for r, n in zip(rows, lens)]
    assert picks == [True, False, False, True, True]
    for b, pick in enumerate(picks):
        at = slice(sum(counts[:b]), sum(counts[:b + 1]))
        assert counts[b] == 1 or torch.equal(out[at], forced[at]) == pick


def test_cache_whose_offsets_pass_32_bits():
    """2.2 GB of codes for keys: the pages used lie behind 2^31 bytes."""
    G, P, D, H = 8, 128, 128, 16
    pages = (1 << 31) // (G * P * D // 2) + 40
    small = make_attention(22, [300, 90], [2, 1], H, G, D, P, torch.float16)
    q, k, v, kw, vw, table, start, lens = small
    first = pages - k.shape[0]
    big = [torch.zeros(pages, *t.shape[1:], dtype=t.dtype, device="cuda") for t in (k, v, kw, vw)]
    for b, t in zip(big, (k, v, kw, vw)):
        b[first:] = t
    want, out = check_attention(small, D), torch.empty_like(q)
    far = torch.where(table >= 0, table + first, table)
    ops.kv4_attention(q, *big, far, start, lens, out, D ** -0.5, ops.kv4_attention_workspace("cuda"))
    assert torch.equal(out, want)
    slots = (far[0, :1] * P + torch.arange(20, device="cuda")).to(I32)
    near = (table[0, :1] * P + torch.arange(20, device="cuda")).to(I32)
    got = [[torch.empty(20, G, D, dtype=torch.float16, device="cuda") for _ in range(2)] for _ in range(2)]
    ops.kv4_read(*big, slots, *got[0])
    ops.kv4_read(k, v, kw, vw, near, *got[1])
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


# ---- refusals that need tensors on the GPU -------------------------------------------------------------------------------------------
def test_wrong_shapes_and_types_are_refused():
    z = lambda *s, dtype=I32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    half = lambda *s: z(*s, dtype=torch.float16)  # noqa: E731
    cache = [z(3, 2, 16, 32, dtype=U8), z(3, 2, 16, 32, dtype=U8), z(3, 2, 16, dtype=I16), z(3, 2, 16, dtype=I16)]
    app = [half(3, 8 * 64), half(9, 64), z(3), z(3), *cache, half(3, 4, 64)]
    ops.kv4_append(*app)
    for i, bad in ((0, half(3, 4 * 64)), (0, half(3, 8 * 64 + 1)), (1, z(9, 64, dtype=F32)), (1, half(9, 32)), (2, z(4)), (3, z(3, dtype=torch.int64)), (5, cache[0][:2]),
                   (6, z(3, 2, dtype=I16)), (7, z(3, 2, 16, dtype=I32)), (8, half(3, 3, 64)), (8, half(4, 3, 64).transpose(0, 1)), (4, cache[0].view(torch.int8)),
                   (4, z(3, 2, 16, 64, dtype=U8)[..., ::2])):
        with pytest.raises(ValueError):
            ops.kv4_append(*[bad if j == i else a for j, a in enumerate(app)])
    att = [half(3, 4, 64), *cache, z(2, 4), z(3), z(2), half(3, 4, 64), 0.1, ops.kv4_attention_workspace("cuda")]
    ops.kv4_attention(*att)
    for i, bad in ((0, z(3, 4, 64, dtype=F32)), (0, half(3, 4, 32)), (5, z(8)), (6, z(2)), (7, z(3)), (8, half(3, 4, 64).bfloat16()), (8, half(2, 4, 64)), (9, 0.0), (9, math.nan),
                   (10, z(9, dtype=F32)), (0, half(3, 5, 64)), (10, z(100, dtype=U8))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv4_attention(*[bad if j == i else a for j, a in enumerate(att)])
    with pytest.raises(ValueError):
        ops.kv4_read(*cache, z(3), half(3, 2, 64), half(2, 2, 64))


def test_scales_next_to_a_half_are_those_of_the_formula():
    """(hi - lo) * float32(1 / 15) within a few units of the last place of a border between two scales, on either side: a million rows, most of whose ranges lie there."""
    G, D, P, n = 8, 64, 128, 128 * 1024
    g = gen(30)
    border = (16.5 + torch.randint(0, 16, (n, G), generator=g, device="cuda")) / 16 * 2.0 ** torch.randint(-6, 6, (n, G), generator=g, device="cuda") * 15
    x = torch.randn(n, 3 * G, D, generator=g, device="cuda").clamp(-0.4, 0.4) * border.repeat(1, 3)[..., None] * 0.1
    x[:, 2 * G:, 0] = border * 0.6
    x[:, 2 * G:, 1] = -border * 0.4
    x = x.bfloat16()                                          # (values: as they lie in the rows)
    lo = x[:, 2 * G:].amin(-1).float()
    x[:, 2 * G:, 0] = (border + lo).bfloat16()
    k, v = (torch.zeros(n // P, G, P, D // 2, dtype=U8, device="cuda") for _ in range(2))
    kw, vw = (torch.zeros(n // P, G, P, dtype=I16, device="cuda") for _ in range(2))
    at = i32(range(n))
    cs = torch.cat((torch.ones(n, D // 2), torch.zeros(n, D // 2)), 1).bfloat16().cuda()
    ops.kv4_append(x.flatten(1), cs, at, at, k, v, kw, vw, None)
    for got_c, got_w, rows in ((k, kw, x[:, G:2 * G]), (v, vw, x[:, 2 * G:])):
        c, w = quantised(rows.float())
        assert torch.equal(got_w, w.view(n // P, P, G).transpose(1, 2)) and torch.equal(got_c, c.view(n // P, P, G, D // 2).transpose(1, 2))


# ---- tiles of eight rows: calls that say that no request has more (and hold if one does) ----------------------------------------------
@pytest.fixture
def eights(monkeypatch):
    """`attend` with one token as the most of a request."""
    import sys
    whole = attend
    monkeypatch.setattr(sys.modules[__name__], "attend", lambda form, *args, max_tokens=None, **kw: whole(form, *args, max_tokens=1, **kw))


@pytest.mark.parametrize("H,G,D,P,dtype", [(64, 8, 128, 16, torch.bfloat16), (32, 8, 128, 128, torch.float16), (3, 1, 128, 64, torch.bfloat16), (8, 8, 64, 32, torch.float16), (14, 2, 64, 16, torch.bfloat16)])
@pytest.mark.parametrize("lens,counts", [([1, 2, 31, 32, 33, 700], [1] * 6), ([64, 65, 1000, 5], [2, 1, 2, 0]), ([40000, 3], [1, 2]), ([70] * 300, [1] * 300), ([900] * 33, [1] * 33),
                                         ([130, 400, 9], [130, 17, 3])])
def test_eights_of_requests_of_every_kind(eights, H, G, D, P, dtype, lens, counts):
    check_attention(make_attention(31, lens, counts, H, G, D, P, dtype), D)


def test_eights_of_rows_that_see_nothing_of_scales_and_queries_far_apart_and_of_broken_ones(eights):
    test_attention_rows_that_see_nothing_and_rows_of_no_request("rows")
    test_attention_of_rows_of_very_different_sizes()
    test_attention_of_strided_queries_and_outputs("rows")
    test_attention_walks_no_further_than_the_table("rows")
    for counts in ([1, 2, 1], [40, 2, 70]):
        test_attention_shows_what_is_broken_and_only_there("rows", counts)
        test_attention_with_scales_far_apart("rows", counts)
    for q_scale in (0.0, 1e-30, 1e30):
        test_attention_of_queries_of_any_size(q_scale, "rows")
    for log2 in (-112, 100, 120):
        test_attention_of_queries_and_scales_that_make_up_for_each_other(log2, "rows")
    test_attention_of_scores_far_from_zero("rows")
    test_attention_of_requests_with_more_tokens_than_keys(6, 2, "rows")


def test_eights_are_the_same_every_time_in_a_graph_and_over_their_own_queries():
    case = make_attention(32, [5000, 333, 64, 1800], [1, 1, 1, 1], 32, 8, 128, 64, torch.float16)
    work, out = ops.kv4_attention_workspace("cuda"), torch.empty_like(case[0])
    want = check_attention(case, 128, max_tokens=1, workspace=work)
    ops.kv4_attention(*case, out, 128 ** -0.5, work, max_tokens=1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv4_attention(*case, out, 128 ** -0.5, work, max_tokens=1)
    for _ in range(20):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    q = case[0].clone()
    ops.kv4_attention(q, *case[1:], q, 128 ** -0.5, work, max_tokens=1)
    assert torch.equal(q, want)
    # a workspace serves calls of either kind, one after the other
    sixteen = check_attention(case, 128, max_tokens=5, workspace=work)
    assert torch.equal(check_attention(case, 128, max_tokens=1, workspace=work), want) and torch.equal(check_attention(case, 128, max_tokens=5, workspace=work), sixteen)


@pytest.mark.parametrize("R,lens", [(1, 5000), (54, 700), (55, 700), (56, 700), (75, 90), (130, 33)])
def test_eights_around_where_there_are_more_ctas(R, lens):
    """With eight heads of keys the rule's limit is at three requests for eight SMs."""
    check_attention(make_attention(33, [lens - i % 7 for i in range(R)], [1] * R, 32, 8, 128, 64, torch.float16), 128, max_tokens=1)


# ---- scales of a block of keys that are far apart ------------------------------------------------------------------------------------------
def rescaled(words, table, at, exponents):
    """Words of positions `at` of a request's row of the table, with 2^exponents times their scale."""
    P = words.shape[2]
    pages, rows = table[at // P].long(), at % P
    words[pages, :, rows] = ((words[pages, :, rows].to(I32) & 0xffff) + (exponents[:, None] << 8)).to(I16)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("side", ["keys", "values", "both"])
@pytest.mark.parametrize("by", [20, 29, 31, 45, -45])
@pytest.mark.parametrize("D,P,dtype", [(128, 32, torch.float16), (64, 16, torch.bfloat16)])
def test_attention_of_tokens_whose_keys_are_not_the_blocks_largest(form, side, by, D, P, dtype):
    """Keys 64 .. 127 and 300 .. 399 of a request have scales 2^by times the others': what the tokens in front of them see is exact all the same. (Those behind them see scores that far apart.)"""
    lens, counts = [160, 500], [150, 450]
    q, k, v, kw, vw, table, start, lens = make_attention(40, lens, counts, 8, 2, D, P, dtype)
    for b, ranges in enumerate([[(64, 128)], [(64, 128), (300, 400)]]):
        for lo, hi in ranges:
            for words, name in ((kw, "keys"), (vw, "values")):
                if side in (name, "both"):
                    rescaled(words, table[b], torch.arange(lo, hi, device="cuda"), torch.full((hi - lo,), by if name == "keys" or dtype == torch.bfloat16 else min(by, 10), device="cuda"))
    check_attention((q, k, v, kw, vw, table, start, lens), D, form=form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_over_scales_of_every_size(form, dtype):
    """Values' scales from 2^-88 to 2^2 and keys' from 2^-60 to 2^2, in any order, rows whose words are zero, and more tokens than keys."""
    q, k, v, kw, vw, table, start, lens = make_attention(41, [400, 90, 300], [380, 100, 130], 8, 2, 128, 64, dtype)
    g = gen(41)
    for b, n in enumerate(lens.tolist()):
        at = torch.arange(n, device="cuda")
        rescaled(vw, table[b], at, torch.randint(-88, 3, (n,), generator=g, device="cuda"))
        rescaled(kw, table[b], at, torch.randint(-60, 3, (n,), generator=g, device="cuda"))
        some = at[at % 17 == 3]
        vw[table[b][some // 64].long(), :, some % 64] = 0
        kw[table[b][some // 64].long(), :, some % 64] = 0
    out = check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)
    assert not out[380:390].any() and out[390:].any()


@pytest.mark.parametrize("form", FORMS)
def test_attention_shows_broken_words_among_scales_far_apart(form):
    q, k, v, kw, vw, table, start, lens = make_attention(42, [300, 300], [250, 290], 8, 2, 128, 32, torch.bfloat16)
    for b in range(2):
        rescaled(vw, table[b], torch.arange(0, 300, 3, device="cuda"), torch.full((100,), -60, device="cuda"))
    clean = check_attention((q, k, v, kw, vw, table, start, lens), 128, form=form)
    kw[int(table[0, 5]), 0, 5] = 0xffa3 - 65536               # position 165, head 0; and position 229 of the other request, head 1
    vw[int(table[1, 7]), 1, 5] = 0xff03 - 65536
    out = torch.empty_like(q)
    attend(form, q, k, v, kw, vw, table, start, lens, out, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[165 - 50:250, :4] = True
    bad[250 + 229 - 10:, 4:] = True
    assert out.isnan().all(2).equal(bad) and out.isnan().any(2).equal(bad)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("by", [6, 9, 15, 20, 25, 29])
def test_attention_next_to_a_key_that_counts_for_nothing(by, dtype, form):
    """Values that are all 1, but for one key's, whose scale is 2^by times theirs; its code is the zero point, and its weight 2^-40 of the others'. The first key has as much weight as 1900 others together,
    2^10.9 times each: so the result is 1. Off by its rounding, 2^-11 of a weight that is a normal float16, 2^-25 of one that is not where the largest weight and value scale are 2^(9 - 8) or more
    together (half of the sum or more is the first key's: n 2^-26), and float32 sums, 1.5 n / 4 2^-23."""
    n, G, H, D, P, T = 1900, 1, 4, 64, 64, 40
    pages = -(-n // P)
    ones = torch.ones(pages, G, P, device="cuda")
    k, v = torch.full((pages, G, P, D // 2), 0x88, dtype=U8, device="cuda"), torch.full((pages, G, P, D // 2), 0x99, dtype=U8, device="cuda")
    kw, vw = words_of(ones, 8 * ones), words_of(ones, 8 * ones)
    k[0, 0, 0, 0], k[0, 0, 5, 0], v[0, 0, 5] = 0x89, 0x80, 0x88   # scores of 1 and (with half the scale) of -4, a value of nothing
    kw[0, 0, 5] = int(words_of(torch.tensor(0.5), torch.tensor(8)))
    vw[0, 0, 5] = int(words_of(torch.tensor(2.0 ** by), torch.tensor(8)))
    q = torch.zeros(T, H, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    out = torch.empty_like(q)
    case = (q, k, v, kw, vw, torch.arange(pages, dtype=I32, device="cuda")[None], i32([0, T]), i32([n]))
    attend(form, *case, out, 10.9 / math.log2(math.e), ops.kv4_attention_workspace("cuda"), max_tokens=T)
    bound = torch.finfo(dtype).eps / 2 + 2.0 ** -11 + n * 2.0 ** -26 + 1.5 * n / 4 * 2.0 ** -23
    assert ((out.double() - 1).abs() <= bound).all(), (float((out.double() - 1).abs().max()), bound)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("exponent", [250, 252, 253, 254])
@pytest.mark.parametrize("others", [None, 215])
def test_attention_over_values_as_large_as_there_are(others, exponent, form):
    """Value scales of up to 31 / 16 2^127 (what the writer gives ends at 2^123), alone and among others of 2^88. What weights are divided by that with is 2^-136 and more, a subnormal number that is off
    by 2^-14 of itself at most, and so is the denominator."""
    q, k, v, kw, vw, table, start, lens = make_attention(43, [300, 90], [40, 70], 8, 2, 128, 32, torch.bfloat16)
    v.copy_(0x77 + torch.randint(0, 3, v.shape, generator=gen(43), device="cuda") + 16 * torch.randint(0, 3, v.shape, generator=gen(44), device="cuda"))   # (codes 7 to 9)
    word = (exponent << 8) + (torch.randint(0, 16, vw.shape, generator=gen(45), device="cuda") << 4) + 8
    if others:
        word = torch.where(torch.arange(32, device="cuda") % 5 == 2, word, (word & 0xff) + (others << 8))
    vw.copy_(word.to(I16))
    out = torch.empty_like(q)
    attend(form, q, k, v, kw, vw, table, start, lens, out, 128 ** -0.5, ops.kv4_attention_workspace("cuda"))
    want, bound = attention_in_64_bits(q, k, v, kw, vw, table, start, lens, 128 ** -0.5)
    assert torch.isfinite(out).all()
    assert ((out.to(F64) - want).abs() <= bound + want.abs() * 2.0 ** -14).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_keys_as_large_as_there_are(dtype, form):
    """Key scales of 2^123 and 2^127. Where a row's query is zero in the columns in which they are not, their scores are zero; where it is not, one of them (the largest) takes all."""
    T, H, D, P, n = 40, 4, 128, 32, 200
    pages = -(-n // P)
    ones = torch.ones(pages, 1, P, device="cuda")
    k, v = torch.full((pages, 1, P, D // 2), 0x88, dtype=U8, device="cuda"), torch.randint(0, 256, (pages, 1, P, D // 2), generator=gen(46), device="cuda").to(U8)
    kw, vw = words_of(ones, 8 * ones), words_of(ones, 8 * ones)
    k[..., 0] = 0x99                                          # 1 in the first two columns
    k[0, 0, 3, 0], kw[0, 0, 3] = 0x89, (250 << 8) + 8 - 65536     # 2^123 in the first, and 2^127 for another
    k[1, 0, 7, 0], kw[1, 0, 7] = 0x89, (254 << 8) + 8 - 65536
    q = torch.zeros(T, H, D, dtype=dtype, device="cuda")
    q[:, :, 1] = 1.0
    q[T // 2:, :, 0] = 2.0 ** -9
    case = (q, k, v, kw, vw, torch.arange(pages, dtype=I32, device="cuda")[None], i32([0, T]), i32([n]))
    out = torch.empty_like(q)
    attend(form, *case, out, 1.0, ops.kv4_attention_workspace("cuda"))
    rows = values(v, vw)[:, 0].reshape(-1, D)[:n]
    for t in (0, T // 2 - 1):
        m = n - T + 1 + t
        weight = torch.full((m,), math.e, dtype=F64, device="cuda")
        weight[[3, 39]] = 1.0                                 # scores of 0, the others' are 1
        want = (weight[:, None] * rows[:m]).sum(0) / weight.sum()
        # weights are off by 2^-11, sums by n / 16 2^-23, the result by its rounding
        assert ((out[t].double() - want).abs() <= 8 * (2.0 ** -10 + n / 16 * 2.0 ** -23) + want.abs() * torch.finfo(dtype).eps / 2).all()
    assert (out[T // 2:].double() == rows[39]).all()


def test_a_scale_is_the_range_times_float32_of_a_fifteenth():
    """A million rows of keys in float32, by a multiplication that is written as one (tests above divide by a plain number, which PyTorch makes a multiplication of on CUDA)."""
    G, D, P, n = 8, 64, 128, 128 * 1024
    g = gen(47)
    x = torch.randn(n, 3 * G, D, generator=g, device="cuda").half()
    angle = torch.rand(n, D // 2, generator=g, device="cuda") * 6.28
    cs = torch.cat((angle.cos(), angle.sin()), -1).half()
    k, v = (torch.zeros(n // P, G, P, D // 2, dtype=U8, device="cuda") for _ in range(2))
    kw, vw = (torch.zeros(n // P, G, P, dtype=I16, device="cuda") for _ in range(2))
    at = i32(range(n))
    ops.kv4_append(x.flatten(1), cs, at, at, k, v, kw, vw, None, hadamard=True)
    y = hadamard(rotated(x[:, G:2 * G].float(), cs.float(), F32))
    hi, lo = y.amax(-1).clamp(min=0), y.amin(-1).clamp(max=0)
    scale = lambda r: ((r.view(I32) + (1 << 18)) >> 19 << 19).view(F32)  # noqa: E731
    s = scale((hi - lo) * torch.full_like(hi, 1 / 15))
    z = (-lo / s).round()
    got_s, got_z = scales(kw.transpose(1, 2).reshape(n, G))
    assert torch.equal(got_s, s) and torch.equal(got_z, z)
    assert torch.equal(unpack(k.transpose(1, 2).reshape(n, G, D // 2)).float(), ((y / s[..., None]).round() + z[..., None]).clamp(0, 15))


def test_a_scale_is_not_the_range_divided_by_15():
    """Rotated pairs (x cos - w sin, w cos + x sin) whose range times float32(1 / 15) reaches a border between two scales that their range / 15 does not."""
    pairs = [(2.60546875, -0.76904296875, 0.72705078125, 0.81298828125), (2.044921875, -0.04815673828125, 0.51123046875, 0.65673828125),
             (1.6337890625, -0.241455078125, 0.88818359375, 0.66357421875), (4.19921875, -0.9091796875, 0.66845703125, 0.02276611328125),
             (4.1328125, 0.235595703125, 0.7529296875, 0.70849609375), (7.3671875, -0.76416015625, 0.416259765625, 0.88623046875)]
    n, D = len(pairs), 64
    p = torch.tensor(pairs).half().float()                     # (all are float16)
    x, cs = torch.zeros(n, 3, D), torch.zeros(n, D)
    x[:, 1, 0], x[:, 1, 32], cs[:, 0], cs[:, 32] = p.unbind(1)
    a, b = p[:, 0] * p[:, 2] - p[:, 1] * p[:, 3], p[:, 1] * p[:, 2] + p[:, 0] * p[:, 3]
    r = torch.maximum(a, b).clamp(min=0) - torch.minimum(a, b).clamp(max=0)
    scale = lambda r: ((r.view(I32) + (1 << 18)) >> 19 << 19).view(F32)  # noqa: E731
    want, divided = scale(r * torch.full_like(r, 1 / 15)), scale((r.double() / 15).float())   # (rounded once: 24 bits of 53)
    assert (want > divided).all()
    k, v = (torch.zeros(1, 1, 16, D // 2, dtype=U8, device="cuda") for _ in range(2))
    kw, vw = (torch.zeros(1, 1, 16, dtype=I16, device="cuda") for _ in range(2))
    ops.kv4_append(x.flatten(1).half().cuda(), cs.half().cuda(), i32(range(n)), i32(range(n)), k, v, kw, vw, None)
    assert torch.equal(scales(kw[0, 0, :n])[0].cpu(), want)
