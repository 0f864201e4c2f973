"""Attention over the paged caches where scores are so far from zero that a float32 has no bits left behind the point (what exponents are counted from has a rounding of its own there), or so far from
each other that some have no weight at all, or are no numbers."""
import pytest
import torch

import test_gpu_kv4 as kv4
import test_gpu_kv8 as kv8
from qspec_b200 import ops

pytestmark = pytest.mark.gpu
I32, U8 = torch.int32, torch.uint8
LN2 = 0.6931471824645996                                       # the float32 that, times log2(e) in float32, is 1
N, G, D, P = 700, 2, 128, 32
PAGES = -(-N // P)


def levels(E, times, order, g):
    """log2 of a value scale for each page: a score of 1.5 2^E and that is a float32, exactly. The largest is 0."""
    step = int(max(2.0 ** (E - 23), 1) * times)
    most = min(7, 90 // step)
    at = torch.arange(PAGES, device="cuda") * (most + 1) // PAGES
    at = {"up": at, "down": most - at, "any": torch.randint(0, most + 1, (PAGES,), generator=g, device="cuda")}[order]
    return -(step * (most - at)).float()


def check(out, rows, T, alike=True):
    """Scores that are alike, over values rows [G, n, D] in 64 bits: their mean. Weights 2^(score + log2 of the value scale) are off by 2^-11 (those below 2^-23 of the largest by 2^-34 of it) and 2^-21 by
    the exponential, the result by its rounding; sums of n keys in float32 add n / 16 * 2^-23 in the tensor cores.
    (alike: whether exponents, score and value scale together, are rounded alike. Otherwise each is off by half a last place either way, which is all that can be said of a weight's share: the result is
    a mean by some weights.)"""
    for t in sorted({0, T // 2, T - 1}):
        m = N - T + 1 + t
        want, size = rows[:, :m].mean(1), rows[:, :m].abs().mean(1)
        got = out[t].double().unflatten(0, (G, -1))
        bound = size * (2.0 ** -10 + N / 16 * 2.0 ** -23) + N * 2.0 ** -34 * rows.abs().amax() + want.abs() * torch.finfo(out.dtype).eps / 2 + 2.0 ** -24
        assert torch.isfinite(got).all() and (got.abs().amax((1, 2)) <= rows.abs().amax((1, 2)) * (1 + 2.0 ** -7)).all()
        assert not alike or ((got - want[:, None]).abs() <= bound[:, None]).all(), (t, float((got - want[:, None]).abs().max()))


@pytest.mark.parametrize("form", ["rows", "eights", "prompt", "pairs"])
@pytest.mark.parametrize("order", ["up", "down", "any"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_4_bit_cache(order, form, dtype):
    T = 40 if form in ("prompt", "pairs") else 2
    for E in range(18, 31):
        for times in (1, 2, 3, 4, 6):
            for sign in (1.0, -1.0):
                g = kv4.gen(E)
                k = torch.zeros(PAGES, G, P, D // 2, dtype=U8, device="cuda")
                k[..., 0] = 12
                v = torch.randint(0, 256, (PAGES, G, P, D // 2), generator=g, device="cuda").to(U8)
                ones = torch.ones(PAGES, G, P, device="cuda")
                kw, vw = kv4.words_of(ones * 2.0 ** (E - 3), 0 * ones), kv4.words_of(ones * 2.0 ** levels(E, times, order, g)[:, None, None], 0 * ones + 8)
                q = torch.zeros(T, 8, D, dtype=dtype, device="cuda")
                q[:, :, 0] = sign
                case = (q, k, v, kw, vw, torch.arange(PAGES, dtype=I32, device="cuda")[None], kv4.i32([0, T]), kv4.i32([N]))
                out = torch.empty_like(q)
                kv4.attend("rows" if form == "eights" else form, *case, out, LN2, ops.kv4_attention_workspace("cuda"), max_tokens={"rows": 20, "eights": 1}.get(form, T))
                # (the prompt form's exponents are score + log2 of the block's power of two - 10: in the middle between two floats that are 4 apart, and rounded to the even one of them)
                check(out, kv4.values(v, vw).permute(1, 0, 2, 3).reshape(G, -1, D), T, form in ("rows", "eights") or E != 25 or times % 2 == 0)


@pytest.mark.parametrize("form", ["rows", "prompt", "pairs"])
@pytest.mark.parametrize("order", ["up", "down", "any"])
def test_8_bit_cache(order, form):
    T = 40 if form in ("prompt", "pairs") else 2
    for E in range(18, 31):
        for times in (1, 2, 3, 4, 6):
            for sign in (1.0, -1.0):
                g = kv8.gen(E)
                k = torch.zeros(PAGES, G, P, D, dtype=torch.int8, device="cuda")
                k[..., 0] = 96
                v = (torch.randn(PAGES, G, P, D, generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8)
                ks, vs = torch.full((PAGES, G), 2.0 ** (E - 6), device="cuda"), 2.0 ** levels(E, times, order, g)[:, None].expand(PAGES, G).contiguous()
                q = torch.zeros(T, 8, D, dtype=torch.float16, device="cuda")
                q[:, :, 0] = sign
                case = (q, k, v, ks, vs, torch.arange(PAGES, dtype=I32, device="cuda")[None], kv8.i32([0, T]), kv8.i32([N]))
                work, out = ops.kv8_attention_workspace("cuda"), torch.empty_like(q)
                if form == "rows":
                    ops.kv8_attention(*case, out, LN2, work, max_tokens=T)
                else:
                    kv8.prompt_form(*case, out, LN2, work, pairs=form == "pairs")
                # (the prompt form joins the value scale's log2 with what the codes' 128 adds up to, 2^(E + 1): a float with half of the places)
                check(out, (v.double() * vs.double()[..., None, None]).permute(1, 0, 2, 3).reshape(G, -1, D), T, form == "rows" or times % 2 == 0 or E < 23)


@pytest.mark.parametrize("form", ["rows", "eights", "prompt", "pairs"])
@pytest.mark.parametrize("cache", [4, 8])
@pytest.mark.parametrize("high", [0, 1, 2, 5])
@pytest.mark.parametrize("what", ["page", "key", "value"])
def test_what_is_broken_shows_however_little_its_keys_weigh(what, high, cache, form):
    """Keys of one block of 128 have scores 2^9 above all others'; in every other block something is broken in turn. What weighs less than 2^-127 has no part in a result, but no number has."""
    if form == "eights" and cache == 8:
        return
    T = 40 if form in ("prompt", "pairs") else 2
    k = torch.zeros(PAGES, G, P, D // 2 if cache == 4 else D, dtype=U8 if cache == 4 else torch.int8, device="cuda")
    k[high * 4:high * 4 + 4, ..., 0] = 8                       # pages of the block
    v = torch.ones_like(k)
    one = torch.ones(PAGES, G, P, device="cuda") if cache == 4 else torch.ones(PAGES, G, device="cuda")
    ks, vs = (kv4.words_of(64 * one, 0 * one), kv4.words_of(one, 0 * one)) if cache == 4 else (64 * one, one.clone())
    table = torch.arange(PAGES, dtype=I32, device="cuda")[None]
    q = torch.zeros(T, 8, D, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    start, lens = kv4.i32([0, T]), kv4.i32([N])
    work = ops.kv4_attention_workspace("cuda") if cache == 4 else ops.kv8_attention_workspace("cuda")

    def run(ks, vs, table):
        out, case = torch.full_like(q, 3.0), (q, k, v, ks, vs, table, start, lens)
        if cache == 4:
            kv4.attend("rows" if form == "eights" else form, *case, out, LN2, work, max_tokens={"rows": 20, "eights": 1}.get(form, T))
        elif form == "rows":
            ops.kv8_attention(*case, out, LN2, work, max_tokens=T)
        else:
            kv8.prompt_form(*case, out, LN2, work, pairs=form == "pairs")
        return out
    assert torch.isfinite(run(ks, vs, table)).all()
    for block in range(PAGES // 4):
        if block == high:
            continue
        ks2, vs2, table2 = ks.clone(), vs.clone(), table.clone()
        page = block * 4 + 1                                   # (all tokens see it, and the other pages of its block)
        if what == "page":
            table2[0, page] = -1
        else:
            (ks2 if what == "key" else vs2)[page] = 0xff03 - 65536 if cache == 4 else float("inf")
        assert run(ks2, vs2, table2).isnan().all(), block


@pytest.mark.parametrize("form", ["rows", "eights", "prompt", "pairs"])
@pytest.mark.parametrize("cache", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("query", [float("nan"), float("inf")])
def test_rows_that_see_nothing_are_zeros_whatever_their_queries_are(query, dtype, cache, form):
    """More tokens than keys: those in front of the first key. Others with such a query are no numbers, and their neighbours are right."""
    make, work = (kv4.make_attention, ops.kv4_attention_workspace) if cache == 4 else (kv8.make_attention, ops.kv8_attention_workspace)
    q, *rest = make(3, [20, 130, 0], [60, 70, 5], 8, 2, D, P, dtype)
    outs = []
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for spoil in (False, True):
        x, out = q.clone(), torch.full_like(q, 3.0)
        if spoil:
            for at, head in ((0, 0), (7, 5), (39, 3), (40, 2), (59, 7), (100, 1), (131, 4)):   # (the first 40 tokens, and the last five, see nothing)
                x[at, head, 5] = query
                bad[at, head] = 40 <= at < 130
        case = (x, *rest, out, D ** -0.5, work("cuda"))
        if cache == 4:
            kv4.attend("rows" if form == "eights" else form, *case, max_tokens=1 if form == "eights" else None)
        elif form in ("rows", "eights"):
            ops.kv8_attention(*case, max_tokens=1 if form == "eights" else None)
        else:
            kv8.prompt_form(*case, pairs=form == "pairs")
        outs.append(out)
    assert not outs[1][:40].any() and not outs[1][130:].any()
    assert outs[1].isnan().all(2).equal(bad) and outs[1].isnan().any(2).equal(bad)
    # (an infinite reference takes its warp's rows the way that is for references far from zero: their last bits may differ, within the bounds that either way has)
    want, bound = (kv4 if cache == 4 else kv8).attention_in_64_bits(q, *rest, D ** -0.5)
    assert ((outs[1].double() - want).abs() <= bound)[~bad].all()
    assert query == float("inf") or torch.equal(outs[1][~bad], outs[0][~bad])


@pytest.mark.parametrize("form", ["rows", "eights", "prompt", "pairs"])
@pytest.mark.parametrize("cache", [4, 8])
def test_rows_that_see_nothing_are_zeros_over_scores_beyond_float32(cache, form):
    make, work = (kv4.make_attention, ops.kv4_attention_workspace) if cache == 4 else (kv8.make_attention, ops.kv8_attention_workspace)
    q, k, v, ks, vs, table, start, lens = make(4, [20, 130], [60, 70], 8, 2, D, P, torch.bfloat16, q_scale=1e30)
    ks = ((ks.to(I32) & 0xffff) + (60 << 8)).clamp(max=0xfe00).to(torch.int16) if cache == 4 else ks * 2.0 ** 60
    out = torch.full_like(q, 3.0)
    case = (q, k, v, ks, vs, table, start, lens, out, D ** -0.5, work("cuda"))
    if cache == 4:
        kv4.attend("rows" if form == "eights" else form, *case, max_tokens=1 if form == "eights" else None)
    elif form in ("rows", "eights"):
        ops.kv8_attention(*case, max_tokens=1 if form == "eights" else None)
    else:
        kv8.prompt_form(*case, pairs=form == "pairs")
    assert not out[:40].any()
