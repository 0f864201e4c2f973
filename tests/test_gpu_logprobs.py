"""Log probabilities of given tokens, entropy, ranks and best alternatives on the GPU, against 64 bits and sorts."""
import math

import pytest
import torch

from qspec_b200 import ops

pytestmark = pytest.mark.gpu
F16, BF16, F32, F64, I64 = torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def call(logits, tokens, top, temperature=1.0):
    n = logits.shape[0]
    lp, h = torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    rank = torch.full((n,), -7, device="cuda")
    tlp, tt = torch.full((n, top), 7.0, device="cuda"), torch.full((n, top), -7, device="cuda")
    ops.token_logprobs(logits, tokens, lp, h, rank, *((tlp, tt) if top else (None, None)), temperature=temperature)
    return lp, h, rank, tlp, tt


def check(logits, tokens, top, temperature=1.0):
    """A value y = c (x - max) is rounded once, by 2^-24 |y|, c by 2^-24 of itself, and so is what a weight's exponent gets; weights are off by 2^-22 (ex2.approx) and that; sums of V
    terms in float32, in trees over V / 2048 terms at most one after the other, by (V / 2048 + 16) 2^-24; the logarithm by 2^-22. So a log probability is off by 2^-22 |lp| and
    what log S is off by; the entropy by that and, U / S being an average of |y| <= Y, by the weights' errors times Y (terms beyond e^-40 of the largest have none)."""
    lp, h, rank, tlp, tt = call(logits, tokens, top, temperature)
    z = logits.double() / temperature
    p = torch.log_softmax(z, -1)
    V = logits.shape[1]
    off = (V / 2048 + 16) * 2.0 ** -24 + 2.0 ** -21 + 40 * 2.0 ** -23
    want = p.gather(1, tokens[:, None])[:, 0]
    assert ((lp - want).abs() <= want.abs() * 2.0 ** -22 + off).all(), float((lp - want).abs().max())
    entropy = -torch.special.xlogy(p.exp(), p.exp()).sum(-1)
    assert ((h - entropy).abs() <= entropy * 2.0 ** -20 + off * 41).all(), float((h - entropy).abs().max())
    assert torch.equal(rank, (logits > logits.gather(1, tokens[:, None])).sum(-1) + 1)
    best = logits.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(tt, best)
    want = p.gather(1, best)
    assert ((tlp - want).abs() <= want.abs() * 2.0 ** -22 + off).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 33), (5, 1024), (1, 4096), (7, 8193), (4, 32001), (33, 50257), (2, 128256), (3, 151643), (1, 262144)])
@pytest.mark.parametrize("top", [0, 1, 5, 8, 9, 32])
def test_of_logits_as_models_give_them(rows, V, dtype, top):
    logits = (torch.randn(rows, V, generator=gen(V), device="cuda") * 3).to(dtype)
    check(logits, torch.randint(0, V, (rows,), generator=gen(1), device="cuda"), min(top, V), 0.7 if top == 5 else 1.0)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", ["up", "down", "equal", "two", "steep", "masked", "blocks"])
@pytest.mark.parametrize("V", [1000, 40000, 130001])
def test_of_rows_that_are_out_of_the_ordinary(shape, V, dtype):
    at = torch.arange(V, device="cuda")
    x = {"up": at / V, "down": -at / V, "equal": torch.full((V,), 2.5, device="cuda"), "two": (at % 2).float(), "steep": -at.float().clamp(max=60000),
         "masked": torch.where(at % 7000 == 17, at / V, -math.inf), "blocks": torch.where(at < V // 2, 0.0, torch.where(at > V * 3 // 4, -math.inf, 4.0))}[shape]
    logits = x.to(dtype).repeat(3, 1)
    lp, h, rank, tlp, tt = call(logits, torch.tensor([17, 17, 17], device="cuda"), 20)
    best = logits.sort(dim=-1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(tt, best)
    p = torch.log_softmax(logits.double(), -1)
    want = p.gather(1, best)
    # (sums of V equal terms, V / 2048 of them one after the other)
    torch.testing.assert_close(tlp.double(), want, rtol=2.0 ** -20, atol=(V / 2048 + 60) * 2.0 ** -23)
    torch.testing.assert_close(lp.double(), p[:, 17], rtol=2.0 ** -20, atol=(V / 2048 + 60) * 2.0 ** -23)
    torch.testing.assert_close(h.double(), -torch.special.xlogy(p.exp(), p.exp()).sum(-1), rtol=2.0 ** -18, atol=(V / 2048 + 60) * 2.0 ** -20)
    assert torch.equal(rank, (logits > logits[:, 17:18]).sum(-1) + 1)


def test_zeros_of_either_sign_are_equal():
    logits = torch.zeros(2, 5000, device="cuda")
    logits[0, ::2] = -0.0
    logits[1, 1::2] = -0.0
    assert call(logits, torch.zeros(2, dtype=I64, device="cuda"), 6)[4].tolist() == [list(range(6))] * 2


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [100, 70000])
def test_rows_of_nothing_of_infinity_and_of_no_numbers(dtype, V):
    logits = torch.randn(6, V, generator=gen(3), device="cuda").to(dtype)
    logits[1] = -math.inf
    logits[2, 50] = math.inf
    logits[3, 60] = math.nan
    logits[4, :] = -math.inf
    logits[4, 99] = 3.0
    tokens = torch.tensor([7, 7, 50, 7, 99, 7], device="cuda")
    clean = call(logits[5:], tokens[5:], 4)
    lp, h, rank, tlp, tt = call(logits, tokens, 4)
    assert lp[1] == -math.inf and h[1] == 0 and (tlp[1] == -math.inf).all() and tt[1].tolist() == [0, 1, 2, 3] and rank[1] == 1
    for row, first in ((2, 50), (3, 60)):
        assert lp[row].isnan() and h[row].isnan() and tlp[row].isnan().all() and tt[row, 0] == first
        assert tt[row].tolist() == logits[row].sort(descending=True, stable=True).indices[:4].tolist()
    assert lp[4] == 0 and h[4] == 0 and rank[4] == 1 and tt[4].tolist() == [99, 0, 1, 2] and (tlp[4, 1:] == -math.inf).all()
    assert all(torch.equal(a[5:], b) for a, b in zip((lp, h, rank, tlp, tt), clean))


def test_tokens_that_are_none():
    logits = torch.randn(4, 3000, generator=gen(4), device="cuda").half()
    lp, h, rank, _, _ = call(logits, torch.tensor([-1, 3000, 2999, -100], device="cuda"), 0)
    assert lp[0] == 0 and lp[3] == 0 and lp[1] == -math.inf and lp[2] < 0 and rank.tolist()[0:2] == [0, 0] and rank[2] > 0 and rank[3] == 0 and (h > 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V,stride,shift", [(5001, 5001, 0), (5001, 5003, 1), (70001, 70007, 3), (70000, 70016, 8), (128, 1000, 5)])
def test_rows_that_begin_anywhere(V, stride, shift, dtype):
    wide = torch.full((7, stride + 16), 100.0, device="cuda").to(dtype)   # what stands beside a row is larger than all in it
    logits = wide.view(-1)[shift:shift + 6 * stride].view(6, stride)[:, :V]
    logits.copy_(torch.randn(6, V, generator=gen(5), device="cuda"))
    check(logits, torch.randint(0, V, (6,), generator=gen(6), device="cuda"), 10)


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0, 30.0])
def test_temperatures(temperature):
    logits = torch.randn(5, 33000, generator=gen(7), device="cuda")
    lp, h, rank, tlp, tt = call(logits, logits.argmax(-1), 3, temperature)
    p = torch.log_softmax(logits.double() / temperature, -1)
    # (c is rounded by 2^-24, products by as much: relative errors of log probabilities)
    torch.testing.assert_close(tlp.double(), p.topk(3).values, rtol=2.0 ** -21, atol=80 * 2.0 ** -23)
    assert (rank == 1).all()


def test_results_that_are_not_wanted_and_calls_of_nothing():
    logits = torch.randn(9, 20000, generator=gen(8), device="cuda").half()
    tokens = torch.randint(0, 20000, (9,), generator=gen(9), device="cuda")
    lp, h, rank, tlp, tt = call(logits, tokens, 5)
    for only in range(4):
        out = [torch.zeros_like(t) for t in (lp, h, rank, tlp, tt)]
        want = (lp, h, rank, tlp, tt)
        wanted = [(0,), (1,), (2,), (3, 4)][only]
        ops.token_logprobs(logits, tokens if only in (0, 2) else None, *[out[i] if i in wanted else None for i in range(5)])
        assert all(torch.equal(out[i], want[i]) for i in wanted)
    ops.token_logprobs(logits[:0], tokens[:0], lp[:0])
    ops.token_logprobs(logits, tokens)


def test_the_same_every_time_in_a_graph_and_on_other_streams():
    logits = (torch.randn(70, 128256, generator=gen(10), device="cuda") * 3).half()
    tokens = logits.argmax(-1)
    want = call(logits, tokens, 20)
    out = [torch.zeros_like(t) for t in want]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.token_logprobs(logits, tokens, *out)
    for _ in range(5):
        for t in out:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[torch.zeros_like(t) for t in want] for _ in range(2)]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            ops.token_logprobs(logits, tokens, *o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_what_is_refused():
    x, t = torch.zeros(3, 100, device="cuda"), torch.zeros(3, dtype=I64, device="cuda")
    lp, tlp, tt = torch.zeros(3, device="cuda"), torch.zeros(3, 4, device="cuda"), torch.zeros(3, 4, dtype=I64, device="cuda")
    ops.token_logprobs(x, t, lp, lp.clone(), t.clone(), tlp, tt)
    for args, kw in (((x.double(), t, lp), {}), ((x.t(), t, lp), {}), ((x[0], t, lp), {}), ((x, t.int(), lp), {}), ((x, t[:2], lp), {}), ((x, t, lp.half()), {}), ((x, t, lp[:2]), {}),
                     ((x, None, lp), {}), ((x, None, None, None, t), {}), ((x, t, lp, None, None, tlp), {}), ((x, t, lp, None, None, tlp, tt[:, :3].contiguous()), {}),
                     ((x, t, lp), dict(temperature=0.0)), ((x, t, lp), dict(temperature=-1.0)), ((x, t, lp), dict(temperature=math.nan)), ((x, t, lp), dict(temperature=math.inf)),
                     ((x, t, lp), dict(temperature=1e-40)), ((x, t, lp, lp), {}), ((x, t, x[0, :3]), {}), ((x, t, None, None, t), {}),
                     ((x, t, None, None, None, torch.zeros(3, 33, device="cuda"), torch.zeros(3, 33, dtype=I64, device="cuda")), {}),
                     ((x[:, :3].contiguous(), t, None, None, None, tlp, tt), {}), ((x[:, :0], t, lp), {})):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args, **kw)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", ["random", "rising", "ties", "few larger ones in every batch", "up"])
@pytest.mark.parametrize("top", [1, 5, 8, 9])
def test_best_of_long_rows_that_a_cta_has_to_itself(shape, top, dtype):
    """Spans of more than eight batches: the best are first brought up to date in their middle, from candidates of many batches."""
    rows, V = 600, 140003
    at = torch.arange(V, device="cuda")
    x = torch.randn(V, generator=gen(5), device="cuda")
    x = {"random": 3 * x, "rising": x + at / 30000, "ties": (3 * x).round(), "up": at / V,
         "few larger ones in every batch": torch.where(at % 2001 == 1000, 6.0 + at // 40000 + (at // 2001 % 3) / 4, x)}[shape].to(dtype)
    logits = x.roll(11)[None].repeat(rows, 1)
    logits[1::2] = logits[1::2].roll(977, 1)
    tokens = torch.randint(0, V, (rows,), generator=gen(2), device="cuda")
    _, _, rank, tlp, tt = call(logits, tokens, top)
    for row in (0, 1):                                        # the even rows are alike, and the odd ones
        best = logits[row].sort(descending=True, stable=True).indices[:top]
        assert torch.equal(tt[row::2], best.expand(rows // 2, top)), row
        p = torch.log_softmax(logits[row].double(), -1)[best]
        assert ((tlp[row::2] - p).abs() <= p.abs() * 2.0 ** -22 + (V / 2048 + 16) * 2.0 ** -24 + 2.0 ** -21 + 40 * 2.0 ** -23).all()
        assert torch.equal(rank[row::2], (logits[row] > logits[row, tokens[row::2]][:, None]).sum(-1) + 1)


@pytest.mark.parametrize("dtype,V", [(F16, 128256), (BF16, 90007), (F32, 151643)])
@pytest.mark.parametrize("top", [5, 9, 20, 32])
def test_best_of_rows_whose_larger_values_come_after_batches_without_any(top, dtype, V):
    """A CTA has a row to itself and walks it in batches of 16 KB. The best so far are all in the first batch, batches 1 to 3 have none (so that a look at the candidates finds nothing), larger
    ones come from batch 4 on, in some batches and not in others."""
    rows, batch = 600, 16384 // torch.empty(0, dtype=dtype).element_size()
    at = torch.arange(V, device="cuda")
    x = torch.rand(rows, V, generator=gen(13), device="cuda")
    x[:, :batch:97] += 4
    for b in range(4, V // batch):                            # odd rows: three in each of them; even ones: in every third
        x[1::2, b * batch + 500:b * batch + 503] = 8 + b / 4
        if b % 3 == 0:
            x[::2, b * batch + batch - 40:b * batch + batch - 3] = 6 + b / 8
    x[:, (at % 5000 == 4999) & (at > 10 * batch)] += 7.5
    logits = x.to(dtype)
    best = logits.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    for _ in range(5):
        lp, h, rank, tlp, tt = call(logits, best[:, 1].contiguous(), top)
        assert torch.equal(tt, best)
        assert torch.equal(rank, (logits > logits.gather(1, best[:, 1:2])).sum(-1) + 1)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [3, 600])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("gap", [8, 20, 30])
def test_of_rows_that_are_sure_of_a_token_wherever_it_stands(gap, temperature, rows, dtype):
    """The best token is `gap` nats above the next ones, at the begin, in the middle, at the end of a row or anywhere. Its log probability is - ln S, S = 1 + the others' weights, of which the
    sum is R: never above zero. Off by R times the weights' errors (2^-22 of ex2.approx, and a rounding each of the difference, of c and of the product, at exponents up to 2 gap / T * 1.4427 where there is
    weight: 2^-17 at most), by the logarithm's last place (2^-22 of itself), and by sums: 1 and more plus t, rounded to the nearest, is off by 2^-24 at most (half a last place) and by t at
    most (1 itself is a float, and no sum rounds past it). The terms t of the thread and pair that the 1 is in are V / 256 / 2 values at most and then 21 joins with other threads and spans, and
    together no more than R: the smaller of (V / 512 + 21) 2^-24 and R. The entropy, a sum of positive terms: by its own 2^-17 and what the logarithm is off by, and U by its roundings, 2^-24 of U each."""
    V = 60007
    logits = (torch.rand(rows, V, generator=gen(17), device="cuda") * 2 - 2).to(dtype)
    at = torch.randint(0, V, (rows,), generator=gen(18), device="cuda")
    at[:3] = torch.tensor([0, V // 2, V - 1], device="cuda")
    logits.scatter_(1, at[:, None], torch.full_like(logits[:, :1], gap * temperature))
    lp, h, rank, tlp, tt = call(logits, at, 5, temperature)
    p = torch.log_softmax(logits.double() / temperature, -1)
    top = p.gather(1, at[:, None])[:, 0]
    R = torch.expm1(-top)
    sums = torch.clamp(R, max=(V / 512 + 21) * 2.0 ** -24)
    bound = R * 2.0 ** -17 + top.abs() * 2.0 ** -22 + sums
    assert (lp <= 0).all() and (tlp <= 0).all() and (h >= 0).all() and (rank == 1).all()
    assert ((lp - top).abs() <= bound).all(), float(((lp - top).abs() / bound).max())
    assert torch.equal(tlp[:, 0], lp) and torch.equal(tt[:, 0], at)
    entropy = -torch.special.xlogy(p.exp(), p.exp()).sum(-1)
    assert ((h - entropy).abs() <= entropy * (2.0 ** -17 + (V / 512 + 21) * 2.0 ** -24) + 2 * bound).all(), float((h - entropy).abs().max())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V,top", [(1, 1), (2, 2), (7, 3), (33, 32), (5000, 8), (70000, 9)])
def test_a_first_token_that_is_no_number_is_the_best(V, top, dtype):
    """Like no numbers elsewhere in a row: the first one of them first; all of a row, and one of a kind."""
    logits = torch.randn(5, V, generator=gen(19), device="cuda").to(dtype)
    logits[0, 0] = math.nan
    logits[1, 0], logits[1, V - 1] = math.nan, math.nan
    logits[2] = math.nan
    logits[3, 0] = math.inf
    logits[4] = -math.inf
    logits[4, 0] = math.nan
    lp, h, rank, tlp, tt = call(logits, torch.zeros(5, dtype=I64, device="cuda"), top)
    assert torch.equal(tt, logits.sort(dim=-1, descending=True, stable=True).indices[:, :top])
    assert lp.isnan().all() and h.isnan().all() and tlp.isnan().all() and (rank == 1).all()
