"""Verification of drafted tokens with given random numbers, on the GPU -- against fractions and 64-bit sums."""
import math

import pytest
import torch

from qspec_b200 import ops

pytestmark = pytest.mark.gpu
F64, I64 = torch.float64, torch.int64


def make(seed, B, k, V, agree=0.5, sharp=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    target = torch.softmax(torch.randn(B, k + 1, V, generator=g, device="cuda") * sharp, -1)
    if not k:
        return None, None, target, torch.rand(B, 1, generator=g, device="cuda")
    draft = torch.softmax(target[:, :k].log() + torch.randn(B, k, V, generator=g, device="cuda") * sharp * (1 - agree), -1)
    drafted = torch.multinomial(draft.reshape(B * k, V), 1, generator=g).reshape(B, k)
    return drafted, draft, target, torch.rand(B, k + 1, generator=g, device="cuda")


def by_hand(drafted, draft, target, uniform, counts=None):
    """(tokens, emitted, how far the border between tokens is from the random number, as a share of the sum)."""
    B, k = target.shape[0], target.shape[1] - 1
    tokens, emitted, margin = torch.full((B, k + 1), -1, dtype=I64), torch.zeros(B, dtype=I64), torch.ones(B, dtype=F64)
    for b in range(B):
        n = k if counts is None else min(max(int(counts[b]), 0), k)
        taken = 0
        while taken < n:
            d = int(drafted[b, taken])
            if not 0 <= d < target.shape[2] or not float(uniform[b, taken]) * float(draft[b, taken, d]) < float(target[b, taken, d]):
                break
            taken += 1
        p = target[b, taken].to(F64)
        rest = (p - draft[b, taken].to(F64)).clamp(min=0) if taken < n else p
        if not rest.sum() > 0:
            rest = p
        upto = rest.cumsum(0)
        border = float(uniform[b, k]) * float(upto[-1])
        tokens[b, :taken] = drafted[b, :taken] if k else tokens[b, :0]
        tokens[b, taken] = int((upto <= border).sum()) if upto[-1] > 0 else 0
        emitted[b] = taken + 1
        if upto[-1] > 0:
            margin[b] = float((upto - border).abs().min() / upto[-1])
    return tokens, emitted, margin


def run(drafted, draft, target, uniform, counts=None):
    B, k = target.shape[0], target.shape[1] - 1
    tokens, emitted = torch.full((B, k + 1), -9, dtype=I64, device="cuda"), torch.full((B,), -9, dtype=I64, device="cuda")
    ops.verify_drafts(drafted, draft, target, uniform, tokens, emitted, draft_counts=counts)
    return tokens.cpu(), emitted.cpu()


def check(*case, counts=None):
    tokens, emitted, margin = by_hand(*case, counts=counts)
    got = run(*case, counts=counts)
    # 64-bit sums of V terms differ by V * 2^-53 of the sum at most with their order: a random number that is nearer to a border may fall on either side
    clear = margin > case[2].shape[2] * 2.0 ** -52
    assert clear.float().mean() > 0.9
    assert torch.equal(got[1], emitted) and torch.equal(got[0][clear], tokens[clear])
    return got


@pytest.mark.parametrize("B,k,V", [(1, 0, 1), (1, 1, 2), (3, 2, 31), (2, 3, 255), (5, 1, 256), (4, 3, 257), (7, 4, 2049), (64, 3, 4100), (3, 31, 1000), (4, 3, 128256), (2, 5, 151643), (74, 1, 5000), (75, 1, 5000), (90, 2, 128256), (130, 3, 32001)])
def test_verified_tokens_are_those_of_the_rule(B, k, V):
    for seed in range(3):
        check(*make(seed, B, k, V, agree=0.7))


def test_drafts_of_unequal_number():
    case = make(5, 40, 4, 3000, agree=0.9)
    counts = torch.tensor([0, 1, 2, 3, 4, 7, -2, 4] * 5, dtype=torch.int32, device="cuda")
    tokens, emitted = check(*case, counts=counts)
    assert (emitted <= counts.cpu().clamp(0, 4) + 1).all()


def test_a_draft_that_is_the_target_is_always_taken_and_one_that_is_impossible_never():
    drafted, draft, target, uniform = make(6, 20, 3, 1000)
    same = target[:, :3].contiguous()
    drafted = torch.multinomial(same.reshape(60, -1), 1).reshape(20, 3)
    uniform[:, :3] = 1 - 2.0 ** -24
    tokens, emitted = check(drafted, same, target, uniform)
    assert (emitted == 4).all()
    target = target.clone()
    target[:, 1].scatter_(1, drafted[:, 1:2], 0.0)            # the target cannot have said it
    uniform[:, 1] = 0.0
    tokens, emitted = check(drafted, same, target, uniform)
    assert (emitted == 2).all() and (tokens[:, 2:] == -1).all()


def test_rows_with_little_in_them():
    B, V = 8, 5000
    g = torch.Generator(device="cuda").manual_seed(3)
    target = torch.zeros(B, 2, V, device="cuda")
    draft = torch.zeros(B, 1, V, device="cuda")
    drafted = torch.full((B, 1), 17, dtype=I64, device="cuda")
    uniform = torch.rand(B, 2, generator=g, device="cuda")
    draft[:, 0, 17] = 1.0
    target[0, 0, 4999] = 1.0                                  # refused, one token left: the last
    target[1, 0, 0] = 1.0                                     # the first
    target[2, 0, 17], target[2, 1, 300] = 1.0, 1.0            # taken, then a row of one token
    target[3, 0] = 0.0                                        # nothing at all: token 0
    target[4, 0, [5, 6]], draft[4, 0] = 0.5, 1.0              # refused, and nothing over the draft: from the target
    uniform[4] = torch.tensor([0.9, 0.75], device="cuda")
    draft[4, 0, 17] = 1.0
    target[5, 0, 100:200] = 0.01
    uniform[5] = torch.tensor([0.5, 0.0], device="cuda")      # the first with anything
    target[6, 0, 100:200] = 0.01
    uniform[6] = torch.tensor([0.5, 1 - 2.0 ** -24], device="cuda")
    target[7, 0, 100] = math.nan                              # no number counts as none
    target[7, 0, 200] = 0.25
    tokens, emitted = run(drafted, draft, target, uniform)
    assert emitted.tolist() == [1, 1, 2, 1, 1, 1, 1, 1]
    assert tokens[:, 0].tolist() == [4999, 0, 17, 0, 6, 100, 199, 200] and tokens[2, 1] == 300


def test_drafted_tokens_and_random_numbers_outside_their_range():
    drafted, draft, target, uniform = make(9, 6, 2, 700)
    drafted[0, 0], drafted[1, 1] = -1, 700
    uniform[2, 2], uniform[3, 2], uniform[4, 2] = 2.0, -1.0, math.nan
    tokens, emitted = run(drafted, draft, target, uniform)
    assert emitted[0] == 1 and emitted[1] <= 2 and ((tokens >= -1) & (tokens < 700)).all()
    for b in range(6):
        assert (tokens[b, :emitted[b]] >= 0).all() and (tokens[b, emitted[b]:] == -1).all()


def test_strided_rows():
    drafted, draft, target, uniform = make(10, 9, 3, 1001)
    want = run(drafted, draft, target, uniform)
    wide = torch.zeros(9, 5, 1037, device="cuda")
    wide[:, 1:, 3:1004] = target
    pairs = torch.zeros(3, 9, 1001, device="cuda")
    pairs.copy_(draft.transpose(0, 1))
    got = run(drafted, pairs.transpose(0, 1), wide[:, 1:, 3:1004], uniform)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("V", [1, 33, 1024, 32001, 128256])
def test_sampled_tokens(V):
    probs = torch.softmax(torch.randn(50, V, device="cuda") * 2, -1)
    uniform = torch.rand(50, device="cuda")
    got = ops.sample_probs(probs, uniform, torch.empty(50, dtype=I64, device="cuda")).cpu()
    want, _, margin = by_hand(None, None, probs[:, None], uniform[:, None])
    clear = margin > V * 2.0 ** -52
    assert torch.equal(got[clear], want[clear, 0]) and clear.float().mean() > 0.9


def test_what_is_emitted_is_distributed_as_the_target():
    """First tokens over 40,000 requests with one distribution: each count within 5 standard deviations (V = 12 counts: false alarm below 1e-5)."""
    N, V = 40000, 12
    g = torch.Generator(device="cuda").manual_seed(1)
    p, q = (torch.softmax(torch.randn(V, generator=g, device="cuda") * 1.5, -1) for _ in range(2))
    target = p.expand(N, 2, V)
    draft = q.expand(N, 1, V)
    drafted = torch.multinomial(q.expand(N, V), 1, generator=g)
    uniform = torch.rand(N, 2, generator=g, device="cuda")
    tokens, emitted = run(drafted, draft, target, uniform)
    count = torch.bincount(tokens[:, 0], minlength=V).double()
    want = p.cpu().double() * N
    assert ((count - want).abs() <= 5 * (want * (1 - p.cpu().double())).sqrt() + 1).all()
    second = tokens[emitted == 2, 1]                          # the token behind a taken draft is the target's too
    want = p.cpu().double() * len(second)
    assert ((torch.bincount(second, minlength=V).double() - want).abs() <= 5 * want.sqrt() + 1).all()


def test_in_a_graph():
    case = make(12, 16, 3, 9000)
    tokens, emitted = torch.empty(16, 4, dtype=I64, device="cuda"), torch.empty(16, dtype=I64, device="cuda")
    ops.verify_drafts(*case, tokens, emitted)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.verify_drafts(*case, tokens, emitted)
    other = make(13, 16, 3, 9000)
    for a, b in zip(case, other):
        a.copy_(b)
    graph.replay()
    want = run(*other)
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(emitted.cpu(), want[1])


def test_wrong_shapes_types_and_overlaps_are_refused():
    drafted, draft, target, uniform = make(1, 4, 2, 50)
    tokens, emitted = torch.empty(4, 3, dtype=I64, device="cuda"), torch.empty(4, dtype=I64, device="cuda")
    args = [drafted, draft, target, uniform, tokens, emitted]
    for i, bad in ((0, None), (1, None), (0, drafted.int()), (0, drafted[:, :1]), (1, draft.double()), (1, draft[:, :, ::2]), (2, target[0]), (2, target[:, :2]), (2, target.half()),
                   (3, uniform[:, :2]), (4, tokens[:3]), (5, emitted.int()), (4, tokens.t().contiguous().t())):
        with pytest.raises(ValueError):
            ops.verify_drafts(*[bad if j == i else a for j, a in enumerate(args)])
    with pytest.raises(ValueError):
        ops.verify_drafts(drafted, draft, target[:, :1], uniform[:, :1].contiguous(), tokens[:, :1].contiguous(), emitted)
    with pytest.raises(ValueError, match="must not lie over"):
        big = torch.zeros(20, dtype=I64, device="cuda")
        ops.verify_drafts(big[:8].view(4, 2), draft, target, uniform, big[6:18].view(4, 3), emitted)
    with pytest.raises(ValueError):
        ops.verify_drafts(*args, draft_counts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.sample_probs(target[:, 0], uniform[:, 0], emitted)   # (random numbers with a stride)


def test_results_over_other_tensors_of_the_call_are_refused():
    drafted, draft, target, uniform = make(1, 4, 2, 50)
    counts = torch.full((4,), 2, dtype=torch.int32, device="cuda")
    z = lambda n, dtype=I64: torch.zeros(n, dtype=dtype, device="cuda")  # noqa: E731
    args = dict(drafted=drafted, draft_probs=draft, target_probs=target, uniform=uniform, tokens=z(12).view(4, 3), emitted=z(4), draft_counts=counts)
    ops.verify_drafts(**args)
    big = z(40)
    for bad in (dict(tokens=big[:12].view(4, 3), emitted=big[11:15]), dict(emitted=big[:4], drafted=big[3:11].view(4, 2)), dict(tokens=big[4:16].view(4, 3), drafted=big[:8].view(4, 2)),
                dict(emitted=big[:4], uniform=big.view(torch.float32)[7:19].view(4, 3)), dict(tokens=big[:12].view(4, 3), draft_counts=big.view(torch.int32)[20:24])):
        with pytest.raises(ValueError, match="must not lie over"):
            ops.verify_drafts(**{**args, **bad})
    side = dict(tokens=big[:12].view(4, 3), emitted=big[12:16], drafted=big[16:24].view(4, 2))
    side["drafted"].copy_(drafted)
    ops.verify_drafts(**{**args, **side})
    assert torch.equal(side["tokens"], args["tokens"]) and torch.equal(side["emitted"], args["emitted"])
