"""Log probabilities in the scheduler's bookkeeping: whose they are, how many, once each, over a model and an operator on the host."""
import types

import pytest
import torch

from qspec_b200 import scheduler
from qspec_b200.scheduler import Scheduler
from test_scheduler_host import PROMPTS, Counting


def token_logprobs(logits, tokens, logprobs, entropy, ranks, top_logprobs=None, top_tokens=None, temperature=1.0):
    p = torch.log_softmax(logits.double() / temperature, -1)
    given = p.gather(1, tokens[:, None])
    logprobs.copy_(given[:, 0])
    entropy.copy_(-(p.exp() * p).sum(-1))
    ranks.copy_((p > given).sum(-1) + 1)
    if top_tokens is not None:
        best = p.sort(dim=-1, descending=True, stable=True).indices[:, :top_tokens.shape[1]]
        top_tokens.copy_(best)
        top_logprobs.copy_(p.gather(1, best))


@pytest.fixture(autouse=True)
def host_operators(monkeypatch):
    monkeypatch.setattr(scheduler, "ops", types.SimpleNamespace(argmax_rows=lambda x: x.argmax(-1), token_logprobs=token_logprobs, max_top_logprobs=lambda: 32))


@pytest.mark.parametrize("refuse", [set(), {0}, {1}, {2, 3}, {0, 4, 6, 7}])
def test_every_token_has_one_score_whatever_was_refused(refuse):
    s = Scheduler(Counting(refuse), prefill_portion=9)
    wanted = [3, None, 0]
    for i, p in enumerate(PROMPTS):
        s.add(i, p, 4, logprobs=wanted[i])
    while s.has_work():
        try:
            s.step()
        except RuntimeError:
            pass
    plain = Scheduler(Counting()).generate(PROMPTS, 4)
    for i, top in enumerate(wanted):
        r = s.finished[i]
        assert r.output == plain[i]
        if top is None:
            assert r.scores == []
            continue
        assert [x.token for x in r.scores] == r.output and all(x.rank == 1 and len(x.top) == top for x in r.scores)
        for x in r.scores:                                    # one logit of 1, the others 0
            assert abs(x.logprob - float(torch.log_softmax(torch.tensor([1.0] + [0.0] * 999), 0)[0])) < 1e-5
            assert not top or (x.top[0][0] == x.token and [t for t, _ in x.top[1:]] == [t for t in range(4) if t != x.token][:top - 1])


@pytest.mark.parametrize("portion", [1, 4, 9, 16])
def test_scores_of_texts(portion):
    model = Counting()
    s = Scheduler(model, prefill_portion=portion)
    texts = [[1, 1, 2, 4, 9], [7], list(range(1, 40))]
    scores = s.score(texts, 1)
    assert [len(x) for x in scores] == [4, 0, 38]
    for text, of in zip(texts, scores):
        for i, x in enumerate(of):                            # the model names the sum so far
            total = sum(text[:i + 1])
            assert x.token == text[i + 1] and x.top[0][0] == total and (x.rank == 1) == (total == text[i + 1])
    assert s.generate(PROMPTS, 4) == Scheduler(Counting()).generate(PROMPTS, 4)   # every slot is back


def test_what_is_refused():
    s = Scheduler(Counting())
    for top in (-1, 33):
        with pytest.raises(ValueError):
            s.add("x", [1], 2, logprobs=top)
        with pytest.raises(ValueError):
            s.score([[1, 2]], top)
    with pytest.raises(ValueError):
        s.score([[]])
    assert not s.has_work()


@pytest.mark.parametrize("texts,error", [([[1, 2, 3], []], ValueError), ([[1, 2, 3], [1] * 52], RuntimeError)])
def test_texts_are_looked_at_before_any_is_scored(texts, error):
    model = Counting()
    model.max_seq_len = 50
    s = Scheduler(model)
    with pytest.raises(error):
        s.score(texts)
    assert model.calls == 0 and [len(x) for x in s.score([[1] * 51, [1, 2]])] == [50, 1]


@pytest.mark.parametrize("tokens", [[-1], [1000], [1, 2, 1 << 40], [5, -7, 3]])
def test_tokens_outside_the_vocabulary_are_refused(tokens):
    model = Counting()
    s = Scheduler(model)
    with pytest.raises(ValueError, match="tokens are 0 to 999"):
        s.add("x", tokens, 2)
    with pytest.raises(ValueError, match="tokens are 0 to 999"):
        s.score([[1, 2], tokens])
    with pytest.raises(ValueError, match="tokens are 0 to 999"):
        s.generate([[1], tokens], 2)
    assert model.calls == 0 and not s.has_work() and [x.token for x in s.score([[0, 999]])[0]] == [999]
    assert s.generate(PROMPTS, 3) == Scheduler(Counting()).generate(PROMPTS, 3)
