"""The commands' output, over a scheduler that is none."""
import json
import math
import types

import pytest

from qspec_b200 import __main__ as command
from qspec_b200.scheduler import TokenScore


def strict(line):
    def refuse(name):
        raise ValueError(name)
    return json.loads(line, parse_constant=refuse)


def fake(monkeypatch, scores):
    s = types.SimpleNamespace(score=lambda prompts, top: [scores for _ in prompts],
                              generate_requests=lambda prompts, n, eos, logprobs: [types.SimpleNamespace(output=[1, 2], scores=scores) for _ in prompts])
    monkeypatch.setattr(command, "_scheduler", lambda args, new_tokens: (s, [[3, 1, 2]]))


@pytest.mark.parametrize("logprobs,perplexity", [([-1.0, -3.0], math.exp(2)), ([-1.0, math.nan], None), ([-1.0, -math.inf], None), ([-1000.0, -500.0], None), ([], None)])
def test_scores_are_json_whatever_they_hold(monkeypatch, capsys, logprobs, perplexity):
    fake(monkeypatch, [TokenScore(i, x, 1 + i, x * 0 + 0.5, [(7, x), (8, -0.25)]) for i, x in enumerate(logprobs)])
    assert command.main(["score", "--model", "none", "--prompt", "3,1,2"]) == 0
    line = strict(capsys.readouterr().out)
    assert line["perplexity"] == perplexity and line["prompt"] == [3, 1, 2]
    plain = [x if math.isfinite(x) else None for x in logprobs]
    assert [s["logprob"] for s in line["scores"]] == plain and [s["top"] for s in line["scores"]] == [[[7, x], [8, -0.25]] for x in plain]
    assert [s["entropy"] for s in line["scores"]] == [None if x is None else 0.5 for x in plain]
    assert command.main(["generate", "--model", "none", "--prompt", "3,1,2", "--logprobs", "2"]) == 0
    line = strict(capsys.readouterr().out)
    assert line["tokens"] == [1, 2] and [s["logprob"] for s in line["scores"]] == plain
