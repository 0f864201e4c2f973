"""What the engine does with logits, on the host."""
import types

import pytest
import torch

from qspec_b200.engine import QSpecEngine


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_probabilities_leave_logits_that_are_given_as_they_are(dtype):
    logits = torch.randn(5, 33, generator=torch.Generator().manual_seed(1)).to(dtype)
    engine = types.SimpleNamespace(temperature=0.5, model=types.SimpleNamespace(logits=lambda hidden: logits.clone()))
    kept = logits.clone()
    given, own = QSpecEngine._probs(engine, None, logits=logits), QSpecEngine._probs(engine, None)
    assert torch.equal(logits, kept) and torch.equal(given, own) and torch.equal(own, torch.softmax(kept.float() * 2, -1))
    out = torch.empty(5, 33)
    assert QSpecEngine._probs(engine, None, out, logits).data_ptr() == out.data_ptr() and torch.equal(out, own) and torch.equal(logits, kept)
