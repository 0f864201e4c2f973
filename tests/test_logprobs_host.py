"""Refusals of the log probabilities' entry points that need no GPU."""
import math

import pytest
import torch

from qspec_b200 import _lib, ops

P = 1 << 20                       # stands for a pointer, never followed


@pytest.fixture(scope="module")
def lib():
    return _lib.load_seq()


def call(lib, logits=P, stride=1000, tokens=P, logprobs=P, entropy=P, ranks=P, top_logprobs=P, top_tokens=P, rows=3, V=1000, top=5, temperature=1.0, dtype=0):
    return lib.qspec_seq_token_logprobs(logits, stride, tokens, logprobs, entropy, ranks, top_logprobs, top_tokens, rows, V, top, temperature, dtype, None)


@pytest.mark.parametrize("kw,what", [(dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(top_logprobs=None), "null"), (dict(top_tokens=None), "null"), (dict(rows=-1), "rows="),
                                     (dict(V=0), "vocabulary"), (dict(stride=999), "stride"), (dict(top=-1), "best"), (dict(top=33), "best"), (dict(V=4, top=5), "best"),
                                     (dict(dtype=3), "float16"), (dict(dtype=2, logits=P + 2), "boundaries"), (dict(logits=P + 1), "boundaries"), (dict(tokens=P + 4), "boundaries"),
                                     (dict(V=(1 << 24) + 1, stride=1 << 25), "too large"),
                                     *((dict(temperature=t), "temperature") for t in (0.0, -1.0, math.nan, math.inf, 1e-40))])
def test_refusals(lib, kw, what):
    status = call(lib, **kw)
    text = lib.qspec_last_error().decode()
    assert status in (1, 2) and what in text, (status, text)


def test_no_rows_are_no_error(lib):
    assert call(lib, rows=0) == 0


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64), torch.zeros(2))
    assert ops.max_top_logprobs() == 32
