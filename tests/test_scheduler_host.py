"""The scheduler's bookkeeping where a model refuses a step, over a model that keeps its tokens on the host."""
import types

import pytest
import torch

from qspec_b200 import ops, scheduler
from qspec_b200.scheduler import Scheduler


class Counting:
    """Logits name the sum of all tokens of a request so far; refuses the steps in `refuse` (numbered from 0), and counts every slot's tokens."""
    n_slots, max_step_tokens, vocab_size, device = 2, 16, 1000, "cpu"

    def __init__(self, refuse=()):
        self.refuse, self.calls, self.sums, self.released = set(refuse), 0, {}, []

    def forward_batch(self, ids, meta):
        self.calls += 1
        if self.calls - 1 in self.refuse:
            raise RuntimeError("full")
        rows, at = [], 0
        for rid, slot, first, n in meta.segments:
            total, held = self.sums.get(slot, (0, 0)) if first else (0, 0)
            assert held == first, (rid, held, first)          # every token once, in its place
            for t in ids[at:at + n].tolist():
                total += t
                rows.append(total)
            self.sums[slot] = (total, first + n)
            at += n
        return torch.tensor(rows)[:, None].float()

    def logits(self, hidden):
        return torch.nn.functional.one_hot(hidden[:, 0].long() % self.vocab_size, self.vocab_size).float()

    def release_slot(self, slot):
        self.released.append(slot)


@pytest.fixture(autouse=True)
def host_arg_max(monkeypatch):
    monkeypatch.setattr(scheduler, "ops", types.SimpleNamespace(argmax_rows=lambda x: x.argmax(-1)))
    assert hasattr(ops, "argmax_rows")


PROMPTS = [list(range(1, 30)), [5, 6, 7], list(range(3, 24))]


@pytest.mark.parametrize("refuse", [{0}, {1}, {2, 3}, {0, 4, 6, 7}])
def test_a_refused_step_can_be_made_again(refuse):
    want = Scheduler(Counting()).generate(PROMPTS, 4)
    model = Counting(refuse)
    s = Scheduler(model, prefill_portion=9)
    for i, p in enumerate(PROMPTS):
        s.add(i, p, 4)
    refusals = 0
    while s.has_work():
        try:
            s.step()
        except RuntimeError:
            refusals += 1
    assert refusals == len(refuse) and [s.finished[i].output for i in range(3)] == want


def test_a_request_that_is_given_up_is_not_fed_again():
    model = Counting({1})
    s = Scheduler(model, prefill_portion=9)
    for i, p in enumerate(PROMPTS):
        s.add(i, p, 4)
    s.step()
    with pytest.raises(RuntimeError):
        s.step()
    s.release(0)                                              # one that runs, its prompt half in
    s.release(2)                                              # one that waits
    assert [r.rid for r in s.running] == [1] and not s.waiting and s.table.pool.free == 1
    while s.has_work():
        s.step()
    assert list(s.finished) == [1] and s.finished[1].output == Scheduler(Counting()).generate(PROMPTS[1:2], 4)[0]
    assert len(model.released) >= 2


def test_a_new_scheduler_takes_every_slot_back():
    model = Counting()
    first = Scheduler(model)
    first.add("left", PROMPTS[0], 4)
    first.step()
    model.released.clear()
    Scheduler(model)
    assert sorted(model.released) == [0, 1]
