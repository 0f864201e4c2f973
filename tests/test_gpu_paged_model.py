"""The int4 decoder over the paged 8-bit cache, and speculative decoding with rejection sampling: page plan, append, attention and verification as one run."""
import math

import pytest
import torch

from qspec_b200 import ops
from qspec_b200.engine import QSpecEngine
from qspec_b200.model import QSpecLlamaConfig, QSpecLlamaModel
from qspec_b200.paged import PagedKV8Cache
from qspec_b200.scheduler import Scheduler

pytestmark = pytest.mark.gpu


def config(**kw):
    return QSpecLlamaConfig.tiny(max_seq_len=256, **kw)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("page", [16, 64, 128])
def test_a_pass_over_the_8_bit_cache_is_near_one_over_the_16_bit_cache(page):
    """A code is off by a step / sqrt(12) as a root mean square, and a step is amax / 127: at pages whose largest of 2048 to 16384 values is up to 4.2 spreads 1 % of a
    spread, and 1.3 times that where a page's older rows went through a scale that grew. Keys and values each, in two layers, the second's input being the
    first's result: 0.01 * 1.3 * sqrt(2) * 2 = 3.7 % of the hidden states at most."""
    B, P, n = 3, 70, 4
    ids = torch.randint(0, 1000, (B, P + n), generator=torch.Generator().manual_seed(1)).cuda()
    models = [QSpecLlamaModel(config(kv_cache=kind, kv_page=page), max_batch=B, max_tokens=B * (P + n), seed=3) for kind in ("f16", "int8")]
    at = lambda lo, hi: torch.arange(lo, hi, dtype=torch.int32, device="cuda").repeat(B)  # noqa: E731
    seq = lambda m: torch.arange(B, dtype=torch.int32, device="cuda").repeat_interleave(m)  # noqa: E731
    cache = models[1].paged
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    step = cache.plan(zero, zero + P, B * P, P)
    cache.commit()
    outs = [models[0].forward(ids[:, :P].reshape(-1), at(0, P), seq(P), w4a4=False).clone(), models[1].forward(ids[:, :P].reshape(-1), None, None, w4a4=False, step=step).clone()]
    assert rel(outs[1], outs[0]) < 0.037
    for w4a4 in (True, False):                                # a draft-shaped and a verify-shaped pass over the same positions
        step = cache.plan(zero + P, zero + n, B * n, n)
        cache.commit()
        outs = [models[0].forward(ids[:, P:].reshape(-1), at(P, P + n), seq(n), w4a4=w4a4).clone(),
                models[1].forward(ids[:, P:].reshape(-1), None, None, w4a4=w4a4, step=step).clone()]
        if w4a4:
            # int4 activations next to a border fall on either side: a difference of 1 % of the spread moves 2 % of the values by a step of 0.45 of it, 6 % of the
            # vector, and there are eight quantisers in a row. What the first layer writes does not depend on attention: it is the same.
            for b in range(B):
                for got, want in zip(cache.read(0, b, P + n), (models[0].cache_k[0, b, :P + n], models[0].cache_v[0, b, :P + n])):
                    assert rel(got[P:], want[P:]) < 0.03
        else:
            assert rel(outs[1], outs[0]) < 0.037
    # what the cache holds is what the other cache holds, to half a step of each page's scale and what older rows lost when it grew
    for layer in range(2):
        for b in range(B):
            for got, want in zip(cache.read(layer, b, P), (models[0].cache_k[layer, b, :P], models[0].cache_v[layer, b, :P])):
                assert rel(got, want) < 0.03
    assert cache.refused() == 0


def test_steps_of_the_operators_together_against_64_bits():
    """Requests come, grow by drafts of which some are refused, and end, over a shared pool; after every step attention over the pages equals attention over the
    rows that were written, in 64 bits, as far as their codes go."""
    B, H, G, D, P, k = 5, 8, 2, 128, 32, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = PagedKV8Cache(1, G, D, B, 400, B * 120, "cuda", page_tokens=P, pages=40)
    cs = torch.rand(400, D, generator=g, device="cuda").half()
    rows = {b: None for b in range(B)}                        # 16-bit keys and values of each request, rotated
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    for turn in range(12):
        counts = [(90 + 10 * b if turn == b % 3 else 0) if rows[b] is None else (-1 if (turn + b) % 7 == 6 else k + 1) for b in range(B)]
        T = sum(max(c, 0) for c in counts)
        if T == 0:
            continue
        step = cache.plan(lengths, torch.tensor(counts, dtype=torch.int32, device="cuda"), T, max(counts))
        cache.commit()
        qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device="cuda").half()
        q, out = torch.empty(T, H, D, dtype=torch.float16, device="cuda"), torch.empty(T, H, D, dtype=torch.float16, device="cuda")
        cache.append(0, qkv, cs, step, q)
        cache.attend(0, q, step, out, D ** -0.5)
        start = 0
        for b, c in enumerate(counts):
            if c < 0:
                rows[b] = None
                lengths[b] = 0
                continue
            if c == 0:
                continue
            n = int(lengths[b]) + c
            keys, values = (t.double() for t in cache.read(0, b, n))
            x = qkv[start:start + c].double().view(c, H + 2 * G, D)
            c0, s0 = cs[n - c:n].double()[:, None].chunk(2, -1)
            lo, hi = x[:, H:H + G].chunk(2, -1)
            new_k, new_v = torch.cat((lo * c0 - hi * s0, hi * c0 + lo * s0), -1), x[:, H + G:]
            held = rows[b] if rows[b] is not None else (new_k[:0], new_v[:0])
            rows[b] = (torch.cat([held[0][:n - c], new_k]), torch.cat([held[1][:n - c], new_v]))
            for got, want in zip((keys, values), rows[b]):
                assert rel(got, want) < 0.03                  # codes: a step is amax / 127
            for h in range(H):
                z = q[start:start + c, h].double() @ keys[:, h // 4].T * D ** -0.5
                hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - c, n, device="cuda")[:, None]
                want = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ values[:, h // 4]
                # (the reader rounds a code's value to float16 once more: 2^-11)
                assert (out[start:start + c, h].double() - want).abs().max() < 4e-3
            start += c
            taken = c if c > k + 1 else 1 + (turn + b) % (k + 1)   # drafts that were refused are written over in the next step
            lengths[b] += taken
            rows[b] = tuple(t[:int(lengths[b])] for t in rows[b])
    assert cache.refused() == 0
    held = cache.state.tolist()
    assert sum(held) == 40 and all(h * P >= n for h, n in zip(held, lengths.tolist()))


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("graph", [False, True])
def test_speculative_decoding_over_the_8_bit_cache(temperature, graph):
    B, k, P = 4, 3, 20
    model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16), max_batch=B, max_tokens=B * (k + 1), seed=5)
    model.make_modes_agree(6)                                 # drafts that are accepted now and then
    engine = QSpecEngine(model, B, k, use_cuda_graph=graph, temperature=temperature, seed=11)
    prompts = torch.randint(0, 1000, (B, P), generator=torch.Generator().manual_seed(2)).cuda()
    runs = []
    for _ in range(2):
        if temperature:
            engine.generator.manual_seed(11)
        engine.prefill(prompts)
        first = engine.cur_tok.tolist()
        got = [[] for _ in range(B)]
        for _ in range(8):
            engine.step()
            engine.stream.synchronize()
            for b, (row, n) in enumerate(zip(engine.out_tokens.tolist(), engine.out_count.tolist())):
                assert 1 <= n <= k + 1 and all(t >= 0 for t in row[:n]) and all(t == -1 for t in row[n:])
                got[b] += row[:n]
        assert engine.seq_len.tolist() == [P + len(t) for t in got]
        m = engine.metrics()
        assert m["emitted_tokens"] == sum(map(len, got)) and model.paged.refused() == 0
        runs.append((first, got))
    assert runs[0] == runs[1]                                 # the same random numbers, the same tokens; no page of the first run is left behind
    assert model.paged.free() + sum(model.paged.state.tolist()[:-1]) == model.paged.pages


def test_sampling_at_a_low_temperature_is_greedy():
    B, k, P = 2, 2, 9
    out = []
    for temperature in (0.0, 1e-4):
        model = QSpecLlamaModel(config(), max_batch=B, max_tokens=B * (k + 1), seed=6)
        engine = QSpecEngine(model, B, k, use_cuda_graph=True, temperature=temperature)
        engine.prefill(torch.arange(B * P, device="cuda").view(B, P))
        tokens = [engine.cur_tok.tolist()]
        for _ in range(5):
            engine.step()
            engine.stream.synchronize()
            tokens.append((engine.out_tokens.tolist(), engine.out_count.tolist()))
        out.append(tokens)
    assert out[0] == out[1]


def test_the_scheduler_serves_from_pages_and_gets_them_back():
    """More requests than slots, over a pool of fewer pages than every slot at its longest: the same tokens as with room for everyone, and none left held."""
    prompts = [list(range(3 + i, 3 + i + 5 + 11 * i)) for i in range(6)]
    model = QSpecLlamaModel(config(), max_batch=3, max_tokens=64, seed=7)
    assert model.n_slots == 3
    texts = []
    for pages in (None, 15):                                  # 256 / 16 = 16 pages would be one slot's
        model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=pages), max_batch=3, max_tokens=64, seed=7)
        s = Scheduler(model, prefill_portion=13)
        texts.append(s.generate(prompts, 7))
        model.paged.plan(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3,), -1, dtype=torch.int32, device="cuda"), 0)
        model.paged.commit()
        assert model.paged.free() == model.paged.pages and model.paged.refused() == 0
    assert texts[0] == texts[1] and all(len(t) == 7 for t in texts[0])


def test_a_pool_that_is_too_small_is_reported():
    model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=3), max_batch=2, max_tokens=64, seed=8)
    with pytest.raises(RuntimeError, match="full"):
        Scheduler(model).generate([list(range(40)), list(range(40))], 20)
    engine = QSpecEngine(QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=3), max_batch=2, max_tokens=64, seed=8), 2, 3)
    engine.prefill(torch.arange(46, device="cuda").view(2, 23))   # two pages each
    with pytest.raises(RuntimeError, match="no page"):
        engine.step()
    with pytest.raises(RuntimeError, match="no page"):
        engine.metrics()


def test_what_the_model_and_the_engine_refuse():
    with pytest.raises(ValueError, match="kv_cache"):
        QSpecLlamaModel(config(kv_cache="int4"), max_batch=1, max_tokens=8)
    with pytest.raises(ValueError, match="pages of"):
        QSpecLlamaModel(config(kv_cache="int8", kv_page=24), max_batch=1, max_tokens=8)
    with pytest.raises(ValueError, match="Hadamard"):
        QSpecLlamaModel(config(kv_cache="int8", qk_hadamard=True), max_batch=1, max_tokens=8)
    model = QSpecLlamaModel(config(kv_cache="int8"), max_batch=2, max_tokens=8)
    with pytest.raises(ValueError, match="step of that cache"):
        model.forward(torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), w4a4=False)
    with pytest.raises(ValueError, match="max_step_tokens"):
        model.paged.plan(torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), 9)
    with pytest.raises(ValueError, match="sequences"):
        QSpecEngine(model, 1, 3)
    for t in (-1.0, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            QSpecEngine(model, 2, 3, temperature=t)


def test_a_step_that_found_no_pages_is_made_again_once_there_are_some():
    """What is refused costs nothing: neither pages nor what the other sequences hold, nor the steps behind it."""
    texts = [list(range(40)), list(range(100, 140)), list(range(200, 220))]
    logits = {}
    for pages in (None, 5):
        model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=pages), max_batch=3, max_tokens=64, seed=8)
        s = Scheduler(model)
        got = [s.feed([("a", texts[0], [39])]), s.feed([("c", texts[2], [19])])]     # three pages, two pages
        if pages:
            for _ in range(2):
                with pytest.raises(RuntimeError, match="full"):
                    s.feed([("b", texts[1], [39])])
                assert model.paged.free() == 0 and model.paged.state.tolist() == [3, 2, 0, 0]
        got.append(s.feed([("c", [7, 8], [1])]))              # a step that needs no page
        if pages:
            with pytest.raises(RuntimeError, match="full"):
                s.feed([("c", list(range(20)), [19]), ("a", [5], [0])])
        s.release("a")
        got += [s.feed([("b", texts[1], [39])]), s.feed([("c", [9], [0]), ("b", [3, 4], [1])])]
        logits[pages] = torch.cat(got)
        assert model.paged.refused() == 0
    assert torch.equal(logits[None], logits[5])


def test_pages_of_requests_that_an_earlier_scheduler_left_come_back():
    model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=4), max_batch=3, max_tokens=64, seed=8)
    left = Scheduler(model)
    left.feed([("a", list(range(10)), []), ("b", list(range(10)), []), ("c", list(range(10)), [])])   # three of the four pages
    want = Scheduler(QSpecLlamaModel(config(kv_cache="int8", kv_page=16), max_batch=3, max_tokens=64, seed=8)).generate([list(range(50))], 6)
    assert Scheduler(model).generate([list(range(50))], 6) == want


@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("graph", [False, True])
def test_a_sequence_without_a_page_emits_nothing_and_stays_where_it_is(graph, temperature):
    """Three pages: after a step that needs two more, the second sequence has no place for its tokens. Once there is one it goes on; a new prefill begins with all pages."""
    B, k, P = 2, 3, 14
    model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=3), max_batch=B, max_tokens=32, seed=8)
    engine = QSpecEngine(model, B, k, use_cuda_graph=graph, temperature=temperature)
    prompts = torch.arange(B * P, device="cuda").view(B, P)
    engine.prefill(prompts)
    token = engine.cur_tok.tolist()
    before = [t.clone() for t in model.paged.read(0, 1, P)]
    for _ in range(3):
        engine.step()
        engine.stream.synchronize()
        assert engine.out_count[0] >= 1 and engine.out_count[1] == 0 and engine.out_tokens[1].tolist() == [-1] * (k + 1)
        assert engine.seq_len[1] == P and engine.cur_tok[1] == token[1] and engine.d_out_pack[1].tolist() == [-1] * (k + 1) + [0]
        if engine.seq_len[0] > 27:
            break
    assert model.paged.state.tolist() == [2, 1, 0]
    with pytest.raises(RuntimeError, match="no page"):
        engine.metrics()
    assert all(torch.equal(a, b) for a, b in zip(before, model.paged.read(0, 1, P)))
    # the first sequence ends: its pages are there for the second
    model.paged.plan(engine.seq_len, torch.tensor([-1, 0], dtype=torch.int32, device="cuda"), 0)
    model.paged.commit()
    engine.seq_len[0] = 0
    engine.step()
    engine.stream.synchronize()
    assert engine.out_count[1] >= 1 and engine.seq_len[1] == P + engine.out_count[1]
    # a new prefill, with room enough
    for e in (engine, QSpecEngine(QSpecLlamaModel(config(kv_cache="int8", kv_page=16), max_batch=B, max_tokens=32, seed=8), B, k, use_cuda_graph=graph, temperature=temperature)):
        if temperature:
            e.generator.manual_seed(3)
        e.prefill(prompts[:, :6])
        e.step()
        e.stream.synchronize()
        assert e.metrics()["emitted_tokens"] == int(e.out_count.sum())
        if e is engine:
            kept = e.out_tokens.clone()
    assert torch.equal(kept, e.out_tokens)


def test_a_prompt_without_pages_is_reported_by_the_next_step_whatever_came_before():
    model = QSpecLlamaModel(config(kv_cache="int8", kv_page=16, kv_pages=3), max_batch=2, max_tokens=64, seed=8)
    engine = QSpecEngine(model, 2, 3, use_cuda_graph=False)
    engine.prefill(torch.arange(8, device="cuda").view(2, 4))
    engine.step()
    engine.prefill(torch.arange(80, device="cuda").view(2, 40))
    with pytest.raises(RuntimeError, match="no page"):
        engine.step()
    engine.prefill(torch.arange(8, device="cuda").view(2, 4))
    engine.step()
    engine.stream.synchronize()
    assert engine.out_count.min() >= 1 and engine.metrics()["draft_tokens"] == 6


@pytest.mark.parametrize("kv_cache", ["f16", "int8"])
def test_what_is_read_back_is_behind_the_steps_that_are_queued(kv_cache):
    """Lengths, refusals and counters are read, and a new prefill is begun, while a step has yet to run (the engine's stream is kept busy for some tenths of a second)."""
    kw = dict(kv_cache="int8", kv_page=16, kv_pages=3) if kv_cache == "int8" else {}
    model = QSpecLlamaModel(config(**kw), max_batch=2, max_tokens=32, seed=8)
    engine = QSpecEngine(model, 2, 3)
    prompts = torch.arange(28, device="cuda").view(2, 14)

    def late_step():
        with torch.cuda.stream(engine.stream):
            torch.cuda._sleep(400_000_000)
        engine.step()

    engine.prefill(prompts[:, :5])
    engine.step()
    engine.stream.synchronize()
    before = engine.seq_len.max().item()
    late_step()
    assert engine.sync_lengths() > before and engine.sync_lengths() == engine.seq_len.max().item()
    late_step()
    steps = engine.metrics()["draft_tokens"]
    assert steps == 3 * 2 * 3
    late_step()
    engine.prefill(prompts)                                   # behind that step, whose lengths and pages are not the new sequences'
    engine.stream.synchronize()
    torch.cuda.synchronize()
    assert engine.seq_len.tolist() == [14, 14]
    if kv_cache == "int8":
        assert model.paged.state.tolist() == [1, 1, 1] and model.paged.refused() == 0
        engine._steps = 1
        late_step()                                           # a page for one of the two
        engine._steps = 64
        with pytest.raises(RuntimeError, match="no page"):
            engine.step()


def test_reading_more_of_a_request_than_it_can_hold_is_refused_on_the_host():
    cache = PagedKV8Cache(2, 2, 64, 3, 40, 8, "cuda", page_tokens=16)
    for tokens in (49, -1, 1 << 30):
        with pytest.raises(ValueError, match="read:"):
            cache.read(0, 0, tokens)
    for tokens in (0, 1, 48):
        k, v = cache.read(-1, 2, tokens)
        assert k.shape == v.shape == (tokens, 2, 64)
    torch.cuda.synchronize()


def test_temperatures_next_to_zero():
    model = QSpecLlamaModel(config(), max_batch=2, max_tokens=8, seed=6)
    for t in (1e-34, 5e-324):
        with pytest.raises(ValueError, match="temperature"):
            QSpecEngine(model, 2, 3, temperature=t)
    tokens = []
    for t in (0.0, 1e-33, 1e30):
        engine = QSpecEngine(model, 2, 3, use_cuda_graph=False, temperature=t)
        engine.prefill(torch.arange(12, device="cuda").view(2, 6))
        engine.step()
        engine.stream.synchronize()
        tokens.append([engine.cur_tok.tolist(), engine.out_tokens.tolist()])
    assert tokens[0] == tokens[1] and tokens[2] != tokens[0]


@pytest.mark.parametrize("kv_cache", ["f16", "int8"])
@pytest.mark.parametrize("temperature", [0.0, 1e-4])
def test_an_engine_without_drafts_decodes_token_by_token(kv_cache, temperature):
    model = QSpecLlamaModel(config(kv_cache=kv_cache, kv_page=16), max_batch=2, max_tokens=8, seed=6)
    engine = QSpecEngine(model, 2, 0, temperature=temperature)
    engine.prefill(torch.arange(12, device="cuda").view(2, 6))
    got = [engine.cur_tok.tolist()]
    for _ in range(4):
        engine.step()
        engine.stream.synchronize()
        assert engine.out_count.tolist() == [1, 1]
        got.append(engine.out_tokens[:, 0].tolist())
    want = Scheduler(QSpecLlamaModel(config(kv_cache=kv_cache, kv_page=16), max_batch=2, max_tokens=8, seed=6)).generate([list(range(6)), list(range(6, 12))], 5)
    assert [list(t) for t in zip(*got)] == want


def test_more_drafts_than_are_verified_are_refused_when_the_engine_is_made():
    model = QSpecLlamaModel(config(), max_batch=1, max_tokens=40, seed=6)
    with pytest.raises(ValueError, match="at most 31"):
        QSpecEngine(model, 1, 32, temperature=0.5)
    QSpecEngine(model, 1, 32)
    engine = QSpecEngine(model, 1, 31, use_cuda_graph=False, temperature=0.5)
    engine.prefill(torch.arange(6, device="cuda").view(1, 6))
    engine.step()
    engine.stream.synchronize()
    assert 1 <= int(engine.out_count) <= 32


def test_tokens_from_the_host_come_behind_what_the_caller_has_queued():
    """A prefill that has yet to run must not write its own last tokens over those that `step_host` brings."""
    results = []
    for late in (False, True):
        model = QSpecLlamaModel(config(), max_batch=2, max_tokens=32, seed=8)
        engine = QSpecEngine(model, 2, 3)
        prompts = torch.arange(12, device="cuda").view(2, 6)
        engine.prefill(prompts)
        engine.capture()                                      # (waits for everything, once)
        tokens = torch.tensor([400, 500])
        if late:
            torch.cuda._sleep(400_000_000)
        engine.prefill(prompts)
        if not late:
            torch.cuda.synchronize()
        results.append(engine.step_host(tokens).clone())
    assert torch.equal(*results)
