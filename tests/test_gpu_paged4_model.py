"""The int4 decoder over the paged 4-bit cache, and log probabilities of what models emit: page plan, append, attention, verification and scores as one run."""
import json
import math

import pytest
import torch

from qspec_b200 import ops
from qspec_b200.engine import QSpecEngine
from qspec_b200.model import QSpecLlamaConfig, QSpecLlamaModel
from qspec_b200.paged import PagedKV4Cache
from qspec_b200.scheduler import Scheduler

pytestmark = pytest.mark.gpu


def config(**kw):
    return QSpecLlamaConfig.tiny(max_seq_len=256, **({"kv_cache": "uint4", "kv_page": 16} | kw))


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def turn_back(k):
    """The Hadamard matrix / sqrt(D) is its own inverse."""
    x, s = k.double(), 1
    while s < x.shape[-1]:
        a, b = x.unflatten(-1, (-1, 2, s)).unbind(-2)
        x = torch.stack((a + b, a - b), -2).flatten(-3)
        s *= 2
    return x * x.shape[-1] ** -0.5


@pytest.mark.parametrize("page", [16, 64, 128])
def test_a_pass_over_the_4_bit_cache_is_near_one_over_the_16_bit_cache(page):
    """A step is a row's range / 15, up to 1/32 more, and a range of 128 normal values is 5.3 spreads (6.5 in one row of a hundred): a code is off by 6.5 / 15 * 1.04 / sqrt(12) =
    13 % of a spread as a root mean square. Attention averages over keys, so that the first layer's result is off by less; two layers and two sides: sqrt(2) * 2 * 13 % at most."""
    B, P, n = 3, 70, 4
    ids = torch.randint(0, 1000, (B, P + n), generator=torch.Generator().manual_seed(1)).cuda()
    models = [QSpecLlamaModel(config(kv_cache=kind, kv_page=page), max_batch=B, max_tokens=B * (P + n), seed=3) for kind in ("f16", "uint4")]
    at = lambda lo, hi: torch.arange(lo, hi, dtype=torch.int32, device="cuda").repeat(B)  # noqa: E731
    seq = lambda m: torch.arange(B, dtype=torch.int32, device="cuda").repeat_interleave(m)  # noqa: E731
    cache = models[1].paged
    assert isinstance(cache, PagedKV4Cache) and cache.hadamard
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    step = cache.plan(zero, zero + P, B * P, P)
    cache.commit()
    outs = [models[0].forward(ids[:, :P].reshape(-1), at(0, P), seq(P), w4a4=False).clone(), models[1].forward(ids[:, :P].reshape(-1), None, None, w4a4=False, step=step).clone()]
    assert rel(outs[1], outs[0]) < 0.37
    step = cache.plan(zero + P, zero + n, B * n, n)
    cache.commit()
    outs = [models[0].forward(ids[:, P:].reshape(-1), at(P, P + n), seq(n), w4a4=False).clone(), models[1].forward(ids[:, P:].reshape(-1), None, None, w4a4=False, step=step).clone()]
    assert rel(outs[1], outs[0]) < 0.37
    for b in range(B):                                        # the first layer writes the same keys and values
        k, v = cache.read(0, b, P + n)
        assert rel(turn_back(k), models[0].cache_k[0, b, :P + n]) < 0.14 and rel(v, models[0].cache_v[0, b, :P + n]) < 0.14
    assert cache.refused() == 0


def test_drafts_leave_nothing_behind():
    """A verify pass gives the same, bit for bit, whether its rows were written by a draft before or not: every row has a scale of its own."""
    B, P, n = 2, 30, 4
    ids = torch.randint(0, 1000, (B, P + n), generator=torch.Generator().manual_seed(2)).cuda()
    outs = []
    for draft in (False, True):
        model = QSpecLlamaModel(config(), max_batch=B, max_tokens=B * (P + n), seed=3)
        zero = torch.zeros(B, dtype=torch.int32, device="cuda")
        step = model.paged.plan(zero, zero + P, B * P, P)
        model.paged.commit()
        model.forward(ids[:, :P].reshape(-1), None, None, w4a4=False, step=step)
        step = model.paged.plan(zero + P, zero + n, B * n, n)
        model.paged.commit()
        if draft:
            model.forward(ids[:, :n].reshape(-1), None, None, w4a4=True, step=step)
        outs.append(model.forward(ids[:, P:].reshape(-1), None, None, w4a4=False, step=step).clone())
    assert torch.equal(*outs)


def test_steps_of_the_operators_together_against_64_bits():
    """Requests come, grow by drafts of which some are refused, and end, over a shared pool; after every step attention over the pages equals attention over the rows that
    they hold, in 64 bits."""
    B, H, G, D, P, k = 5, 8, 2, 128, 32, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = PagedKV4Cache(1, G, D, B, 400, B * 120, "cuda", page_tokens=P, pages=40)
    cs = torch.rand(400, D, generator=g, device="cuda").half()
    alive = [False] * B
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    for turn in range(12):
        counts = [(90 + 10 * b if turn == b % 3 else 0) if not alive[b] else (-1 if (turn + b) % 7 == 6 else k + 1) for b in range(B)]
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
                alive[b] = False
                lengths[b] = 0
            if c <= 0:
                continue
            alive[b] = True
            n = int(lengths[b]) + c
            keys, values = (t.double() for t in cache.read(0, b, n))
            x = qkv[start:start + c].double().view(c, H + 2 * G, D)
            assert rel(values[n - c:], x[:, H + G:]) < 0.14   # (a code is off by 13 % of a spread)
            for h in range(H):
                z = q[start:start + c, h].double() @ keys[:, h // 4].T * D ** -0.5
                hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - c, n, device="cuda")[:, None]
                want = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ values[:, h // 4]
                # (the reader gives a code's value exactly: nine bits; weights are off by 2^-11, the result by 2^-11)
                assert (out[start:start + c, h].double() - want).abs().max() < 4e-3
            start += c
            lengths[b] += c if c > k + 1 else 1 + (turn + b) % (k + 1)   # drafts that were refused are written over in the next step
    assert cache.refused() == 0
    held = cache.state.tolist()
    assert sum(held) == 40 and all(h * P >= n for h, n in zip(held, lengths.tolist()))


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("graph", [False, True])
def test_speculative_decoding_over_the_4_bit_cache(temperature, graph):
    B, k, P = 4, 3, 20
    model = QSpecLlamaModel(config(), max_batch=B, max_tokens=B * (k + 1), seed=5)
    model.make_modes_agree(6)                                 # drafts that are accepted now and then
    engine = QSpecEngine(model, B, k, use_cuda_graph=graph, temperature=temperature, seed=11, logprobs=3)
    prompts = torch.randint(0, 1000, (B, P), generator=torch.Generator().manual_seed(2)).cuda()
    runs = []
    for _ in range(2):
        if temperature:
            engine.generator.manual_seed(11)
        engine.prefill(prompts)
        got = [engine.cur_tok.tolist()]
        for _ in range(6):
            engine.step()
            engine.stream.synchronize()
            got.append([t.tolist() for t in (engine.out_tokens, engine.out_count, engine.out_logprobs, engine.out_ranks, engine.out_entropy, engine.out_top_logprobs, engine.out_top_tokens)])
        assert engine.metrics()["emitted_tokens"] == sum(sum(s[1]) for s in got[1:]) and model.paged.refused() == 0
        runs.append(got)
    assert runs[0] == runs[1]                                 # the same random numbers, the same tokens and scores
    assert model.paged.free() + sum(model.paged.state.tolist()[:-1]) == model.paged.pages


def test_pages_of_the_4_bit_cache_through_the_scheduler():
    prompts = [list(range(3 + i, 3 + i + 5 + 11 * i)) for i in range(6)]
    texts = []
    for pages in (None, 15):                                  # 256 / 16 = 16 pages would be one slot's
        model = QSpecLlamaModel(config(kv_pages=pages), max_batch=3, max_tokens=64, seed=7)
        texts.append(Scheduler(model, prefill_portion=13).generate(prompts, 7))
        model.paged.plan(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3,), -1, dtype=torch.int32, device="cuda"), 0)
        model.paged.commit()
        assert model.paged.free() == model.paged.pages and model.paged.refused() == 0
    assert texts[0] == texts[1] and all(len(t) == 7 for t in texts[0])
    with pytest.raises(RuntimeError, match="4-bit cache is full"):
        Scheduler(QSpecLlamaModel(config(kv_pages=3), max_batch=2, max_tokens=64, seed=8)).generate([list(range(40)), list(range(40))], 20)


def test_the_variant_with_turned_queries_and_keys_takes_the_4_bit_cache():
    """The Hadamard matrix of queries and keys that the model has anyway is the cache's: the same scores as over 16-bit rows, but for the cache's codes (13 % of a spread)."""
    ids = torch.randint(0, 1000, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    outs = []
    for kind in ("f16", "uint4"):
        model = QSpecLlamaModel(config(kv_cache=kind, qk_hadamard=True), max_batch=1, max_tokens=40, seed=3)
        step = None
        if kind == "uint4":
            step = model.paged.plan(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 40, dtype=torch.int32, device="cuda"), 40, 40)
            model.paged.commit()
        at = torch.arange(40, dtype=torch.int32, device="cuda")
        outs.append(model.forward(ids, *((None, None) if step else (at, torch.zeros_like(at))), w4a4=False, step=step).clone())
    assert rel(outs[1], outs[0]) < 0.37


# ---- log probabilities of what is emitted ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv_cache", ["f16", "uint4"])
@pytest.mark.parametrize("temperature", [0.0, 0.6])
def test_scores_of_a_step_are_those_of_its_logits(temperature, kv_cache, monkeypatch):
    B, k = 3, 2
    model = QSpecLlamaModel(config(kv_cache=kv_cache), max_batch=B, max_tokens=16, seed=5)
    model.make_modes_agree(5)
    engine = QSpecEngine(model, B, k, use_cuda_graph=False, temperature=temperature, logprobs=4)
    seen = []
    logits = model.logits
    monkeypatch.setattr(model, "logits", lambda h: seen.append(logits(h)) or seen[-1])
    engine.prefill(torch.arange(B * 5, device="cuda").view(B, 5))
    for _ in range(4):
        engine.step()
        engine.stream.synchronize()
        z = seen[-1].double().view(B, k + 1, -1) / (temperature or 1.0)   # (the verification's are a step's last)
        p = torch.log_softmax(z, -1)
        for b in range(B):
            n = int(engine.out_count[b])
            tokens = engine.out_tokens[b, :n]
            want = p[b, :n].gather(1, tokens[:, None])[:, 0]
            torch.testing.assert_close(engine.out_logprobs[b, :n].double(), want, rtol=2.0 ** -20, atol=2.0 ** -18)
            assert engine.out_ranks[b, :n].tolist() == [1 + int((z[b, i] > z[b, i, t]).sum()) for i, t in enumerate(tokens.tolist())]
            assert (engine.out_logprobs[b, n:] == 0).all() and (engine.out_ranks[b, n:] == 0).all()
        assert torch.equal(engine.out_top_tokens, z.sort(dim=-1, descending=True, stable=True).indices[..., :4])
        torch.testing.assert_close(engine.out_entropy.double(), -(p.exp() * p).sum(-1), rtol=2.0 ** -18, atol=2.0 ** -18)
        if not temperature:
            assert all(engine.out_ranks[b, int(engine.out_count[b]) - 1] == 1 for b in range(B))


def test_an_engine_without_scores_is_what_it_was():
    got = []
    for n in (None, 0, 2):
        model = QSpecLlamaModel(config(), max_batch=2, max_tokens=16, seed=5)
        engine = QSpecEngine(model, 2, 3, temperature=0.8, seed=3, logprobs=n)
        engine.prefill(torch.arange(10, device="cuda").view(2, 5))
        for _ in range(3):
            engine.step()
        engine.stream.synchronize()
        got.append(engine.out_tokens.tolist())
        assert hasattr(engine, "out_logprobs") == (n is not None)
    assert got[0] == got[1] == got[2]
    for n in (-1, 33):
        with pytest.raises(ValueError, match="logprobs"):
            QSpecEngine(model, 2, 3, logprobs=n)


@pytest.mark.parametrize("kv_cache", ["f16", "int8", "uint4"])
def test_a_text_is_scored_as_its_logits_say(kv_cache):
    model = QSpecLlamaModel(config(kv_cache=kv_cache), max_batch=2, max_tokens=16, seed=7)
    texts = [torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (40, 2, 1, 17)]
    s = Scheduler(model)
    scores = s.score(texts, top=3)
    assert s.table.pool.free == model.n_slots
    for text, got in zip(texts, scores):
        assert [x.token for x in got] == text[1:]
        if len(text) == 1:
            continue
        # (the same portions: in 8 bits a page's scale is that of the rows that came with it)
        parts = [text[at:min(at + 16, len(text) - 1)] for at in range(0, len(text) - 1, 16)]
        logits = torch.cat([s.feed([("again", part, list(range(len(part))))]) for part in parts]).double()
        s.release("again")
        p = torch.log_softmax(logits, -1)
        for i, x in enumerate(got):
            assert abs(x.logprob - float(p[i, x.token])) < 1e-4 and x.rank == 1 + int((logits[i] > logits[i, x.token]).sum())
            assert [t for t, _ in x.top] == logits[i].sort(descending=True, stable=True).indices[:3].tolist()
            assert abs(x.entropy + float((p[i].exp() * p[i]).sum())) < 1e-4
    with pytest.raises(ValueError, match="empty"):
        s.score([[]])
    with pytest.raises(ValueError, match="best"):
        s.score([[1, 2]], top=33)
    with pytest.raises(RuntimeError, match="cache takes"):
        s.score([[1] * 300])
    assert s.table.pool.free == model.n_slots


def test_generated_tokens_come_with_scores_for_those_who_want_them():
    model = QSpecLlamaModel(config(), max_batch=3, max_tokens=32, seed=7)
    prompts = [[1, 2, 3], [9, 8, 7, 6], [30] * 20]
    want = Scheduler(model).generate(prompts, 5)
    s = Scheduler(model)
    for i, (p, n) in enumerate(zip(prompts, (None, 0, 4))):
        s.add(i, p, 5, logprobs=n)
    while s.has_work():
        s.step()
    assert [s.finished[i].output for i in range(3)] == want
    assert s.finished[0].scores == [] and [x.token for x in s.finished[1].scores] == want[1] and all(x.top == [] and x.rank == 1 for x in s.finished[1].scores)
    for x in s.finished[2].scores:
        assert len(x.top) == 4 and x.top[0] == (x.token, x.logprob) and x.logprob < 0 and x.entropy > 0
    with pytest.raises(ValueError, match="best"):
        s.add("more", [1], 5, logprobs=40)


def test_the_command_scores_and_generates(tmp_path, capsys):
    from qspec_b200.__main__ import main
    (tmp_path / "config.json").write_text(json.dumps(dict(architectures=["LlamaForCausalLM"], hidden_size=512, intermediate_size=28 * 64, num_attention_heads=4, num_key_value_heads=2,
                                                          head_dim=128, num_hidden_layers=2, vocab_size=1024, max_position_embeddings=128)))
    argv = ["--model", str(tmp_path), "--prompt", "5,17,3,9", "--slots", "2", "--step-tokens", "16"]
    for kv in ("f16", "uint4"):
        assert main(["score", *argv, "--top", "2", "--kv-cache", kv]) == 0
        line = json.loads(capsys.readouterr().out)
        assert [s["token"] for s in line["scores"]] == [17, 3, 9] and all(len(s["top"]) == 2 for s in line["scores"])
        assert math.isclose(line["perplexity"], math.exp(-sum(s["logprob"] for s in line["scores"]) / 3))
        assert main(["generate", *argv, "--max-new-tokens", "4", "--logprobs", "0", "--kv-cache", kv]) == 0
        line = json.loads(capsys.readouterr().out)
        assert [s["token"] for s in line["scores"]] == line["tokens"] and len(line["tokens"]) == 4
    assert main(["generate", *argv, "--max-new-tokens", "4"]) == 0
    assert set(json.loads(capsys.readouterr().out)) == {"prompt", "tokens"}


def test_what_is_refused():
    with pytest.raises(ValueError, match="pages of"):
        QSpecLlamaModel(config(kv_page=24), max_batch=1, max_tokens=8)
    with pytest.raises(ValueError, match="4-bit cache takes heads"):
        PagedKV4Cache(1, 2, 96, 1, 64, 8, "cuda")
    cache = PagedKV4Cache(2, 2, 64, 3, 40, 8, "cuda", page_tokens=16, hadamard=False)
    for tokens in (49, -1):
        with pytest.raises(ValueError, match="read:"):
            cache.read(0, 0, tokens)
    k, v = cache.read(-1, 2, 48)
    assert k.shape == v.shape == (48, 2, 64) and not k.any()
    assert ops.max_top_logprobs() == 32


@pytest.mark.parametrize("kv_cache", ["f16", "int8", "uint4"])
@pytest.mark.parametrize("temperature", [0.0, 0.6])
@pytest.mark.parametrize("n", [0, 4])
def test_the_first_token_has_scores_as_well(n, temperature, kv_cache, monkeypatch):
    """What a prefill emits: with the steps' scores behind it, those of the whole of a generated text."""
    B = 3
    model = QSpecLlamaModel(config(kv_cache=kv_cache), max_batch=B, max_tokens=16, seed=5)
    engine = QSpecEngine(model, B, 2, temperature=temperature, logprobs=n, seed=2)
    seen, logits = [], model.logits
    monkeypatch.setattr(model, "logits", lambda h: seen.append(logits(h)) or seen[-1])
    for first in (0, 50):                                     # a second prefill writes over the first one's
        engine.prefill(torch.arange(first, first + B * 5, device="cuda").view(B, 5))
        z = seen[-1].double() / (temperature or 1.0)
        assert z.shape[0] == B
        p = torch.log_softmax(z, -1)
        torch.testing.assert_close(engine.first_logprobs.double(), p.gather(1, engine.cur_tok[:, None])[:, 0], rtol=2.0 ** -20, atol=2.0 ** -18)
        torch.testing.assert_close(engine.first_entropy.double(), -(p.exp() * p).sum(-1), rtol=2.0 ** -18, atol=2.0 ** -18)
        assert torch.equal(engine.first_ranks, 1 + (z > z.gather(1, engine.cur_tok[:, None])).sum(-1))
        assert torch.equal(engine.first_top_tokens, z.sort(dim=-1, descending=True, stable=True).indices[:, :n])
        torch.testing.assert_close(engine.first_top_logprobs.double(), p.gather(1, engine.first_top_tokens), rtol=2.0 ** -20, atol=2.0 ** -18)
        if not temperature:
            assert (engine.first_ranks == 1).all()
    other = QSpecEngine(QSpecLlamaModel(config(kv_cache=kv_cache), max_batch=B, max_tokens=16, seed=5), B, 2, temperature=temperature, seed=2)
    for first in (0, 50):
        other.prefill(torch.arange(first, first + B * 5, device="cuda").view(B, 5))
    assert torch.equal(other.cur_tok, engine.cur_tok) and not hasattr(other, "first_logprobs")


def test_scores_are_read_with_the_tokens():
    """A step with scores reads the device as often as one without."""
    from torch.profiler import ProfilerActivity, profile
    reads = []
    for n in (None, 0, 5):
        s = Scheduler(QSpecLlamaModel(config(), max_batch=3, max_tokens=32, seed=7))
        for i, p in enumerate(([1, 2, 3], [9, 8, 7, 6], [30] * 20)):
            s.add(i, p, 8, logprobs=n)
        for _ in range(3):
            s.step()
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            for _ in range(2):
                s.step()
            torch.cuda.synchronize()
        reads.append(sum("DtoH" in e.name for e in prof.events()))
    assert reads[0] > 0 and reads == reads[:1] * 3, reads
