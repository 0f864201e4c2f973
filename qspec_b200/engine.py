"""QSpec speculative-decode loop around the dual-mode model: k draft passes in W4A4, one verify
pass in W4A16 over the same weights and KV cache, greedy acceptance or rejection sampling.

Mirrors SpecDecodeWorker._run_speculative_decoding_step
(vllm/spec_decode/spec_decode_worker.py:758-858: w4a4=True for the proposer :797-801, w4a4=False
for the MQA scorer :812-813 which scores k+1 tokens per sequence, mqa_scorer.py:65) with greedy
rejection (draft token accepted iff it equals the target argmax), and the metrics of
spec_decode/metrics.py:171-179 (draft_acceptance_rate, system_efficiency).

The whole step (3 x 32 draft layers + 32 verify layers + sampling + acceptance + state update)
is captured once into a CUDA graph (the reference runs ~550 eager launches
per draft step with --enforce_eager); all per-step state lives on the device.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .model import QSpecLlamaModel


class QSpecEngine:
    def __init__(self, model: QSpecLlamaModel, batch: int, k: int = 3, use_cuda_graph: bool = True, temperature: float = 0.0, seed: int = 0, logprobs: Optional[int] = None):
        """temperature 0: greedy, a draft token is accepted iff it is the target's arg max. Above 0: tokens are drawn from softmax(logits / temperature) and draft
        tokens accepted with probability min(1, p / q), so that what is emitted is distributed as the target's own (vllm/model_executor/layers/
        rejection_sampler.py); `seed` decides the random numbers. (Over the 8-bit cache the target depends on the drafts a little: a page's scale does not shrink while its
        first row stands, so that rows of a draft that was refused, or that verification wrote over, may leave the page coarser than without them.)

        logprobs: every step also leaves, on the device, what the target says of the tokens that it emits, under the distribution that they are drawn from (that of the logits if
        greedy): `out_logprobs`, `out_entropy` float32 and `out_ranks` int64 [B, k + 1], and of every place the `logprobs` best tokens, `out_top_logprobs` float32 and
        `out_top_tokens` int64 [B, k + 1, logprobs] (0: none of these; None: nothing); `prefill` leaves the same of the tokens that it emits (cur_tok): `first_logprobs`, `first_entropy`,
        `first_ranks` [B], `first_top_logprobs` and `first_top_tokens` [B, logprobs]. Behind what is emitted (out_count) the log probability and the rank are 0. (The reference gives them
        with its sampler's output, vllm/spec_decode/spec_decode_worker.py.)

        Over a paged cache with fewer pages than all sequences may need, a step may find none for some of them: these emit nothing (out_count 0) and stay where they
        are. `step` raises for that at its first call behind a `prefill` and at every 64th, `metrics` at once; the next `prefill` begins with all pages."""
        self.model, self.B, self.k = model, batch, k
        if not temperature >= 0.0:
            raise ValueError(f"temperature must be 0 (greedy) or positive, got {temperature}")
        if 0.0 < temperature < 1e-33:                                 # (float16 logits, up to 65504, divided by it: beyond float32, and the probabilities no numbers)
            raise ValueError(f"temperature must be 0 (greedy) or at least 1e-33, got {temperature}")
        if temperature and model.tp_size != 1:
            raise NotImplementedError("sampling with a vocab-sharded lm_head")
        if temperature and k > (most := ops.max_verified_drafts()):
            raise ValueError(f"sampling verifies at most {most} draft tokens a step, got k = {k}")
        if logprobs is not None:
            if model.tp_size != 1:
                raise NotImplementedError("log probabilities with a vocab-sharded lm_head")
            most = min(ops.max_top_logprobs(), model.cfg.vocab_size)
            if not 0 <= logprobs <= most:
                raise ValueError(f"logprobs: the best 0 to {most} tokens, got {logprobs}")
        self.temperature, self.n_logprobs = float(temperature), logprobs
        dev = model.device
        B = batch
        assert model.max_tokens >= B * (k + 1)
        self.use_graph = use_cuda_graph
        self.cur_tok = torch.zeros(B, dtype=torch.int64, device=dev)
        self.seq_len = torch.zeros(B, dtype=torch.int32, device=dev)        # tokens already in the KV cache
        self.seq_ids = torch.arange(B, dtype=torch.int32, device=dev)
        self.vseq_ids = self.seq_ids.repeat_interleave(k + 1).contiguous()
        self.arange_k1 = torch.arange(k + 1, dtype=torch.int32, device=dev)
        self.draft_toks = torch.zeros(B, k, dtype=torch.int64, device=dev)
        self.out_tokens = torch.zeros(B, k + 1, dtype=torch.int64, device=dev)
        self.out_count = torch.zeros(B, dtype=torch.int64, device=dev)
        # SpecDecodeWorkerMetrics counters (metrics.py): accepted, draft, emitted
        self.counters = torch.zeros(3, dtype=torch.int64, device=dev)
        if logprobs is not None:
            self.out_logprobs, self.out_entropy = torch.zeros(B, k + 1, device=dev), torch.zeros(B, k + 1, device=dev)
            self.out_ranks = torch.zeros(B, k + 1, dtype=torch.int64, device=dev)
            self.out_top_logprobs = torch.zeros(B, k + 1, logprobs, device=dev)
            self.out_top_tokens = torch.zeros(B, k + 1, logprobs, dtype=torch.int64, device=dev)
            self.first_logprobs, self.first_entropy = torch.zeros(B, device=dev), torch.zeros(B, device=dev)
            self.first_ranks = torch.zeros(B, dtype=torch.int64, device=dev)
            self.first_top_logprobs, self.first_top_tokens = torch.zeros(B, logprobs, device=dev), torch.zeros(B, logprobs, dtype=torch.int64, device=dev)
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.stream = torch.cuda.Stream(device=dev)
        # pinned host mirrors for the end-to-end API
        self.h_in = torch.zeros(B, dtype=torch.int64).pin_memory()
        self.h_out = torch.zeros(B, k + 2, dtype=torch.int64).pin_memory()
        self.d_out_pack = torch.zeros(B, k + 2, dtype=torch.int64, device=dev)
        # Host-side upper bound of max(seq_len): the device-resident lengths advance by at most k + 1 per step and are
        # never read back in the loop. A step touches positions seq_len .. seq_len + k of the KV cache and of the
        # rotary table; `step` refuses to run once that could pass cfg.max_seq_len (the kernels index both unchecked
        # apart from a last-resort early-out).
        self._len_bound = 0
        self._steps = 0
        if self.temperature:
            V = model.cfg.vocab_size
            self.generator = torch.Generator(device=dev).manual_seed(seed)
            self.draft_probs = torch.empty(k, B, V, dtype=torch.float32, device=dev)
            self.uniform = torch.empty(2, B, k + 1, dtype=torch.float32, device=dev)     # for the drafts, and for their verification
        self.paged = getattr(model, "paged", None)                    # the model's paged cache, if it has one
        if self.paged is not None:
            self.counts = torch.full((B,), k + 1, dtype=torch.int32, device=dev)
            self.one_each = torch.arange(B + 1, dtype=torch.int32, device=dev)
            if self.paged.requests != B:
                raise ValueError(f"the model's cache holds {self.paged.requests} sequences, the engine has {B}")

    # ---------------------------------------------------------------------------------------
    @torch.no_grad()
    def prefill(self, prompt_ids: torch.Tensor) -> None:
        """prompt_ids [B, P] (device int64). Verify-mode (W4A16) pass, as the reference's
        _run_no_spec prefill (spec_decode_worker.py:666-720); fills the KV cache."""
        m = self.model
        self._behind_steps()
        B, P = prompt_ids.shape
        assert B == self.B and P + 1 < m.cfg.max_seq_len
        pos = torch.arange(P, dtype=torch.int32, device=m.device)
        if self.paged is not None:                                          # the sequences of before give their pages back
            self.paged.plan(torch.zeros_like(self.seq_len), torch.full_like(self.seq_len, -1), 0)
            self.paged.commit()
            self.paged.refusals.zero_()
            self._steps = 0                                                 # (the first step behind this looks whether the prompts found pages)
            held = torch.zeros_like(self.seq_len)
        chunk = max(1, m.max_tokens)
        last_hidden = torch.empty(B, m.cfg.hidden_size, dtype=torch.float16, device=m.device)
        for b in range(B):
            for s in range(0, P, chunk):
                e = min(P, s + chunk)
                ids = prompt_ids[b, s:e].contiguous()
                if self.paged is not None:
                    counts = torch.zeros_like(held)
                    counts[b] = e - s
                    step = self.paged.plan(held, counts, e - s)
                    self.paged.commit()
                    held[b] = e
                    h = m.forward(ids, None, None, w4a4=False, step=step)
                else:
                    h = m.forward(ids, pos[s:e].contiguous(), torch.full((e - s,), b, dtype=torch.int32, device=m.device),
                                  w4a4=False)
                if e == P:
                    last_hidden[b].copy_(h[e - s - 1])
        logits = m.logits(last_hidden) if self.n_logprobs is not None else None
        if self.temperature:
            self.uniform.uniform_(generator=self.generator)
            ops.sample_probs(self._probs(last_hidden, logits=logits), self.uniform[0, :, 0].contiguous(), self.cur_tok)
        else:
            self.cur_tok.copy_(m.greedy_tokens(last_hidden) if logits is None else ops.argmax_rows(logits))
        if logits is not None:
            self._score(logits, self.cur_tok, self.first_logprobs, self.first_entropy, self.first_ranks, self.first_top_logprobs, self.first_top_tokens)
        self.seq_len.fill_(P)
        self._len_bound = P
        self.counters.zero_()

    # ---------------------------------------------------------------------------------------
    def _probs(self, hidden: torch.Tensor, out: Optional[torch.Tensor] = None, logits: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(logits / temperature), float32 [rows, V]. (Logits that are given are the caller's, and stay as they are, in float32 too.)"""
        x = (self.model.logits(hidden) if logits is None else logits).float()
        return torch.softmax(x * (1.0 / self.temperature) if x is logits else x.mul_(1.0 / self.temperature), -1, out=out)

    def _score(self, logits, tokens, logprobs, entropy, ranks, top_logprobs, top_tokens) -> None:
        ops.token_logprobs(logits, tokens, logprobs, entropy, ranks, *((top_logprobs, top_tokens) if self.n_logprobs else (None, None)), temperature=self.temperature or 1.0)

    @torch.no_grad()
    def _spec_step(self) -> None:
        m, B, k = self.model, self.B, self.k
        tok = self.cur_tok
        vstep = None
        if self.paged is not None:
            # one plan for all passes of the step: pages for k + 1 tokens of each sequence, the slots of token i of all of them in row i
            from .paged import PagedStep
            vstep = self.paged.plan(self.seq_len, self.counts, B * (k + 1), k + 1)
            self.paged.commit()
            slots, positions = (t.view(B, k + 1).t().contiguous() for t in (vstep.slots, vstep.positions))
        if self.temperature:
            self.uniform.uniform_(generator=self.generator)
            draws = self.uniform[0].t().contiguous()
        # ---- proposer: k draft passes, w4a4=True (spec_decode_worker.py:797-801)
        for i in range(k):
            if vstep is not None:
                hidden = m.forward(tok, None, None, w4a4=True, step=PagedStep(self.one_each, positions[i] + 1, positions[i], slots[i], None, 1))
            else:
                pos = self.seq_len + i
                hidden = m.forward(tok, pos, self.seq_ids, w4a4=True)
            if self.temperature:
                tok = ops.sample_probs(self._probs(hidden, self.draft_probs[i]), draws[i], torch.empty_like(tok))
            else:
                tok = m.greedy_tokens(hidden)
            self.draft_toks[:, i].copy_(tok)
        # ---- scorer: one verify pass over k+1 tokens / sequence, w4a4=False (:812-813)
        vt = torch.cat((self.cur_tok.unsqueeze(1), self.draft_toks), dim=1).reshape(-1)
        if vstep is not None:
            hidden = m.forward(vt, None, None, w4a4=False, step=vstep)
        else:
            vpos = (self.seq_len.unsqueeze(1) + self.arange_k1.unsqueeze(0)).reshape(-1).contiguous()
            hidden = m.forward(vt, vpos, self.vseq_ids, w4a4=False)
        logits = m.logits(hidden) if self.n_logprobs is not None else None
        if self.temperature:
            drafts = (self.draft_toks, self.draft_probs.transpose(0, 1)) if k else (None, None)
            ops.verify_drafts(*drafts, self._probs(hidden, logits=logits).view(B, k + 1, -1), self.uniform[1], self.out_tokens, self.out_count)
            n_acc, emitted = self.out_count - 1, self.out_tokens
            nxt = emitted.gather(1, n_acc.unsqueeze(1)).squeeze(1)
        else:
            tgt = (m.greedy_tokens(hidden) if logits is None else ops.argmax_rows(logits)).view(B, k + 1)
            # ---- greedy rejection (spec_decode_worker.py:861-915 with temperature 0)
            match = (tgt[:, :k] == self.draft_toks).to(torch.int64)
            n_acc = match.cumprod(dim=1).sum(dim=1)                     # accepted draft tokens per sequence
            nxt = tgt.gather(1, n_acc.unsqueeze(1)).squeeze(1)          # correction / bonus token
            padded = torch.cat((self.draft_toks, nxt.unsqueeze(1)), dim=1)
            idx = self.arange_k1.unsqueeze(0).to(torch.int64)
            emitted = torch.where(idx < n_acc.unsqueeze(1), padded, torch.where(idx == n_acc.unsqueeze(1), nxt.unsqueeze(1), -1))
            self.out_tokens.copy_(emitted)
            self.out_count.copy_(n_acc + 1)
        if vstep is not None:
            # a sequence that found no pages has seen nothing: it emits nothing and stays where it is, so that its step can be made again
            served = vstep.kv_len > 0
            nxt = torch.where(served, nxt, self.cur_tok)
            n_acc = n_acc * served
            emitted = emitted.masked_fill(~served.unsqueeze(1), -1)
            self.out_tokens.copy_(emitted)
            self.out_count.mul_(served)
        if logits is not None:
            self._score(logits, *(t.flatten(0, 1) for t in (self.out_tokens, self.out_logprobs, self.out_entropy, self.out_ranks, self.out_top_logprobs, self.out_top_tokens)))
        count = self.out_count
        self.cur_tok.copy_(nxt)
        self.seq_len.add_(count.to(torch.int32))
        self.counters[0] += n_acc.sum()
        self.counters[1] += B * k
        self.counters[2] += count.sum()
        self.d_out_pack[:, : k + 1].copy_(emitted)
        self.d_out_pack[:, k + 1].copy_(count)

    def capture(self) -> None:
        """Warm up once eagerly (sets kernel attributes, sizes workspaces), then capture."""
        if not self.use_graph or self.graph is not None:
            return
        self._check_capacity()
        def rng(): return self.generator.get_state() if self.temperature else None
        paged = self.paged
        live = [self.cur_tok, self.seq_len, self.counters] + ([] if paged is None else [paged.state, paged.refusals])   # (tables and lists of pages beyond these mean nothing)
        state, draws = [t.clone() for t in live], rng()

        def restore():
            for t, kept in zip(live, state):
                t.copy_(kept)
            if self.temperature:
                self.generator.set_state(draws)
        self._join_caller_stream()
        with torch.cuda.stream(self.stream):
            if paged is not None:
                self.counts.zero_()                        # a step of no tokens: rows that are written over leave their mark in a page's scale
            self._spec_step()
            if paged is not None:
                self.counts.fill_(self.k + 1)
            torch.cuda.synchronize()
            restore()
            g = torch.cuda.CUDAGraph()
            if self.temperature:
                g.register_generator_state(self.generator)
            with torch.cuda.graph(g, stream=self.stream):
                self._spec_step()
            torch.cuda.synchronize()
            restore()
        torch.cuda.synchronize()
        self.graph = g

    def sync_lengths(self) -> int:
        """Reads the true max(seq_len) back (one small D2H copy + sync) and tightens the host-side bound to it."""
        self._behind_steps()
        self._len_bound = int(self.seq_len.max().item())
        return self._len_bound

    def _check_capacity(self) -> None:
        S, need = self.model.cfg.max_seq_len, self.k + 1
        if self._len_bound + need > S:
            self.sync_lengths()                           # the bound assumes every draft token was accepted
            if self._len_bound + need > S:
                raise RuntimeError(f"KV cache exhausted: a sequence holds {self._len_bound} tokens and a speculative step "
                                   f"writes {need} more, but max_seq_len is {S}")
        if self.paged is not None and self._steps % 64 == 0:
            self._check_pages()
        peers = getattr(self.model, "peers", None)
        if peers is not None and self._steps % 64 == 0 and peers.timeouts():
            raise RuntimeError(f"tensor-parallel peer time-out: {peers.timeouts()} arrival flag(s) never came "
                               "(a rank of the group is gone); the partial sums of those steps are stale")

    def _check_pages(self) -> None:
        self._behind_steps()
        if refused := self.paged.refused():
            raise RuntimeError(f"the {self.paged.bits}-bit cache had no page {refused} time(s) for a sequence of a step, which then emitted nothing, or for a portion of a prompt, which is not in "
                               f"it ({self.paged.pages} pages of {self.paged.page_tokens} tokens)")

    def _behind_steps(self) -> None:
        """What the caller's stream does from here on comes after the steps that are queued on self.stream."""
        cur = torch.cuda.current_stream(self.model.device)
        if cur != self.stream:
            cur.wait_stream(self.stream)

    def _join_caller_stream(self) -> None:
        """self.stream is a non-blocking stream: work the caller queued on ITS stream (prefill, state edits) is ordered before
        the step only by an explicit wait. Without it the step can read seq_len / cur_tok before prefill has written them and
        append draft K/V rows at the wrong cache positions (seen as intermittently
        different tokens when capture() followed prefill() without a synchronize)."""
        cur = torch.cuda.current_stream(self.model.device)
        if cur != self.stream:
            self.stream.wait_stream(cur)

    def step(self) -> None:
        """One speculative step, device-resident state; asynchronous on self.stream (ordered after the work already queued on
        the caller's current stream; the caller synchronises self.stream before reading the outputs)."""
        self._check_capacity()
        self._len_bound += self.k + 1
        self._steps += 1
        self._join_caller_stream()
        if self.use_graph:
            if self.graph is None:
                self.capture()
            with torch.cuda.stream(self.stream):
                self.graph.replay()
        else:
            with torch.cuda.stream(self.stream):
                self._spec_step()

    def step_host(self, host_tokens: torch.Tensor) -> torch.Tensor:
        """End-to-end API: the caller owns the last token of every sequence on the HOST (as the
        reference engine does); returns host [B, k+2] = emitted tokens (-1 padded) + count.
        H2D of the inputs and D2H of the result are part of the call."""
        self.h_in.copy_(host_tokens)
        self._join_caller_stream()                        # (a prefill that has yet to run writes cur_tok, too)
        with torch.cuda.stream(self.stream):
            self.cur_tok.copy_(self.h_in, non_blocking=True)
        self.step()
        with torch.cuda.stream(self.stream):
            self.h_out.copy_(self.d_out_pack, non_blocking=True)
        self.stream.synchronize()
        return self.h_out

    # ---------------------------------------------------------------------------------------
    def metrics(self) -> dict:
        if self.counters.is_cuda:
            self._behind_steps()
        peers = getattr(self.model, "peers", None)
        if peers is not None and peers.timeouts():
            raise RuntimeError(f"tensor-parallel peer time-out: {peers.timeouts()} arrival flag(s) never came")
        if given_up := ops.attn_tile_timeouts():
            raise RuntimeError(f"{given_up} CTA(s) or rows gave up a wait in attention, a linear layer or the rotation before one; the outputs of "
                               "those steps hold NaN")
        if getattr(self.model, "paged", None) is not None:
            self._check_pages()
        acc, draft, emitted = [int(v) for v in self.counters.tolist()]
        steps = draft // (self.B * self.k) if draft else 0
        max_emit = steps * self.B * (self.k + 1)
        return {"accepted_tokens": acc, "draft_tokens": draft, "emitted_tokens": emitted,
                "draft_acceptance_rate": acc / draft if draft else float("nan"),
                "system_efficiency": emitted / max_emit if max_emit else float("nan")}
