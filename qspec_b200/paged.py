"""Key/value caches of the int4 decoder in pages and in 8 or 4 bits: half or a quarter of the float16 cache's bytes, and memory by the tokens that are held instead of the
longest that a sequence may become.

A cache lives on the device as a whole: which pages a request holds, the free pages and the lengths that they follow from are device memory, so that
a captured step (`engine.QSpecEngine`) takes the pages that it needs without the host. Per layer, for keys and for values: `PagedKV8Cache` has codes int8 [pages, kv heads, page,
head dim] and one float32 scale per page and head; `PagedKV4Cache` has codes of four bits, two to a byte, and a word of 16 bits for each row, its scale and zero point.

The reference leaves all of this to vLLM (vllm/core/block_manager.py, vllm/worker/model_runner.py: block tables and slot mappings built on the host and
copied in every step); only the behaviour is restated here.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import ops


@dataclass
class PagedStep:
    """One step's tokens as the cache's operators read them (device int32)."""
    q_start: torch.Tensor          # [requests + 1] first token of each request
    kv_len: torch.Tensor           # [requests] tokens held once the step has run
    positions: torch.Tensor        # [tokens]
    slots: torch.Tensor            # [tokens] page * page_tokens + row; negative: none
    seq_ids: Optional[torch.Tensor]
    max_tokens: int                # an upper bound of the tokens of a request


class PagedCache:
    """What the caches have in common: pages, who holds them, and plans of steps. A subclass allocates the codes (`_allocate`), and appends, attends and reads."""
    bits = 0

    def __init__(self, layers: int, kv_heads: int, head_dim: int, requests: int, max_request_tokens: int, max_step_tokens: int, device, page_tokens: int = 64,
                 pages: Optional[int] = None):
        """pages: of the whole cache; default: enough for every request at its longest (fewer where memory is to be shared: a step that asks for more than
        there is refuses requests, see `short` and `refused`; nothing takes pages from one request for another)."""
        if page_tokens not in ops._PAGE_TOKENS:
            raise ValueError(f"pages of 16, 32, 64 or 128 tokens, got {page_tokens}")
        if head_dim not in (64, 128):
            raise ValueError(f"the {self.bits}-bit cache takes heads of 64 or 128, got {head_dim}")
        width = -(-max_request_tokens // page_tokens)
        pages = requests * width if pages is None else pages
        if pages < 1 or requests < 1:
            raise ValueError("a cache needs a page and a request")
        self.requests, self.page_tokens, self.pages, self.max_step_tokens = requests, page_tokens, pages, max_step_tokens
        self.device = device = torch.device(device)
        i32 = dict(dtype=torch.int32, device=device)
        self._allocate(layers, pages, kv_heads, page_tokens, head_dim)
        self.table = torch.zeros(requests, width, **i32)
        self.free_pages = torch.arange(pages, **i32)
        self.state = torch.zeros(requests + 1, **i32)                 # pages held by each request; free pages
        self.state[requests] = pages
        self.state_out = torch.zeros(requests + 2, **i32)
        self.refusals = torch.zeros(1, dtype=torch.int64, device=device)
        self.q_start, self.kv_len = torch.zeros(requests + 1, **i32), torch.zeros(requests, **i32)
        self.positions, self.seq_ids, self.slots = (torch.zeros(max(max_step_tokens, 1), **i32) for _ in range(3))

    def plan(self, lengths: torch.Tensor, counts: torch.Tensor, tokens: int, max_tokens: Optional[int] = None) -> PagedStep:
        """Pages and slots of a step of `tokens` tokens: lengths, counts int32 [requests] on the device; counts[b] < 0 gives request b's pages back. The result
        lies in buffers that the next plan writes again. `commit` makes the step's pages the requests' own."""
        if tokens > self.max_step_tokens:
            raise ValueError(f"a step of {tokens} tokens exceeds max_step_tokens = {self.max_step_tokens}")
        pos, seq, slots = self.positions[:tokens], self.seq_ids[:tokens], self.slots[:tokens]
        ops.page_plan(lengths, counts, self.table, self.free_pages, self.state, self.page_tokens, self.q_start, self.kv_len, pos, seq, slots, self.state_out)
        return PagedStep(self.q_start, self.kv_len, pos, slots, seq, max_tokens or max(tokens, 1))

    def short(self) -> int:
        """Requests that the last plan refuses pages. Reads the device. A plan that is not committed costs nothing."""
        return int(self.state_out[-1].item())

    def commit(self) -> None:
        self.state.copy_(self.state_out[:-1])
        self.refusals.add_(self.state_out[-1])

    def _slots(self, request: int, tokens: int) -> torch.Tensor:
        """Of a request's first tokens."""
        most = self.table.shape[1] * self.page_tokens
        if not 0 <= tokens <= most:
            raise ValueError(f"read: {tokens} tokens of a request, whose row of the table has pages for {most}")
        at = torch.arange(tokens, dtype=torch.int32, device=self.device)
        return (self.table[request].index_select(0, at // self.page_tokens) * self.page_tokens + at % self.page_tokens).to(torch.int32)

    def refused(self) -> int:
        """Requests that committed steps have refused pages, since the cache was made or `refusals` was set to zero: their tokens of that step are in no page. Reads the device."""
        return int(self.refusals.item())

    def free(self) -> int:
        """Free pages. Reads the device."""
        return int(self.state[self.requests].item())


class PagedKV8Cache(PagedCache):
    bits = 8

    def _allocate(self, layers: int, pages: int, kv_heads: int, page_tokens: int, head_dim: int) -> None:
        self.k = torch.zeros(layers, pages, kv_heads, page_tokens, head_dim, dtype=torch.int8, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.ones(layers, pages, kv_heads, dtype=torch.float32, device=self.device)
        self.v_scale = torch.ones_like(self.k_scale)
        self.workspace = ops.kv8_attention_workspace(self.device)

    def append(self, layer: int, qkv: torch.Tensor, cos_sin: torch.Tensor, step: PagedStep, q_out: torch.Tensor) -> None:
        """Rotated queries of qkv [T, (H + 2 G) D] into q_out [T, H, D]; keys and values into the step's slots."""
        ops.kv8_append(qkv, cos_sin, step.positions, step.slots, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], q_out)

    def attend(self, layer: int, q: torch.Tensor, step: PagedStep, out: torch.Tensor, sm_scale: float) -> torch.Tensor:
        return ops.kv8_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.table, step.q_start, step.kv_len, out, sm_scale,
                                 self.workspace, max_tokens=step.max_tokens)

    def read(self, layer: int, request: int, tokens: int, dtype=torch.float16):
        """Keys and values [tokens, kv heads, head dim] of a request's first tokens, in 16 bits (to check a cache, or to move a sequence out of it)."""
        slots, shape = self._slots(request, tokens), (tokens, self.k.shape[2], self.k.shape[4])
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        ops.kv8_read(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], slots, k, v)
        return k, v


class PagedKV4Cache(PagedCache):
    """hadamard: queries and keys go through the Hadamard matrix of a head / sqrt(head dim) behind the rotary embedding, which leaves their products as they are and keeps
    channels that are large in all keys from taking a row's sixteen codes. Every row has a scale of its own: what a draft leaves behind is gone once its rows are written over."""
    bits = 4

    def __init__(self, *args, hadamard: bool = True, **kw):
        super().__init__(*args, **kw)
        self.hadamard = bool(hadamard)

    def _allocate(self, layers: int, pages: int, kv_heads: int, page_tokens: int, head_dim: int) -> None:
        self.k = torch.zeros(layers, pages, kv_heads, page_tokens, head_dim // 2, dtype=torch.uint8, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.k_words = torch.zeros(layers, pages, kv_heads, page_tokens, dtype=torch.int16, device=self.device)
        self.v_words = torch.zeros_like(self.k_words)
        self.workspace = ops.kv4_attention_workspace(self.device)

    def append(self, layer: int, qkv: torch.Tensor, cos_sin: torch.Tensor, step: PagedStep, q_out: torch.Tensor) -> None:
        """Rotated queries of qkv [T, (H + 2 G) D] into q_out [T, H, D]; keys and values into the step's slots."""
        ops.kv4_append(qkv, cos_sin, step.positions, step.slots, self.k[layer], self.v[layer], self.k_words[layer], self.v_words[layer], q_out, self.hadamard)

    def attend(self, layer: int, q: torch.Tensor, step: PagedStep, out: torch.Tensor, sm_scale: float) -> torch.Tensor:
        return ops.kv4_attention(q, self.k[layer], self.v[layer], self.k_words[layer], self.v_words[layer], self.table, step.q_start, step.kv_len, out, sm_scale,
                                 self.workspace, max_tokens=step.max_tokens)

    def read(self, layer: int, request: int, tokens: int, dtype=torch.float16):
        """Keys and values [tokens, kv heads, head dim] of a request's first tokens, in 16 bits; keys as they lie in the cache (behind the Hadamard matrix, if there is one: it is its own
        inverse)."""
        slots, shape = self._slots(request, tokens), (tokens, self.k.shape[2], 2 * self.k.shape[4])
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        ops.kv4_read(self.k[layer], self.v[layer], self.k_words[layer], self.v_words[layer], slots, k, v)
        return k, v
