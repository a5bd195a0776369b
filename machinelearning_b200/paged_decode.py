"""A Gemma-3 decode step whose sequences are at positions of their own: the
decoder of ``decode.py`` over a paged key/value cache.

Per layer the fused q|k|v rows go through ``PagedKVCache.append`` and ``attend``
(local layers over their sliding window, global ones over the whole cache); after
the lm_head ``process_logits`` applies each sequence's penalties, biases and
grammar state and the largest logit gives the next token. With a cache budget the
global layers accumulate every slot's attention weight, and ``evict()`` keeps the
heaviest and the most recent slots of each kv head. The reference's decode pass
(llmserve/llmmodel/model/main/src/core/forward.rs:107-239) is the same step for
one position and a dense f32 cache.
"""
from __future__ import annotations

import numpy as np
import torch

from .decode import Gemma3Config, Gemma3Decoder
from .logits import process_logits
from .paged import PagedKVCache


class PagedGemma3Decoder(Gemma3Decoder):
    """``batch`` sequences, each idle or at its own position (``start``, ``stop``).

    ``cfg.ctx`` is the capacity of a sequence; ``window`` the sliding window of the
    local layers (0: none); ``budget`` > 0 the slots the global layers keep of a
    sequence when ``evict()`` is called, ``recent`` of them the latest positions.
    """

    def __init__(self, cfg: Gemma3Config, weights: dict, batch: int, device: int = 0, page_size: int = 16,
                 cache_dtype: torch.dtype = torch.bfloat16, window: int = 512, budget: int = 0, recent: int = 0):
        if budget and not 0 <= recent <= budget:
            raise ValueError(f"recent {recent} outside 0..{budget}")
        self.page_size, self.cache_dtype = page_size, cache_dtype
        self.window, self.budget, self.recent = window, budget, recent
        super().__init__(cfg, weights, batch, device)

    def _alloc_cache(self) -> None:
        cfg, B, dev = self.cfg, self.batch, self.dev
        per = -(-cfg.ctx // self.page_size)
        shape = (cfg.n_layers, B * per, cfg.n_kv_heads, self.page_size, cfg.head_dim)
        self.k_pages = torch.zeros(shape, dtype=self.cache_dtype, device=dev)
        self.v_pages = torch.zeros(shape, dtype=self.cache_dtype, device=dev)
        self.block_table = torch.arange(B * per, dtype=torch.int32, device=dev).view(B, per)
        self.caches = [PagedKVCache(k, v, self.block_table) for k, v in zip(self.k_pages, self.v_pages)]
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        cap = self.caches[0].capacity
        self.positions = ints(B) - 1   # of the next token; -1: idle
        self.active = ints(B)          # 1, or 0 for an idle sequence
        self.slots = ints(B)           # cached slots of the global layers (fewer than positions after evictions)
        self.seen, self.global_seen = ints(B), ints(B)
        self.history, self.prompt_lengths = ints(B, cfg.ctx), ints(B)
        self.next_tokens = ints(B)
        self.processed = torch.zeros(B, cfg.vocab, dtype=torch.float32, device=dev)
        self.host_positions = [-1] * B
        self.global_layers = [li for li in range(cfg.n_layers) if (li + 1) % cfg.pattern == 0]
        self.slot_weights, self.slot_positions = {}, {}
        if self.budget:
            for li in self.global_layers:
                self.slot_weights[li] = torch.zeros(B, cfg.n_kv_heads, cap, dtype=torch.float32, device=dev)
                self.slot_positions[li] = ints(B, cfg.n_kv_heads, cap) - 1
            # where a step that stays at its position leaves its sums
            self.unused_weights = torch.zeros(B, cfg.n_kv_heads, cap, dtype=torch.float32, device=dev)
        one, zero = torch.ones(B, device=dev), torch.zeros(B, device=dev)
        self.penalties = {"repetition": one, "presence": zero.clone(), "frequency": zero.clone()}
        self.bias_ids = self.bias_values = self.mask = self.mask_rows = None
        self.caches[0].reserve(cfg.n_heads, weights=bool(self.budget), budget=self.budget, stream=self.stream)

    # ---- sequences ---------------------------------------------------------------------
    def _check_seq(self, seq: int) -> None:
        if not 0 <= seq < self.batch:
            raise ValueError(f"sequence {seq} of {self.batch}")

    def start(self, seq: int, prompt_length: int = 0) -> None:
        """Begins a sequence at position 0 with an empty cache; the first ``prompt_length``
        tokens count for the repetition penalty only."""
        self._check_seq(seq)
        with self._ordered():
            self.positions[seq], self.active[seq], self.slots[seq] = 0, 1, 0
            self.prompt_lengths[seq] = prompt_length
            for li in self.slot_weights:
                self.slot_weights[li][seq].zero_()
        self.host_positions[seq] = 0

    def stop(self, seq: int) -> None:
        """Leaves a sequence idle: its rows of a step store nothing and attend to nothing."""
        self._check_seq(seq)
        with self._ordered():
            self.positions[seq], self.active[seq], self.slots[seq] = -1, 0, 0
        self.host_positions[seq] = -1

    def set_position(self, pos: int) -> None:
        raise NotImplementedError("sequences have their own positions: start(), stop()")

    def set_penalties(self, repetition=None, presence=None, frequency=None) -> None:
        """Per-sequence penalties (a number or one per sequence)."""
        given = {"repetition": repetition, "presence": presence, "frequency": frequency}
        with self._ordered():
            for name, value in given.items():
                if value is not None:
                    v = np.broadcast_to(np.asarray(value, np.float32), (self.batch,)).copy()
                    self.penalties[name].copy_(torch.from_numpy(v))

    def set_constraints(self, bias_ids=None, bias_values=None, mask=None, mask_rows=None) -> None:
        """Biases and grammar states as ``process_logits`` takes them (None: none). A captured
        step goes on with the tensors it was captured with, which it keeps alive: change those in
        place, or capture again."""
        self.bias_ids, self.bias_values, self.mask, self.mask_rows = bias_ids, bias_values, mask, mask_rows

    # ---- one step ----------------------------------------------------------------------
    def _attention(self, li: int, lw: dict, cos: torch.Tensor, sin: torch.Tensor) -> None:
        cfg, cache = self.cfg, self.caches[li]
        far = (li + 1) % cfg.pattern == 0
        q = cache.append(self.qkv, self.positions, self.slots if far else self.positions, cos, sin,
                         n_heads=cfg.n_heads, q_norm=lw["q_norm"], k_norm=lw["k_norm"], offset=cfg.offset, eps=cfg.eps,
                         out=self.q.view(self.batch, cfg.n_heads, cfg.head_dim))
        out = self.attn.view(self.batch, cfg.n_heads, cfg.head_dim)
        if not far:
            cache.attend(q, self.seen, self.inv_scale, window=self.window, out=out)
            return
        weights = self.slot_weights.get(li)
        cache.attend(q, self.global_seen, self.inv_scale, weights=weights,
                     weights_out=weights if weights is None or self._accumulates else self.unused_weights, out=out)
        if self.budget:  # the new slot's position (of idle sequences: what is there)
            at = self.slots.long().clamp(max=cache.capacity - 1)[:, None, None].expand(-1, cfg.n_kv_heads, 1)
            held = self.slot_positions[li]
            new = torch.where(self.active[:, None, None] > 0, self.positions[:, None, None], held.gather(2, at))
            held.scatter_(2, at, new)

    def _advance(self) -> None:
        self.positions.add_(self.active)
        self.slots.add_(self.active)

    def _launch(self, advance: bool):
        self._accumulates = advance
        # the step's token joins its sequence's history; idle rows keep what they hold
        at = self.positions.clamp(min=0, max=self.cfg.ctx - 1).long()[:, None]
        token = torch.where(self.active[:, None] > 0, self.tokens[:, None], self.history.gather(1, at))
        self.history.scatter_(1, at, token)
        torch.add(self.positions, 1, out=self.seen)
        torch.add(self.slots, 1, out=self.global_seen)
        self.global_seen.mul_(self.active)
        super()._launch(False)
        process_logits(self.logits, tokens=self.history, token_lengths=self.seen, prompt_lengths=self.prompt_lengths,
                       **self.penalties, bias_ids=self.bias_ids, bias_values=self.bias_values, mask=self.mask,
                       mask_rows=self.mask_rows, out=self.processed)
        self.next_tokens.copy_(self.processed.argmax(-1))
        if advance:
            self._advance()

    def capture(self, advance: bool = True) -> None:
        super().capture(advance)
        self._captured_advance = advance
        self._captured_constraints = self.bias_ids, self.bias_values, self.mask, self.mask_rows  # read by replays

    def step(self, tokens=None, advance: bool = True) -> torch.Tensor:
        """Processed logits [batch][vocab] of one step of all started sequences (rows of idle
        ones mean nothing); ``next_tokens`` holds their largest entries. Without ``advance`` the
        step can be repeated: positions and accumulated weights stay as they were."""
        if any(p >= self.cfg.ctx for p in self.host_positions):
            raise ValueError(f"a sequence is at the cache's capacity of {self.cfg.ctx} positions")
        if self.graph is not None:
            advance = self._captured_advance
        super().step(tokens, advance)
        if advance:
            self.host_positions = [p + (p >= 0) for p in self.host_positions]
        return self.processed

    def evict(self) -> None:
        """Brings the global layers down to ``budget`` slots a sequence and kv head."""
        if not self.budget:
            raise ValueError("no cache budget")
        with self._ordered():
            lengths = self.slots
            for li in self.global_layers:
                lengths, w, p = self.caches[li].evict(self.slots, self.slot_weights[li], self.slot_positions[li],
                                                      self.positions, self.budget, self.recent)
                self.slot_weights[li].copy_(w)
                self.slot_positions[li].copy_(p)
            self.slots.copy_(lengths)

    def generate(self, prompts: list[list[int]], max_new_tokens: int, evict_every: int = 0) -> list[list[int]]:
        """The most likely continuations of up to ``batch`` prompts, fed one token a step and
        each sequence's own tokens from there on; with a budget, evicts every so many steps.
        Begins the first sequences anew, one a prompt, and leaves them idle; the others have to be."""
        if len(prompts) > self.batch or any(not p for p in prompts):
            raise ValueError(f"at most {self.batch} prompts, of at least one token")
        if max_new_tokens < 0 or any(len(p) + max_new_tokens - 1 > self.cfg.ctx for p in prompts):
            raise ValueError(f"a prompt and {max_new_tokens} new tokens exceed {self.cfg.ctx} positions")
        if evict_every and not self.budget:
            raise ValueError("no cache budget to evict to")
        if not prompts or not max_new_tokens:
            return [[] for _ in prompts]
        if any(p >= 0 for p in self.host_positions[len(prompts):]):
            raise ValueError("a sequence without a prompt is started: it would be fed tokens of nobody's")
        graph = self.graph
        if graph is not None and not self._captured_advance:
            self.graph = None  # a step that stays where it is and adds no weights is not this loop's
        try:
            return self._generate(prompts, max_new_tokens, evict_every)
        finally:
            self.graph = graph

    def _generate(self, prompts: list[list[int]], max_new_tokens: int, evict_every: int) -> list[list[int]]:
        for s, p in enumerate(prompts):
            self.start(s, len(p))
        out: list[list[int]] = [[] for _ in prompts]
        last = [0] * self.batch
        steps = 0
        while any(len(o) < max_new_tokens for o in out):
            tokens = list(last)
            for s, p in enumerate(prompts):
                if 0 <= self.host_positions[s] < len(p):
                    tokens[s] = p[self.host_positions[s]]
            self.step(tokens)
            last = self.next_tokens.tolist()
            for s, p in enumerate(prompts):
                if self.host_positions[s] >= len(p):
                    out[s].append(last[s])
                    if len(out[s]) == max_new_tokens:
                        self.stop(s)
            steps += 1
            if evict_every and steps % evict_every == 0:
                self.evict()
        return out
