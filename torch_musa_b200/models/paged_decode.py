"""Serving the Llama model from a paged key-value cache: sequences of different lengths come and go, each owns pages of a
common pool, and a step decodes one token for all of them or checks several drafted tokens at once.

Lengths, block tables and tokens live in fixed device buffers that the kernels read themselves, so the step is captured into
a graph and replayed while the host only hands out pages.  With a sliding window the pages behind it go back to the pool.
No counterpart in the reference, whose caches are contiguous (reference torch_musa/musa_graph/graphs.py:44-132 is the graph
runtime that its decoding loops use).
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from ..ops import functional as BF
from .llama import Llama


class PagedLlamaDecoder:
    """``sequences`` slots over ``pages`` pages of ``page_size`` tokens.  ``add`` puts a prompt into a free slot, ``step`` decodes
    one greedy token for every slot in use, ``check`` verifies drafted tokens for all of them, ``remove`` gives a slot back."""

    def __init__(self, model: Llama, sequences: int, pages: int, page_size: int = 64, max_len: Optional[int] = None, device=None,
                 dtype: Optional[torch.dtype] = None):
        cfg = model.cfg
        self.model, self.cfg, self.B, self.page_size = model, cfg, sequences, page_size
        self.max_len = max_len or cfg.max_seq_len
        self.device = torch.device(device) if device is not None else next(model.parameters()).device
        dt = dtype or next(model.parameters()).dtype
        shape = (cfg.n_layers, pages, cfg.kv_heads, page_size, cfg.head_dim)
        self.k_pages = torch.zeros(shape, device=self.device, dtype=dt)
        self.v_pages = torch.zeros_like(self.k_pages)
        width = -(-self.max_len // page_size)
        self._table = torch.full((sequences, width), -1, dtype=torch.int32)                     # the host's copy
        self.block_table = self._table.to(self.device)
        self.seq_lens = torch.zeros(sequences, dtype=torch.int32, device=self.device)           # tokens in the cache
        self.active = torch.zeros(sequences, dtype=torch.int32, device=self.device)
        self.tokens = torch.zeros(sequences, 1, dtype=torch.long, device=self.device)           # the next step's input
        self.lens: List[Optional[int]] = [None] * sequences                                     # the host's copy of the lengths
        self.free = list(range(pages - 1, -1, -1))
        self._pages: List[dict] = [{} for _ in range(sequences)]                                # table index -> page, per slot
        cos, sin = BF.precompute_rope_cache(self.max_len, cfg.head_dim, cfg.rope_theta)
        self.cos, self.sin = cos.to(self.device), sin.to(self.device)
        self._graph = None

    # ------------------------------------------------------------------ pages
    def _reserve(self, slots: Sequence[int], new: int) -> List[Tuple[int, int]]:
        """Pages for ``new`` more tokens of each slot; pages that no later token can see go back to the pool.  Returns what
        ``_give_up`` takes back."""
        size, changed = self.page_size, False
        wanted = []
        for b in slots:
            end = self.lens[b] + new
            if end > self.max_len:
                raise ValueError(f"slot {b}: {end} tokens do not fit into max_len = {self.max_len}")
            mine = self._pages[b]
            if self.cfg.window is not None:
                oldest = self.lens[b] + 1 - self.cfg.window           # the first key that the next token still sees
                for index in [i for i in mine if (i + 1) * size <= oldest and i * size >= self.cfg.attention_sinks]:
                    self.free.append(mine.pop(index))
            wanted += [(b, i) for i in range(self.lens[b] // size, -(-end // size)) if i not in mine]
        if len(wanted) > len(self.free):
            raise RuntimeError(f"the page pool is exhausted: {len(wanted)} pages wanted, {len(self.free)} free")
        for b, i in wanted:
            self._pages[b][i] = page = self.free.pop()
            self._table[b, i] = page
            changed = True
        if changed:
            self.block_table.copy_(self._table)
        return wanted

    def _give_up(self, reserved: Sequence[Tuple[int, int]]) -> None:
        """After a step that failed: its new pages are free again, the device's lengths are the host's."""
        for b, i in reserved:
            self.free.append(self._pages[b].pop(i))
        self.seq_lens.copy_(torch.tensor([n or 0 for n in self.lens], dtype=torch.int32))

    def remove(self, slot: int) -> None:
        """Ends the sequence in ``slot``: its pages and the slot are free again."""
        if self.lens[slot] is None:
            raise ValueError(f"slot {slot} is not in use")
        self.free += self._pages[slot].values()
        self._pages[slot] = {}
        self.lens[slot] = None
        self.seq_lens[slot] = 0
        self.active[slot] = 0

    # ------------------------------------------------------------------ the model over new tokens
    def _add_norm(self, norm, x, delta):
        """(norm(x + delta), x + delta); residual add and RMS norm are one kernel on the device."""
        if delta is None:
            return norm(x), x
        eps = norm.eps if norm.eps is not None else torch.finfo(x.dtype).eps
        return BF.rms_norm_residual(delta, x, norm.weight, eps)

    def _layers(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """The hidden rows of packed ``tokens`` [T] after the last norm; ``attend(layer index, q, k, v)`` writes the cache and attends."""
        cfg, m = self.cfg, self.model
        h, kv, hd = cfg.n_heads, cfg.kv_heads, cfg.head_dim
        x, delta = m.tok_emb(tokens), None
        for li, layer in enumerate(m.layers):
            hn, x = self._add_norm(layer.attn_norm, x, delta)
            a = layer.attn
            if cfg.fused_qkv:
                q, k, v = a.wqkv(hn).view(-1, h + 2 * kv, hd).split([h, kv, kv], dim=1)
            else:
                q, k, v = a.wq(hn).view(-1, h, hd), a.wk(hn).view(-1, kv, hd), a.wv(hn).view(-1, kv, hd)
            hn, x = self._add_norm(layer.ffn_norm, x, a.wo(attend(li, q, k, v).reshape(-1, h * hd)))
            delta = layer.ffn(hn)
        return self._add_norm(m.norm, x, delta)[0]

    @torch.no_grad()
    def add(self, prompts: Sequence[torch.Tensor]) -> List[int]:
        """Runs the prompts (1-D token tensors) packed through the model and returns their slots; ``tokens`` then holds the greedy
        next token of each."""
        slots = [b for b in range(self.B) if self.lens[b] is None][:len(prompts)]
        if len(slots) < len(prompts):
            raise RuntimeError(f"{len(prompts)} prompts, {len(slots)} free slots")
        sizes = [int(p.numel()) for p in prompts]
        if not sizes or min(sizes) == 0:
            raise ValueError("a prompt needs at least one token")
        for b in slots:
            self.lens[b] = 0
        try:
            self._prefill(slots, prompts, sizes)
        except Exception:
            for b in slots:
                self.remove(b)
            raise
        for b, n in zip(slots, sizes):
            self.lens[b] = n
        return slots

    def _prefill(self, slots: List[int], prompts: Sequence[torch.Tensor], sizes: List[int]) -> None:
        for b, n in zip(slots, sizes):
            self._reserve([b], n)
        rows = torch.tensor(slots, device=self.device)
        table, lens = self.block_table[rows], torch.tensor(sizes, dtype=torch.int32, device=self.device)
        cu = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).to(self.device)
        positions = torch.cat([torch.arange(n) for n in sizes]).to(self.device).view(1, -1)
        window, sinks = self.cfg.window, self.cfg.attention_sinks

        def attend(li, q, k, v):
            turned = BF.paged_rope_cache(q, k, v, self.cos, self.sin, self.k_pages[li], self.v_pages[li], table, lens, cu)
            k = BF.rope(k.unsqueeze(0), self.cos, self.sin, positions).squeeze(0)
            return BF.flash_attn_varlen_func(turned, k, v, cu, cu, max(sizes), max(sizes), causal=True, window=window, sinks=sinks)

        last = self._layers(torch.cat([p.to(self.device) for p in prompts]), attend)[cu[1:].long() - 1]
        self.tokens[rows] = self.model.lm_head(last).argmax(-1, keepdim=True)
        self.seq_lens[rows] = lens
        self.active[rows] = 1

    def _new_tokens(self, tokens: torch.Tensor) -> torch.Tensor:
        """Hidden rows [B, n, dim] of n new tokens per slot; ``seq_lens`` counts them already."""
        B, n = tokens.shape

        def attend(li, q, k, v):
            turned = BF.paged_rope_cache(q, k, v, self.cos, self.sin, self.k_pages[li], self.v_pages[li], self.block_table, self.seq_lens)
            return BF.paged_attention(turned.view(B, n, *turned.shape[1:]), self.k_pages[li], self.v_pages[li], self.block_table,
                                      self.seq_lens, self.cfg.window, self.cfg.attention_sinks)

        return self._layers(tokens.reshape(-1), attend).view(B, n, -1)

    def _step(self) -> None:
        self.seq_lens.add_(self.active)
        self.tokens.copy_(self.model.lm_head(self._new_tokens(self.tokens)).argmax(-1))

    @torch.no_grad()
    def step(self) -> torch.Tensor:
        """Decodes one greedy token for every slot in use; returns the tokens that went into the cache, [B] (a copy)."""
        used = [b for b in range(self.B) if self.lens[b] is not None]
        reserved = self._reserve(used, 1)
        went_in = self.tokens[:, 0].clone()
        try:
            if self._graph is not None:
                self._graph.replay()
            else:
                self._step()
        except Exception:
            self._give_up(reserved)
            raise
        for b in used:
            self.lens[b] += 1
        return went_in

    @torch.no_grad()
    def check(self, drafts: torch.Tensor, uniforms: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
              temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Verifies ``drafts`` [B, n] (what a draft model proposes after ``tokens``) in one pass over n + 1 tokens per slot, as
        ``ops.verify_drafts`` does with the model's probabilities (float32) at ``temperature``: ``drafts`` are int64, ``uniforms`` and
        ``draft_probs`` float32, all on the decoder's device.  The caches keep the taken tokens only, ``tokens`` becomes the drawn
        ones.  Returns (taken [B], tokens [B, n + 1]); rows of slots not in use mean nothing.  A call that fails changes nothing."""
        if temperature <= 0:
            raise ValueError(f"temperature must be positive, got {temperature}")
        n = drafts.shape[-1]
        if (tuple(drafts.shape) != (self.B, n) or drafts.dtype != torch.long
                or tuple(uniforms.shape) != (self.B, n + 1) or uniforms.dtype != torch.float32
                or (draft_probs is not None and (tuple(draft_probs.shape) != (self.B, n, self.cfg.vocab_size)
                                                 or draft_probs.dtype != torch.float32))):
            raise ValueError("int64 drafts [sequences, n], float32 uniforms [sequences, n + 1] and float32 draft_probs "
                             "[sequences, n, vocabulary] expected")
        for t in (drafts, uniforms, draft_probs):
            if t is not None and t.device != self.seq_lens.device:
                raise ValueError(f"the decoder is on {self.seq_lens.device}, an argument on {t.device}")
        used = [b for b in range(self.B) if self.lens[b] is not None]
        reserved = self._reserve(used, n + 1)
        try:
            self.seq_lens.add_(self.active * (n + 1))
            inputs = torch.cat((self.tokens, drafts.clamp(0, self.cfg.vocab_size - 1)), 1)
            logits = self.model.lm_head(self._new_tokens(inputs)).float()
            taken, out = BF.verify_drafts(torch.softmax(logits / temperature, -1), drafts, uniforms, draft_probs)
            drawn, counts = out.gather(1, taken[:, None]).clamp_min(0), taken.tolist()
            self.seq_lens.sub_(self.active * (n - taken).to(torch.int32))
        except Exception:
            self._give_up(reserved)
            raise
        self.tokens.copy_(drawn)
        for b, t in enumerate(counts):
            if self.lens[b] is not None:
                self.lens[b] += t + 1
        return taken, out

    def capture(self, warmup: int = 2) -> None:
        """Records ``step`` into a device graph.  The warm-up steps run on empty slots: no sequence may be in use."""
        import torch_musa_b200 as bw

        if any(n is not None for n in self.lens):
            raise RuntimeError("capture before the first prompt")
        side = bw.Stream()
        side.wait_stream(bw.current_stream())
        with torch.no_grad(), bw.stream(side):
            for _ in range(warmup):
                self._step()
        bw.current_stream().wait_stream(side)
        graph = bw.BlackwellGraph()
        with torch.no_grad(), bw.graph(graph):
            self._step()
        self._graph = graph
