"""Keys and values of a model's attention layers, kept between generation steps.

The reference's ``SlidingWindowAttention`` (model.py:129-181) is stateless
across calls: a decode step attends to itself alone.  ``AttentionCache``
gives it a memory of its window: paged e4m3 codes with one power-of-two scale
per page and head (``native.kv_append``, ``native.kv_attention``), one pool per
attention layer, one page table and one length per sequence for all of them.

``BeamCache`` is the memory of a beam search: the beams of a prompt share pages, which
are counted, forked when a beam goes on from another (``native.kv_fork``) and free when
none has them; attention reads what all beams of a prompt share once
(``native.kv_attention_shared``).

A layer looks ``window`` tokens back, so a sequence needs only the pages of its
last ``window + max_step`` tokens: the table repeats them as a ring, and a page
that has left the window is written again from its first slot on.
"""
from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch
from torch import Tensor

from .. import native

Layer = Tuple[Tensor, Tensor, Tensor, Tensor]      # k codes, k scales, v codes, v scales


class AttentionCache:
    """The attention memory of ``batch`` sequences of at most ``max_tokens`` tokens.

    ``page``: tokens that share a scale (16, 32 or 64); ``max_step``: the most new
    tokens that one attention call takes (longer inputs are taken in pieces)."""

    def __init__(self, config, batch: int, max_tokens: int, device, page: int = 32, max_step: int = 16) -> None:
        heads = config.attn_heads
        head_dim = config.d_model // heads
        if config.n_attn_layers < 1:
            raise ValueError(f"the model '{config.model_name}' has no attention layers to keep a cache for")
        if head_dim not in (64, 128) or config.d_model != heads * head_dim:
            raise ValueError(f"the attention cache takes heads of 64 or 128, not {config.d_model} / {heads}")
        if page not in (16, 32, 64):
            raise ValueError(f"page must be 16, 32 or 64, got {page}")
        if batch < 1 or max_tokens < 1 or max_step < 1:
            raise ValueError("batch, max_tokens and max_step must be at least 1")
        self.batch, self.page, self.max_step, self.window = batch, page, max_step, config.attn_window
        blocks = -(-max_tokens // page)
        self.max_tokens = blocks * page
        # pages that the window and the new tokens behind it can touch at once
        ring = min(blocks, -(-(self.window + max_step) // page) + 2)
        self.ring = ring
        self._make_layers(config, batch * ring, heads, head_dim, device)
        rows = torch.arange(batch, device=device, dtype=torch.int32)[:, None] * ring
        self.table = rows + (torch.arange(blocks, device=device, dtype=torch.int32) % ring)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)     # tokens of each sequence so far
        self.filled = 0                                                          # the same on the host: sequences move together

    def _make_layers(self, config, pages: int, heads: int, head_dim: int, device) -> None:
        shape = (pages, heads, self.page, head_dim)
        self.layers: Dict[str, Layer] = {}
        for i in range(config.n_layers):
            if (i + 1) % config.attn_every == 0:
                self.layers[str(i)] = (torch.zeros(shape, device=device, dtype=torch.float8_e4m3fn),
                                       torch.zeros(shape[:2], device=device),
                                       torch.zeros(shape, device=device, dtype=torch.float8_e4m3fn),
                                       torch.zeros(shape[:2], device=device))

    def rows(self, a: int, b: int) -> "AttentionCache":
        """The cache of sequences a..b-1 (the same memory)."""
        part = object.__new__(AttentionCache)
        part.__dict__.update(self.__dict__)
        part.batch, part.table, part.lengths = b - a, self.table[a:b], self.lengths[a:b]
        return part

    def reset(self) -> None:
        """Forget every sequence."""
        self.lengths.zero_()
        self.filled = 0

    def require_batch(self, batch: int) -> None:
        if self.batch != batch:
            raise ValueError(f"the attention cache is for {self.batch} sequences, got {batch}")

    def require(self, tokens: int) -> None:
        """Refuses `tokens` more where they do not fit."""
        if self.filled + tokens > self.max_tokens:
            raise ValueError(f"the attention cache holds {self.max_tokens} tokens a sequence; "
                             f"{self.filled} + {tokens} do not fit")

    def move(self, tokens: int) -> None:
        """Counts `tokens` more on the host (a replayed graph counts on the device itself)."""
        self.require(tokens)
        self.filled += tokens

    def advance(self, tokens: int) -> None:
        """`tokens` more tokens of every sequence are about to be written."""
        self.move(tokens)
        self.lengths += tokens

    def append(self, layer: str, k: Tensor, v: Tensor, lengths: Tensor) -> None:
        """Writes rotated keys and values [B, T, H, D]; `lengths`: of the sequences with them."""
        native.kv_append(k, v, *self.layers[layer], self.table, lengths)

    def attend(self, layer: str, q: Tensor, lengths: Tensor) -> Tensor:
        """Attention of q [B, T, H, D], the last T of `lengths` tokens, over the window."""
        return native.kv_attention(q, *self.layers[layer], self.table, lengths, window=self.window)


class BeamCache(AttentionCache):
    """The attention memory of ``beams`` beams for each of ``prompts`` prompts.

    Row p * beams + k is beam k of prompt p.  ``begin`` makes room for the prompts, which
    run as ``prompt_rows()`` (the first beam of each); ``fork`` lets every row go on from
    another (or stay) and makes room for its next token."""

    def __init__(self, config, prompts: int, beams: int, max_tokens: int, device, page: int = 32) -> None:
        super().__init__(config, 1, max_tokens, device, page, max_step=1)
        if beams < 1 or prompts < 1 or prompts * beams > 1024:
            raise ValueError(f"{prompts} prompts of {beams} beams: at least one of each, 1024 in all")
        R = prompts * beams
        self.prompts, self.beams, self.batch = prompts, beams, R
        blocks = self.max_tokens // page
        # a page more a row: when a begun page is forked, it is held until the copies are made
        heads, head_dim = config.attn_heads, config.d_model // config.attn_heads
        self._make_layers(config, R * (self.ring + 1), heads, head_dim, device)
        self.table = torch.full((R, blocks), -1, device=device, dtype=torch.int32)
        self.refs = torch.zeros(R * (self.ring + 1), device=device, dtype=torch.int32)
        self.lengths = torch.zeros(R, device=device, dtype=torch.int32)
        row = torch.arange(R, device=device, dtype=torch.int32)
        self._first = torch.where(row % beams == 0, row, -1)             # the prompts' rows alone
        self.shared: Optional[Tensor] = None

    def reset(self) -> None:
        """Forget every sequence; all pages are free."""
        super().reset()
        self.table.fill_(-1)
        self.refs.zero_()

    def begin(self, tokens: int) -> None:
        """Room for prompts of `tokens` tokens: the pages that their window still sees at the end."""
        native.kv_fork(self.table, self.refs, self.lengths, self._first, self.page, tokens=tokens, window=self.window)

    def prompt_rows(self) -> AttentionCache:
        """The cache of the prompts, one row each (the same memory)."""
        part = object.__new__(AttentionCache)
        part.__dict__.update(self.__dict__)
        part.batch, part.table, part.lengths = self.prompts, self.table[::self.beams], self.lengths[::self.beams]
        return part

    def fork(self, rows: Tensor) -> None:
        """Row r goes on from row rows[r] of its prompt, with room for one token."""
        copies, self.shared = native.kv_fork(self.table, self.refs, self.lengths, rows, self.page, tokens=1, window=self.window,
                                             group=self.beams)
        native.kv_copy_pages(list(self.layers.values()), copies)

    def attend(self, layer: str, q: Tensor, lengths: Tensor) -> Tensor:
        return native.kv_attention_shared(q, *self.layers[layer], self.table, lengths, self.shared, window=self.window)
