"""Beam search: the best continuations of each prompt under the model, a step at a time on the device.

The reference samples one continuation per prompt (model.py:301-370).  Here K beams of a
prompt go on at once.  A step lets the attention memory's pages and the block states
follow the chosen beams (``native.kv_fork`` and ``kv_copy_pages``, ``native.reorder_rows``),
runs one token of every beam through the model, and chooses the next ones
(``native.beam_select``); beams keep their places where they go on (``stay``), so what
survives is not moved.  A beam that has ended keeps the states ahead of its stop token.  The whole step is captured as one CUDA graph and replayed without
the host: tokens and parents are read once at the end, where the best beam is followed back.
"""
from __future__ import annotations

import weakref
from typing import List, Optional, Tuple

import torch
from torch import Tensor

from .. import native
from ..core.cache import BeamCache
from ..core.fused import BlockState
from ..core.rotary import Seen
from .decode import capturing


def _wide(t: Tensor) -> Tensor:
    """The rows of a contiguous tensor as the widest elements that make them up, which torch moves fastest: a step of
    the large preset's 64 rows takes 6600 us with stop tokens, 9315 by bf16, 6350 without (where states are copied whole)."""
    t = t.flatten(1)
    row = t.shape[1] * t.element_size()
    for dtype, size in ((torch.complex128, 16), (torch.int64, 8), (torch.int32, 4)):
        if row % size == 0:
            return t.view(dtype)
    return t


class BeamStep:
    """A step of ``beams`` beams for each of ``prompts`` prompts, with its buffers; captured unless ``capture`` is False."""

    def __init__(self, model, prompts: int, beams: int, device, dtype, cache_tokens: int, length_penalty: float,
                 stop: Tuple[int, ...], capture: bool = True) -> None:
        cfg = model.config
        R, di = prompts * beams, cfg.d_model * cfg.expand
        self.model = model          # weakly: the model holds the step, which holds what it reads instead
        self.prompts, self.beams, self.alpha = prompts, beams, length_penalty
        self.tok = torch.zeros((R, 1), dtype=torch.int64, device=device)
        self.rows = torch.arange(R, dtype=torch.int32, device=device)
        self.scores = torch.zeros((prompts, beams), dtype=torch.float32, device=device)
        self.finished = torch.zeros((prompts, beams), dtype=torch.bool, device=device)
        self.lengths = torch.zeros((prompts, beams), dtype=torch.int32, device=device)
        self.stop = torch.tensor(stop, dtype=torch.int64, device=device) if stop else None
        self.pad = stop[0] if stop else 0
        self.mem = [torch.zeros((R, di), dtype=dtype, device=device) for _ in model.blocks]
        self.st = [torch.zeros((R, di, cfg.d_state), dtype=dtype, device=device) for _ in model.blocks]
        self.ws = torch.empty(native.block_workspace_bytes(dtype, R, 1, cfg.d_model, di, cfg.d_state), dtype=torch.uint8, device=device)
        # two tokens more than asked for: the capture's own
        self.cache = BeamCache(cfg, prompts, beams, cache_tokens + 2, device) if cache_tokens else None
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        if capture:
            self._capture(device)
        layers = model.attn_layers.values()
        self.frequencies = [Seen(a.rope.inv_freq) for a in layers]
        self.held = [(a.rope.cos_cached, a.rope.sin_cached, getattr(a, "_rope_freq", None)) for a in layers]
        self.held += [list(model.children()), [getattr(b, "_cache", None) for b in model.blocks]]

    @property
    def model(self):
        return self._model()

    @model.setter
    def model(self, model) -> None:
        self._model = weakref.ref(model)

    def frequencies_hold(self) -> bool:
        """Whether every attention layer still has the frequencies that were captured."""
        return all(f.still(a.rope.inv_freq) for f, a in zip(self.frequencies, self.model.attn_layers.values()))

    def _step(self) -> None:
        if self.cache is not None:
            self.cache.fork(self.rows)
        native.reorder_rows(self.mem + self.st, self.rows, group=self.beams)
        states = [BlockState(membrane=m, ssm_state=s) for m, s in zip(self.mem, self.st)]
        logits, new, _ = self.model.forward_device(self.tok, states, workspace=self.ws, attn_cache=self.cache)
        ended = self.finished.view(-1, 1)               # they wait with the states ahead of their stop token
        for m, s, ns in zip(self.mem, self.st, new):
            if self.stop is None:                       # none ends
                m.copy_(ns.membrane)
                s.copy_(ns.ssm_state)
            else:
                for old, now in ((m, ns.membrane), (s, ns.ssm_state)):
                    old, now = _wide(old), _wide(now)
                    torch.where(ended, old, now, out=old)
        self._choose(logits[:, -1, :])

    def _choose(self, logits: Tensor) -> None:
        scores, rows, tokens = native.beam_select(logits, self.scores, finished=self.finished, lengths=self.lengths,
                                                  length_penalty=self.alpha, pad=self.pad, stay=True)
        beam = (rows % self.beams).long()
        done = self.finished.gather(1, beam)
        self.lengths.copy_(self.lengths.gather(1, beam) + (~done).int())
        self.finished.copy_(done if self.stop is None else done | self._stops(tokens))
        self.scores.copy_(scores)
        self.rows.copy_(rows.view(-1))
        self.tok.copy_(tokens.view(-1, 1))

    def _stops(self, tokens: Tensor) -> Tensor:
        return (tokens[..., None] == self.stop).any(-1)

    def _capture(self, device) -> None:
        def stand():
            # a token ahead of the step, so that its attention reads the cache; forgotten by begin()
            if self.cache is not None:
                self.cache.reset()
                self.cache.begin(1)
                self.cache.advance(1)
                self.rows.copy_(torch.arange(self.rows.numel(), device=device) // self.beams * self.beams)

        side = torch.cuda.Stream(device=device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side), torch.no_grad():
            for _ in range(2):
                stand()
                self._step()
            stand()
        torch.cuda.current_stream(device).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), capturing(self.graph):
            self._step()

    def begin(self, ids: Tensor, states) -> None:
        """Runs the prompts and chooses their first tokens."""
        P, K = self.prompts, self.beams
        cache = None
        if self.cache is not None:
            self.cache.reset()
            cache = self.cache.prompt_rows()
            self.cache.begin(min(ids.shape[1], self.model.config.max_seq_len))
        logits, states, _ = self.model.forward_device(ids, states, last_only=True, attn_cache=cache)
        if cache is not None:
            self.cache.filled = cache.filled
        for i, ns in enumerate(states):
            self.mem[i].copy_(ns.membrane.repeat_interleave(K, 0))
            self.st[i].copy_(ns.ssm_state.repeat_interleave(K, 0))
        scores, _, tokens = native.beam_select(logits[:, -1, :], torch.zeros((P, 1), device=ids.device), n=K, pad=self.pad)
        self.scores.copy_(scores)
        self.tok.copy_(tokens.view(-1, 1))
        self.rows.copy_(torch.arange(P * K, device=ids.device) // K * K)
        self.lengths.fill_(1)
        self.finished.copy_(self._stops(tokens) if self.stop is not None else torch.zeros_like(self.finished))

    def run(self) -> None:
        """One step."""
        if self.graph is None:
            self._step()
            return
        if self.cache is not None:
            self.cache.move(1)
        self.graph.replay()


def beam_search(model, ids: Tensor, max_new_tokens: int, beams: int, length_penalty: float, stop: List[int], states,
                use_graph: bool, attn_cache: bool) -> Tuple[Tensor, List[BlockState]]:
    """(tokens of the best beam of each prompt behind the prompt, its block states); see ``generate``."""
    P, prompt = ids.shape
    tokens = min(prompt, model.config.max_seq_len) + max_new_tokens if attn_cache else 0
    step = model.beam_step(P, beams, ids.device, model.lm_head.weight.dtype, tokens, length_penalty, tuple(stop),
                           use_graph and ids.is_cuda and max_new_tokens > 1)
    step.begin(ids, states)
    made, parents = [step.tok.view(P, beams).clone()], []
    for i in range(1, max_new_tokens):
        # a read of the device now and then: finished beams only wait
        if stop and i % 8 == 0 and bool(step.finished.all()):
            break
        step.run()
        made.append(step.tok.view(P, beams).clone())
        parents.append(step.rows.view(P, beams) % beams)
    # the best beam by its score, and the way back
    rank = step.scores.double() / step.lengths.clamp(min=1).double().pow(length_penalty)
    best = rank.argmax(1, keepdim=True)
    rows = (best + beams * torch.arange(P, device=ids.device)[:, None]).view(-1)
    at, out = best, []
    for i in range(len(made) - 1, -1, -1):
        out.append(made[i].gather(1, at))
        if i:
            at = parents[i - 1].gather(1, at).long()
    new = torch.cat(out[::-1], dim=1)
    if new.shape[1] < max_new_tokens:
        new = torch.cat([new, torch.full((P, max_new_tokens - new.shape[1]), step.pad, dtype=new.dtype, device=new.device)], 1)
    # the chosen beams' states are those of the rows that they went on from
    source = step.rows.long()[rows]
    state_cls = model.blocks[0]._state_cls
    return torch.cat([ids, new], 1), [state_cls(membrane=m[source], ssm_state=s[source]) for m, s in zip(step.mem, step.st)]
