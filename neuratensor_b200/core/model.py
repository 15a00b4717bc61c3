"""NeuraTensorModel on the B200 block kernels.

Interface mirror of NeuraTensor's ``neuratensor/core/model.py``:
``ModelConfig`` (model.py:32-85), ``RotaryEmbedding`` / ``apply_rotary`` /
``SlidingWindowAttention`` (model.py:88-181) and ``NeuraTensorModel``
(model.py:184-396) keep their names, fields, submodule layout and
initialisation order (embedding, blocks with attention interleaved, final
norm, tied lm_head, then ``_init_weights``), so a seed gives the reference's
weights and checkpoints load either way.

The spike blocks, the embedding gather, the sliding-window attention layers
(RMSNorm, projections and the windowed attention core) and the final RMSNorm +
tied lm_head (bf16 logits on the tcgen05 GEMM) run on the native kernels.
The forward collects every block's spike count in one device buffer and
reads it once, instead of the reference's three host syncs per block.

Beyond the reference, the attention layers can keep an 8-bit cache between
calls (``core/cache.py``; the reference's are stateless), and ``generate``
takes frequency and presence penalties, biases and masks beside the
repetition penalty, all on the device (``native.logits_process``).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Dict, List, Optional, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from .cache import AttentionCache
from .fused import BlockState, FusedSpikeBlock, rate_like_reference
from .rotary import Seen


@dataclass
class ModelConfig:
    """Full model configuration (model.py:32-85)."""
    vocab_size: int = 32_000
    d_model: int = 512
    n_layers: int = 8
    d_state: int = 16
    expand: int = 2
    beta_init: float = 0.9
    learn_beta: bool = True
    dropout: float = 0.0
    tie_weights: bool = True
    max_seq_len: int = 2048
    attn_every: int = 0
    attn_heads: int = 4
    attn_window: int = 256
    model_name: str = "custom"

    @property
    def n_attn_layers(self) -> int:
        return 0 if self.attn_every <= 0 else self.n_layers // self.attn_every

    def n_params_estimate(self) -> int:
        di = self.d_model * self.expand
        block = (2 * self.d_model + 4 * self.d_model * di + di + 2 * di * self.d_state + di * di + di
                 + di * self.d_state + di + 1)
        attn = (2 * self.d_model + 4 * self.d_model * self.d_model) if self.attn_every > 0 else 0
        head = 0 if self.tie_weights else self.vocab_size * self.d_model
        return self.vocab_size * self.d_model + self.n_layers * block + self.n_attn_layers * attn + head


class RotaryEmbedding(nn.Module):
    """Rotary position embedding tables (model.py:88-116), rebuilt when ``inv_freq`` is replaced or written."""

    def __init__(self, dim: int, max_seq_len: int = 8192, base: float = 10000.0) -> None:
        super().__init__()
        inv_freq = 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self._max_cached = 0
        self.register_buffer("cos_cached", torch.empty(0), persistent=False)
        self.register_buffer("sin_cached", torch.empty(0), persistent=False)
        self._made_from = Seen(inv_freq)                   # what the tables hold the angles of

    def _apply(self, fn, *args, **kw):
        current = self._made_from.still(self.inv_freq)
        super()._apply(fn, *args, **kw)
        if current:                                         # moved or cast, the tables with it
            self._made_from = Seen(self.inv_freq)
        return self

    def _build_cache(self, seq_len: int, device, dtype) -> None:
        if seq_len <= self._max_cached and self.cos_cached.dtype == dtype and self.cos_cached.device == device \
                and self._made_from.still(self.inv_freq):
            return
        self._max_cached = seq_len
        self._made_from = Seen(self.inv_freq)
        pos = torch.arange(seq_len, device=device, dtype=torch.float32)
        ang = torch.outer(pos, self.inv_freq.to(device))
        ang = torch.cat([ang, ang], dim=-1)
        self.cos_cached = ang.cos().to(dtype)
        self.sin_cached = ang.sin().to(dtype)

    def forward(self, x: Tensor, offset: int = 0) -> Tuple[Tensor, Tensor]:
        T = x.shape[-2]
        self._build_cache(offset + T, x.device, x.dtype)
        return self.cos_cached[offset:offset + T], self.sin_cached[offset:offset + T]


def _rotate_half(x: Tensor) -> Tensor:
    a, b = x.chunk(2, dim=-1)
    return torch.cat([-b, a], dim=-1)


def apply_rotary(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """RoPE on x [B, H, T, hd]."""
    return x * cos + _rotate_half(x) * sin


class SlidingWindowAttention(nn.Module):
    """Causal multi-head attention limited to the last ``window`` keys (model.py:129-181).

    For T <= window plain causal attention; for T > window query i sees keys
    j with i - window <= j <= i.  Stateless across calls, like the reference
    (a T=1 decode step attends to itself only).
    """

    def __init__(self, d_model: int, n_heads: int = 4, window: int = 256, max_seq_len: int = 8192) -> None:
        super().__init__()
        self.d_model = d_model
        self.n_heads = n_heads
        self.head_dim = d_model // n_heads
        self.window = window
        self.norm = nn.RMSNorm(d_model)
        self.qkv = nn.Linear(d_model, d_model * 3, bias=False)
        self.o_proj = nn.Linear(d_model, d_model, bias=False)
        self.rope = RotaryEmbedding(self.head_dim, max_seq_len=max_seq_len)
        self._mask = None

    def _window_mask(self, T: int, device) -> Tensor:
        m = getattr(self, "_mask", None)
        if m is None or m.shape[-1] != T or m.device != device:
            i = torch.arange(T, device=device)
            rel = i[:, None] - i[None, :]
            m = self._mask = ((rel >= 0) & (rel <= self.window))[None, None]
        return m

    def forward(self, x: Tensor) -> Tensor:
        if x.is_cuda and x.dtype == torch.bfloat16 and self.head_dim in (64, 128):
            return self.forward_native(x)
        return self.forward_torch(x)

    def forward_native(self, x: Tensor, workspace: Optional[Tensor] = None) -> Tensor:
        """The whole layer in one native call (nt_attention_forward): RMSNorm, the
        qkv projection and o_proj + residual on the tcgen05 GEMM, RoPE and the
        windowed causal softmax attention in one kernel."""
        from .. import native
        cos, sin = self.rope(x)                     # rows [0, T) in x's dtype
        return native.attention_forward(x, self.norm.weight, self.qkv.weight, self.o_proj.weight, self.n_heads,
                                        self.window, cos, sin, workspace=workspace)

    def forward_cached(self, x: Tensor, cache: AttentionCache, layer: str) -> Tensor:
        """The layer with a memory: x [B, T, d_model], the last T of cache.lengths tokens.

        The first call of a sequence is the plain layer (its keys are all in x) and
        leaves its window in the cache; later calls attend over the cache."""
        from .. import native
        B, T, dm = x.shape
        H, hd = self.n_heads, self.head_dim
        held = getattr(self, "_rope_freq", None)
        src = self.rope.inv_freq
        if held is None or not held[0].still(src) or held[1].device != x.device:
            held = self._rope_freq = (Seen(src), src.to(x.device, torch.float32))
        freq = held[1]
        before = cache.filled - T                       # tokens of the sequences ahead of x

        def heads(a: int, b: int) -> Tensor:            # q | k | v heads [B, b - a, 3H, hd] of tokens a..b-1 of x
            qkv = native.lm_head(x[:, a:b], self.norm.weight, self.qkv.weight)      # RMSNorm and one projection
            return qkv.view(B, b - a, 3 * H, hd)

        if before == 0:
            # the window of the tokens to come, from a page's first slot on
            a = max(0, T - self.window) // cache.page * cache.page
            qkv = heads(a, T)
            k = native.rotary(qkv[:, :, H:2 * H], torch.arange(a, T, device=x.device), freq)
            cache.append(layer, k, qkv[:, :, 2 * H:], cache.lengths)
            return self.forward(x)
        out = []
        for a in range(0, T, cache.max_step):
            b = min(T, a + cache.max_step)
            qkv = heads(a, b)
            lengths = cache.lengths - (T - b) if b < T else cache.lengths
            pos = lengths[:, None] + torch.arange(a - b, 0, device=x.device)
            native.rotary(qkv[:, :, :2 * H], pos, freq, out=qkv[:, :, :2 * H])
            cache.append(layer, qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], lengths)
            out.append(cache.attend(layer, qkv[:, :, :H], lengths).view(B, b - a, dm))
        o = out[0] if len(out) == 1 else torch.cat(out, dim=1)
        return native.attention_output(o, self.o_proj.weight, x)

    def forward_torch(self, x: Tensor) -> Tensor:
        """The reference's op sequence (fp32, CPU tensors, head dims other than 64 and 128)."""
        B, T, _ = x.shape
        h = self.norm(x)
        q, k, v = self.qkv(h).view(B, T, 3, self.n_heads, self.head_dim).permute(2, 0, 3, 1, 4).unbind(0)
        cos, sin = self.rope(q)
        q = apply_rotary(q, cos, sin)
        k = apply_rotary(k, cos, sin)
        if T <= self.window:
            o = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        else:
            o = F.scaled_dot_product_attention(q, k, v, attn_mask=self._window_mask(T, x.device))
        return self.o_proj(o.transpose(1, 2).reshape(B, T, self.d_model)) + x


# the largest penalty or bias of `generate`: its sum over a history stays finite in bf16 too
MAX_BIAS = 1e20


def allowed_words(mask: Optional[Tensor], batch: int, vocab: int) -> Optional[Tensor]:
    """A mask of the tokens that may come next as the words of ``native.pack_allowed``,
    checked for a token in every row (one read of the device)."""
    if mask is None:
        return None
    from .. import native
    n = vocab if mask.dtype == torch.bool else (vocab + 31) // 32
    if mask.dtype not in (torch.bool, torch.int32, torch.uint32) or mask.dim() != 2 or mask.shape[0] not in (1, batch) \
            or mask.shape[1] < n:
        raise ValueError(f"allowed must be boolean [{batch} or 1, {vocab}] or int32 words [{batch} or 1, {(vocab + 31) // 32}], "
                         f"got {mask.dtype} {tuple(mask.shape)}")
    words = native.pack_allowed(mask) if mask.dtype == torch.bool else mask
    bits = words.view(torch.int32)
    some = (bits[:, :vocab // 32] != 0).any(1)
    if vocab % 32:
        some = some | ((bits[:, vocab // 32] & ((1 << vocab % 32) - 1)) != 0)
    if not bool(some.all()):
        raise ValueError("allowed leaves no token for a sequence")
    return words


class NeuraTensorModel(nn.Module):
    """Embedding -> FusedSpikeBlocks (+ attention every ``attn_every``) -> RMSNorm -> tied lm_head."""

    def __init__(self, config: ModelConfig) -> None:
        super().__init__()
        self.config = config
        self.embedding = nn.Embedding(config.vocab_size, config.d_model)
        self.blocks = nn.ModuleList()
        self.attn_layers = nn.ModuleDict()
        for i in range(config.n_layers):
            self.blocks.append(FusedSpikeBlock(d_model=config.d_model, d_state=config.d_state,
                                               expand=config.expand, beta_init=config.beta_init,
                                               learn_beta=config.learn_beta, dropout=config.dropout))
            if config.attn_every > 0 and (i + 1) % config.attn_every == 0:
                self.attn_layers[str(i)] = SlidingWindowAttention(d_model=config.d_model, n_heads=config.attn_heads,
                                                                  window=config.attn_window,
                                                                  max_seq_len=config.max_seq_len)
        self.norm = nn.RMSNorm(config.d_model)
        self.lm_head = nn.Linear(config.d_model, config.vocab_size, bias=False)
        if config.tie_weights:
            self.lm_head.weight = self.embedding.weight
        self._init_weights()
        self._ws = None

    def _init_weights(self) -> None:
        nn.init.normal_(self.embedding.weight, std=0.02)
        for blk in self.blocks:
            nn.init.xavier_uniform_(blk.in_proj.weight)
            nn.init.xavier_uniform_(blk.out_proj.weight)
        for attn in self.attn_layers.values():
            nn.init.xavier_uniform_(attn.qkv.weight)
            nn.init.xavier_uniform_(attn.o_proj.weight)

    @classmethod
    def from_preset(cls, name: str) -> "NeuraTensorModel":
        from ..config.presets import get_preset
        return cls(get_preset(name))

    def _workspace(self, x: Tensor) -> Tensor:
        """One block workspace reused by every block of a forward."""
        from .. import native
        c = self.config
        B, T, _ = x.shape
        n = native.block_workspace_bytes(x.dtype, B, T, c.d_model, c.d_model * c.expand, c.d_state)
        ws = getattr(self, "_ws", None)
        if ws is None or ws.numel() < n or ws.device != x.device:
            self._ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        return self._ws

    # The kernels index activations with 32-bit element offsets in places; a
    # forward whose widest activation (the in_proj output [rows, 2*d_inner] or
    # attention's qkv [rows, 3*d_model]) would pass 2^30 elements runs the
    # batch in groups of sequences instead (sequences are independent, so
    # the result is the same).
    MAX_ACTIVATION_ELEMS = 1 << 30

    def group_size(self, seq: int) -> int:
        """Sequences of length `seq` that one pass of the blocks takes at most."""
        c = self.config
        width = max(2 * c.d_model * c.expand, 3 * c.d_model)
        return max(1, self.MAX_ACTIVATION_ELEMS // (max(seq, 1) * width))

    def forward_device(self, input_ids: Tensor, states: Optional[List[Optional[BlockState]]] = None,
                       workspace: Optional[Tensor] = None, last_only: bool = False,
                       attn_cache: Optional[AttentionCache] = None):
        """Forward without any host sync: returns (logits, states, per-layer spike counts on device).

        ``last_only``: logits of the last position only ([B, 1, vocab]), as a
        generation prefill needs them.  ``attn_cache``: the attention layers see
        the tokens of earlier calls with it, and it moves on by this call's."""
        if states is None:
            states = [None] * len(self.blocks)
        if input_ids.shape[1] > self.config.max_seq_len:
            import warnings
            warnings.warn(f"Input sequence length {input_ids.shape[1]} exceeds max_seq_len "
                          f"{self.config.max_seq_len}; truncating.", UserWarning, stacklevel=3)
            input_ids = input_ids[:, : self.config.max_seq_len]
        B, T = input_ids.shape
        if attn_cache is not None:
            attn_cache.require_batch(B)
            attn_cache.advance(T)
        g = self.group_size(T)
        if B <= g:
            return self._forward_rows(input_ids, states, workspace, last_only, attn_cache)
        parts = []
        for a in range(0, B, g):
            sub = [None if s is None else BlockState(membrane=s.membrane[a:a + g], ssm_state=s.ssm_state[a:a + g])
                   for s in states]
            part = None if attn_cache is None else attn_cache.rows(a, min(a + g, B))
            parts.append(self._forward_rows(input_ids[a:a + g], sub, workspace, last_only, part))
        logits = torch.cat([p[0] for p in parts])
        state_cls = self.blocks[0]._state_cls
        new_states = [state_cls(membrane=torch.cat([p[1][i].membrane for p in parts]),
                                ssm_state=torch.cat([p[1][i].ssm_state for p in parts]))
                      for i in range(len(self.blocks))]
        counts = torch.stack([p[2] for p in parts]).sum(0)
        return logits, new_states, counts

    def _forward_rows(self, input_ids: Tensor, states: List[Optional[BlockState]], workspace: Optional[Tensor],
                      last_only: bool, attn_cache: Optional[AttentionCache] = None):
        from .. import native
        x = native.embedding(input_ids, self.embedding.weight)
        counts = torch.zeros(len(self.blocks), dtype=torch.int64, device=x.device)
        ws = workspace if workspace is not None else self._workspace(x)
        new_states: List[BlockState] = []
        with torch.no_grad():
            for i, (blk, st) in enumerate(zip(self.blocks, states)):
                x, ns = blk.forward_native(x, st, counts[i], workspace=ws)
                new_states.append(ns)
                key = str(i)
                if key in self.attn_layers:
                    attn = self.attn_layers[key]
                    x = attn(x) if attn_cache is None else attn.forward_cached(x, attn_cache, key)
            if last_only:
                x = x[:, -1:]
            # final RMSNorm + tied lm_head on the tcgen05 GEMM; the block
            # workspace is free again here and holds the normalised rows
            logits = native.lm_head(x, self.norm.weight, self.lm_head.weight, workspace=ws)
        return logits, new_states, counts

    def metrics_from_counts(self, counts: List[int], numel: int, dtype: torch.dtype) -> Dict:
        rates = [rate_like_reference(c, numel, dtype) for c in counts]
        mean = sum(rates) / len(rates)
        return {"spike_rate": mean, "per_layer_spike_rate": rates, "estimated_sparsity_pct": (1.0 - mean) * 100}

    def forward(self, input_ids: Tensor, states: Optional[List[Optional[BlockState]]] = None
                ) -> Tuple[Tensor, List[BlockState], Dict]:
        """input_ids [B, T] -> (logits [B, T, vocab], states, metrics) (model.py:240-293)."""
        logits, new_states, counts = self.forward_device(input_ids, states)
        B, T = logits.shape[:2]
        di = self.config.d_model * self.config.expand
        metrics = self.metrics_from_counts(counts.tolist(), B * T * di, logits.dtype)
        return logits, new_states, metrics

    def count_parameters(self) -> int:
        return sum(p.numel() for p in self.parameters())

    def count_trainable_parameters(self) -> int:
        return sum(p.numel() for p in self.parameters() if p.requires_grad)

    def _graph_signature(self, cache_tokens: int):
        """What a captured forward reads besides its own buffers and its layers' frequencies.  With an attention
        cache the layers rotate by those alone (``forward_cached``), without one by their tables of them."""
        layers = self.attn_layers.values()
        return (tuple((p.data_ptr(), p._version) for p in self.parameters()),
                () if cache_tokens else tuple((a.rope.cos_cached.data_ptr(), a.rope.sin_cached.data_ptr()) for a in layers))

    @torch.no_grad()
    def step_graph(self, batch: int, seq: int, device, dtype, cache_tokens: int = 0):
        """The captured forward for this (batch, length) (``inference/decode.py``);
        with ``cache_tokens`` the graph has an attention cache of its own for that many
        tokens a sequence (``graph.attn_cache``).
        A graph holds raw addresses, so it is rebuilt when a parameter changes
        (version or storage), an attention layer's frequencies do, or, where it reads
        them, its RoPE tables were rebuilt; the four most recently used shapes are kept."""
        from ..inference.decode import StepGraph
        sig = self._graph_signature(cache_tokens)
        key = (batch, seq, str(device), dtype, cache_tokens)
        cache = self.__dict__.setdefault("_step_graphs", {})
        hit = cache.pop(key, None)
        if hit is None or hit[0] != sig or not hit[1].frequencies_hold():
            hit = None
            while len(cache) >= 4:
                cache.pop(next(iter(cache)))
            with torch.inference_mode(False), torch.no_grad():      # its buffers are written in later calls, which may be outside it
                graph = StepGraph(self, batch, seq, torch.device(device), dtype, cache_tokens)
            hit = (self._graph_signature(cache_tokens), graph)      # its warm-up may have built the tables
        cache[key] = hit                          # most recently used last
        return hit[1]

    def decode_graph(self, batch: int, device, dtype, cache_tokens: int = 0):
        """The captured single-token step for this batch size."""
        return self.step_graph(batch, 1, device, dtype, cache_tokens)

    @torch.no_grad()
    def beam_step(self, prompts: int, beams: int, device, dtype, cache_tokens: int, length_penalty: float,
                  stop: Tuple[int, ...], capture: bool = True):
        """A beam search's step (``inference/beams.py``), captured ones kept like ``step_graph``'s (the last two);
        ``cache_tokens`` 0: without an attention memory."""
        from ..inference.beams import BeamStep
        if not capture:
            return BeamStep(self, prompts, beams, device, dtype, cache_tokens, length_penalty, stop, capture=False)
        cache_tokens = -(-cache_tokens // 1024) * 1024      # so that calls of other lengths find the same graph
        key = (prompts, beams, str(device), dtype, cache_tokens, length_penalty, stop)
        cache = self.__dict__.setdefault("_beam_steps", {})
        hit = cache.pop(key, None)
        if hit is None or hit[0] != self._graph_signature(cache_tokens) or not hit[1].frequencies_hold():
            hit = None
            while len(cache) >= 2:
                cache.pop(next(iter(cache)))
            with torch.inference_mode(False), torch.no_grad():
                step = BeamStep(self, prompts, beams, torch.device(device), dtype, cache_tokens, length_penalty, stop)
            hit = (self._graph_signature(cache_tokens), step)
        cache[key] = hit
        return hit[1]

    def generate(self, input_ids: Tensor, max_new_tokens: int = 50, temperature: float = 1.0, top_k: int = 50,
                 top_p: float = 1.0, repetition_penalty: float = 1.0, stop_tokens: Optional[List[int]] = None,
                 states: Optional[List[Optional[BlockState]]] = None,
                 use_graph: bool = True, attn_cache: Union[bool, AttentionCache] = False,
                 frequency_penalty: float = 0.0, presence_penalty: float = 0.0,
                 logit_bias: Optional[Dict[int, float]] = None,
                 allowed: Union[None, Tensor, Callable[[Tensor], Optional[Tensor]]] = None,
                 num_beams: int = 1, length_penalty: float = 0.0) -> Tuple[Tensor, List[BlockState]]:
        """Autoregressive sampling with carried block state (model.py:301-370).

        On CUDA the per-token steps replay one captured graph of the whole model
        (``inference/decode.py``); ``use_graph=False`` runs them one launch at a
        time.  Both run the same kernels on the same inputs.

        Beyond the reference: ``attn_cache`` lets the attention layers see their window
        of earlier tokens instead of the new one alone (True: for this call; an
        ``AttentionCache`` carries on and is left behind the last token that was run; one
        without room for the call is refused);
        ``frequency_penalty`` and ``presence_penalty`` are taken off per occurrence of a
        generated token and for any; ``logit_bias`` maps token ids to what is added;
        ``allowed`` is a mask of the tokens that may come next, boolean [B or 1, vocab] or
        the int32 words of ``native.pack_allowed``, or a function of the tokens so far
        that returns one (or None).  Penalties and biases are finite (at most 1e20), and a
        mask that leaves a sequence no token is refused; a function's is read for that at
        every step.

        ``num_beams`` above 1 searches instead of sampling (``inference/beams.py``): the
        continuation of largest log-probability among the beams, divided by its length to
        the power of ``length_penalty``; a beam ends with a stop token (then the first of them
        fills up) or with ``max_new_tokens``.  It takes ``stop_tokens``, ``states``,
        ``use_graph`` and ``attn_cache=True``; what shapes a distribution to sample from is
        refused (but for ``top_k``, which is not looked at).  The states are the best beams', which have not run their last
        token, that is the stop token of a beam that ended: what fills up behind it does not reach them."""
        from .. import native
        self.eval()
        if num_beams != 1:
            for name, given in (("temperature", temperature != 1.0), ("top_p", top_p != 1.0), ("repetition_penalty", repetition_penalty != 1.0),
                                ("frequency_penalty", bool(frequency_penalty)), ("presence_penalty", bool(presence_penalty)),
                                ("logit_bias", bool(logit_bias)), ("allowed", allowed is not None),
                                ("an AttentionCache", isinstance(attn_cache, AttentionCache))):
                if given:
                    raise ValueError(f"beam search takes no {name}")
            if not 2 <= num_beams <= 64 or input_ids.shape[0] * num_beams > 1024:
                raise ValueError(f"num_beams must be 1 to 64 and at most 1024 in all, got {num_beams} for {input_ids.shape[0]} prompts")
            if not math.isfinite(length_penalty):
                raise ValueError(f"length_penalty must be finite, got {length_penalty}")
            if any(not 0 <= t < self.config.vocab_size for t in stop_tokens or []):
                raise ValueError(f"stop_tokens outside the vocabulary of {self.config.vocab_size}")
            if max_new_tokens < 1 or input_ids.shape[1] < 1:
                raise ValueError("beam search needs a prompt and at least one new token")
            from ..inference.beams import beam_search
            with torch.no_grad():
                return beam_search(self, input_ids, max_new_tokens, num_beams, float(length_penalty), list(stop_tokens or []), states,
                                   use_graph, bool(attn_cache))
        if length_penalty:
            raise ValueError("length_penalty is for num_beams above 1")
        out = input_ids
        B, prompt = out.shape
        # what would leave a row without a finite largest logit is refused before anything runs:
        # its probabilities are NaN, and there is nothing to sample
        for name, v in (("frequency_penalty", frequency_penalty), ("presence_penalty", presence_penalty)):
            if not abs(v) <= MAX_BIAS:
                raise ValueError(f"{name} must be at most {MAX_BIAS:g} in size, got {v}")
        if not math.isfinite(repetition_penalty) or repetition_penalty == 0:
            raise ValueError(f"repetition_penalty must be finite and not 0, got {repetition_penalty}")
        for i, v in (logit_bias or {}).items():
            if not 0 <= i < self.config.vocab_size:
                raise ValueError(f"logit_bias names token {i} outside the vocabulary of {self.config.vocab_size}")
            if not abs(v) <= MAX_BIAS:
                raise ValueError(f"logit_bias must be at most {MAX_BIAS:g} in size, got {v} for token {i}")
        fixed = None if callable(allowed) else allowed_words(allowed, B, self.config.vocab_size)
        stop = set(stop_tokens or [])
        if isinstance(attn_cache, AttentionCache):
            # a stop token may end the call at once, without one all tokens are run
            attn_cache.require_batch(B)
            attn_cache.require(min(prompt, self.config.max_seq_len) + (0 if stop else max_new_tokens))
        want_graph = use_graph and out.is_cuda and max_new_tokens > 1
        graph = cache = None
        if isinstance(attn_cache, AttentionCache):
            cache, want_graph = attn_cache, False       # a graph has its own
        elif attn_cache:
            tokens = min(prompt, self.config.max_seq_len) + max_new_tokens
            if want_graph:
                tokens = -(-tokens // 1024) * 1024      # so that calls of other lengths find the same graph
                graph = self.decode_graph(B, out.device, self.lm_head.weight.dtype, tokens)
                cache = graph.attn_cache
                cache.reset()
            else:
                cache = AttentionCache(self.config, B, tokens, out.device)
        logits, states, _ = self.forward_device(out, states, last_only=True, attn_cache=cache)
        nxt_logits = logits[:, -1, :]
        if want_graph:
            graph = graph or self.decode_graph(B, out.device, logits.dtype)
            graph.load_states(states)
        made = torch.full((B,), prompt, dtype=torch.int32, device=out.device) if frequency_penalty or presence_penalty else None
        bias_ids = bias = None
        if logit_bias:
            bias_ids = torch.tensor([list(logit_bias)], dtype=torch.int64, device=out.device).expand(B, -1)
            bias = torch.tensor([list(logit_bias.values())], dtype=torch.float32, device=out.device).expand(B, -1)
        # top_k = 1 without nucleus filtering leaves the tied row maxima with
        # equal probability: one kernel picks among them with a uniform drawn
        # here for every step at once (the other filters run as written)
        greedy = out.is_cuda and top_k == 1 and top_p >= 1.0
        if greedy:
            u_all = torch.rand((max_new_tokens, out.shape[0]), device=out.device)
        for step in range(max_new_tokens):
            if repetition_penalty != 1.0:
                # once per occurrence, as the reference's loop over out[b] does
                native.logits_process(nxt_logits, tokens=out, repetition=repetition_penalty, each=True, out=nxt_logits)
            mask = allowed_words(allowed(out), B, self.config.vocab_size) if callable(allowed) else fixed
            if made is not None or bias is not None or mask is not None:
                native.logits_process(nxt_logits, tokens=out if made is not None else None, prompt_lengths=made,
                                      frequency=frequency_penalty, presence=presence_penalty, bias_ids=bias_ids, bias=bias,
                                      allowed=mask, out=nxt_logits)
            if temperature != 1.0:
                nxt_logits = nxt_logits / temperature
            if greedy:
                tok = native.greedy_tokens(nxt_logits, u_all[step])
            elif top_k > 0:
                kth = torch.topk(nxt_logits, min(top_k, nxt_logits.size(-1))).values[:, [-1]]
                nxt_logits[nxt_logits < kth] = float("-inf")
            if top_p < 1.0:
                srt, idx = torch.sort(nxt_logits, descending=True, dim=-1)
                p = torch.softmax(srt, dim=-1)
                drop = p.cumsum(-1) - p > top_p
                srt = srt.masked_fill(drop, float("-inf"))
                nxt_logits = torch.zeros_like(nxt_logits).scatter_(-1, idx, srt)
            if not greedy:
                # a penalty per occurrence can carry logits past the largest number
                if repetition_penalty != 1.0 and not bool(nxt_logits.amax(-1).isfinite().all()):
                    raise ValueError(f"repetition_penalty {repetition_penalty} leaves no finite logits to sample from")
                tok = torch.multinomial(torch.softmax(nxt_logits, dim=-1), num_samples=1)
            out = torch.cat([out, tok], dim=1)
            if stop and tok.item() in stop:
                break
            if graph is not None:
                nxt_logits = graph.step(tok).clone()
            else:
                logits, states, _ = self.forward_device(tok, states, attn_cache=cache)
                nxt_logits = logits[:, -1, :]
        if graph is not None:
            states = graph.states()
        return out, states

    def info(self) -> str:
        c = self.config
        rows = [("Parameters", f"{self.count_parameters():,}"), ("Layers", c.n_layers), ("d_model", c.d_model),
                ("d_state", c.d_state), ("expand", c.expand), ("vocab", f"{c.vocab_size:,}"),
                ("max_seq_len", c.max_seq_len)]
        if c.attn_every > 0:
            rows += [("attn_every", c.attn_every), ("attn_heads", c.attn_heads), ("attn_window", c.attn_window),
                     ("attn_layers", c.n_attn_layers)]
        bar = "=" * 60
        body = "\n".join(f"  {k + ':':<14} {v:>14}" for k, v in rows)
        return f"{bar}\n  NeuraTensor v4 (B200 kernels) -- {c.model_name.upper()}\n{bar}\n{body}\n{bar}"


NeuraTensor = NeuraTensorModel
