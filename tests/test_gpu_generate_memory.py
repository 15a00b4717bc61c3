"""Generation with an attention memory and penalties: the step operators together, as the
model uses them (B200)."""
import math

import pytest
import torch

from test_gpu_step_ops import BF16, DEV, E4M3, F32, U32, attention64, close, half

pytestmark = pytest.mark.gpu


def config(**kw):
    from neuratensor_b200 import ModelConfig
    return ModelConfig(**{**dict(vocab_size=1000, d_model=128, n_layers=4, d_state=16, max_seq_len=512, attn_every=2,
                                 attn_heads=2, attn_window=40), **kw})


def rotate64(x, pos, freq):
    a = pos.double()[..., None, None] * freq.double()
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h].double(), x[..., h:].double()
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prompt,chunks,page", [(1, [1] * 70, 16), (100, [1] * 80, 16), (37, [1, 20, 1, 5, 33], 32), (200, [16, 1], 64)])
def test_layer_with_memory(dtype, prompt, chunks, page):
    """Every call against its definition on the cache it leaves: RMSNorm, projection, rotation at the
    tokens' positions, the window through the ring of pages, output projection and residual."""
    from neuratensor_b200 import AttentionCache
    from neuratensor_b200.core.model import SlidingWindowAttention
    torch.manual_seed(1)
    B, dm, H, window = 2, 128, 2, 40
    cfg = config()
    attn = SlidingWindowAttention(dm, H, window).to(DEV).to(dtype)
    cache = AttentionCache(cfg, B, prompt + sum(chunks), DEV, page=page)
    layer = next(iter(cache.layers))
    freq = attn.rope.inv_freq.float()
    with torch.no_grad():
        x = torch.randn(B, prompt, dm, device=DEV).to(dtype)
        cache.advance(prompt)
        assert torch.equal(attn.forward_cached(x, cache, layer), attn(x))         # the first call is the plain layer
        for T in chunks:
            x = torch.randn(B, T, dm, device=DEV).to(dtype)
            cache.advance(T)
            got = attn.forward_cached(x, cache, layer)
            n = cache.filled
            # q from float64 RMSNorm and projection of what the layer was given
            w = attn.norm.weight.double()
            xn = (x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + torch.finfo(F32).eps) * w)
            q = (xn @ attn.qkv.weight.double()[:dm].t()).view(B, T, H, dm // H)
            q = rotate64(q, (n - T + torch.arange(T, device=DEV)).expand(B, T), freq)
            want, tol = attention64(q.float() if dtype == F32 else q.to(BF16), cache.layers[layer], cache.table, [n] * B, [T] * B, window, page)
            o = want.reshape(B, T, dm) @ attn.o_proj.weight.double().t() + x.double()
            # q, its rotation, o and the sum round in the layer's type, the norm and the projections on the way: q is
            # off by at most 4 half steps of its terms, which moves scores, and so weights, by that times sum |q k|
            Wo = attn.o_proj.weight.double().abs()
            kc, ks = cache.layers[layer][:2]
            kmax = (kc.float().abs().nan_to_num(0).amax((2, 3)) * ks).max().double()
            qterms = (xn.abs() @ attn.qkv.weight.double()[:dm].abs().t()).view(B, T, H, dm // H).sum(-1).max()
            shift = 2 * 4 * half(dtype) * qterms * kmax / math.sqrt(dm // H)
            vmax = (cache.layers[layer][2].float().abs().nan_to_num(0).amax((2, 3)) * cache.layers[layer][3]).max().double()
            bound = (tol.reshape(B, T, dm) + (shift + 2 * half(dtype)) * vmax) @ Wo.t() + 3 * half(dtype) * (o.abs() + x.double().abs())
            close(got, o, half(dtype), bound)
            # far closer than that in the mean: a key missed or doubled would not be.  The residual sum itself rounds
            # by up to half a step of each of its elements, in the norm half a step of the norm
            assert (got.double() - o).norm() <= half(dtype) * o.norm() + (4e-2 if dtype == BF16 else 1e-4) * (o - x.double()).norm()


def test_cache_ring_and_refusals():
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    cfg = config()
    c = AttentionCache(cfg, 3, 300, DEV, page=16, max_step=8)
    assert c.ring == 5 and c.max_tokens == 304 and len(c.layers) == 2
    assert c.table[1].tolist() == [5 + i % 5 for i in range(19)]
    part = c.rows(1, 3)
    c.advance(7)
    assert part.lengths.tolist() == [7, 7] and c.lengths.data_ptr() != part.lengths.data_ptr()
    with pytest.raises(ValueError, match="do not fit"):
        c.advance(298)
    c.reset()
    assert c.filled == 0 and c.lengths.sum() == 0
    for bad in (dict(page=8), dict(batch=0), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            AttentionCache(**{**dict(config=cfg, batch=1, max_tokens=10, device=DEV), **bad})
    with pytest.raises(ValueError, match="no attention"):
        AttentionCache(config(attn_every=0), 1, 10, DEV)
    with pytest.raises(ValueError, match="64 or 128"):
        AttentionCache(config(attn_heads=4), 1, 10, DEV)
    model = NeuraTensorModel(cfg).to(DEV).to(BF16).eval()
    with pytest.raises(ValueError, match="for 3 sequences"):
        model.forward_device(torch.zeros(2, 4, dtype=torch.int64, device=DEV), attn_cache=c)


@pytest.mark.parametrize("prompt", [1, 16, 130])
def test_generate_with_memory_graph_matches_eager(prompt):
    """The captured step with its own cache equals the step launched kernel by kernel, twice, and a
    longer prompt reuses it; the memory changes what is generated."""
    from neuratensor_b200 import NeuraTensorModel
    torch.manual_seed(5)
    model = NeuraTensorModel(config()).to(DEV).to(BF16).eval()
    ids = torch.randint(0, 1000, (2, prompt), device=DEV)
    outs = []
    with torch.no_grad():
        for kw in (dict(use_graph=False), dict(), dict()):
            torch.manual_seed(7)
            outs.append(model.generate(ids, max_new_tokens=60, top_k=1, attn_cache=True, **kw)[0])
        torch.manual_seed(7)
        plain = model.generate(ids, max_new_tokens=60, top_k=1)[0]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[1], outs[2])
    assert not torch.equal(outs[0], plain)
    assert len([k for k in model._step_graphs if k[4]]) == 1


def test_generate_carries_a_cache_on():
    """An AttentionCache that is given goes on where the last call left it."""
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    torch.manual_seed(6)
    model = NeuraTensorModel(config()).to(DEV).to(BF16).eval()
    ids = torch.randint(0, 1000, (2, 30), device=DEV)
    cache = AttentionCache(model.config, 2, 200, DEV)
    with torch.no_grad():
        out, states = model.generate(ids, max_new_tokens=5, top_k=1, attn_cache=cache)
        assert cache.filled == 35 and cache.lengths.tolist() == [35, 35]
        out2, _ = model.generate(out[:, -1:], max_new_tokens=3, top_k=1, attn_cache=cache, states=states)
    assert cache.filled == 39 and out2.shape == (2, 4)


def test_forward_in_sequence_groups_with_memory():
    """A batch that runs in groups of sequences fills and reads the cache as one pass does."""
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    torch.manual_seed(8)
    model = NeuraTensorModel(config()).to(DEV).to(BF16).eval()
    ids = torch.randint(0, 1000, (5, 50), device=DEV)
    res = []
    for groups in (False, True):
        if groups:
            model.group_size = lambda seq: 2
        cache = AttentionCache(model.config, 5, 64, DEV)
        with torch.no_grad():
            _, st, _ = model.forward_device(ids, attn_cache=cache)
            logits, _, _ = model.forward_device(ids[:, :1], st, attn_cache=cache)
        res.append((logits, [t.view(torch.uint8) if t.dtype == E4M3 else t for l in cache.layers.values() for t in l]))
    assert torch.equal(res[0][0], res[1][0])
    assert all(torch.equal(a, b) for a, b in zip(res[0][1], res[1][1]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_generate_repetition_penalty_is_the_loop(dtype):
    """The tokens that the host loop over the history gave."""
    from neuratensor_b200 import NeuraTensorModel
    torch.manual_seed(9)
    model = NeuraTensorModel(config(vocab_size=60)).to(DEV).to(dtype).eval()
    ids = torch.randint(0, 60, (2, 12), device=DEV)
    r, new = 1.13, 20
    with torch.no_grad():
        torch.manual_seed(11)
        got, _ = model.generate(ids, max_new_tokens=new, top_k=5, repetition_penalty=r, use_graph=False)
        torch.manual_seed(11)
        out = ids
        logits, states, _ = model.forward_device(out, None, last_only=True)
        for _ in range(new):
            nxt = logits[:, -1, :]
            for b in range(out.shape[0]):
                for tok in out[b].tolist():
                    v = nxt[b, tok]
                    nxt[b, tok] = v / r if v > 0 else v * r
            kth = torch.topk(nxt, 5).values[:, [-1]]
            nxt[nxt < kth] = float("-inf")
            tok = torch.multinomial(torch.softmax(nxt, dim=-1), num_samples=1)
            out = torch.cat([out, tok], dim=1)
            logits, states, _ = model.forward_device(tok, states)
    assert torch.equal(got, out)


def test_generate_penalties_biases_and_masks():
    from neuratensor_b200 import InferenceEngine, NeuraTensorModel
    torch.manual_seed(10)
    eng = InferenceEngine(NeuraTensorModel(config()), device=DEV, dtype=BF16)
    ids = torch.randint(0, 1000, (2, 10))
    out = eng.generate(ids, max_new_tokens=8, top_k=1, logit_bias={17: 1e4})
    assert (out[:, 10:] == 17).all()
    out = eng.generate(ids, max_new_tokens=8, top_k=1, logit_bias={17: 1e4}, presence_penalty=2e4, attn_cache=True)
    assert (out[:, 10] == 17).all() and (out[:, 11:] != 17).all()            # once made, its bias is outweighed
    out = eng.generate(ids, max_new_tokens=8, top_k=1, logit_bias={17: 1e4}, frequency_penalty=4e3)
    assert (out[:, 10:13] == 17).all() and (out[:, 13:] != 17).all()         # 1e4 - 3 * 4e3 < 0 beside logits of a few units
    mask = torch.zeros(1, 1000, dtype=torch.bool, device=DEV)
    mask[0, 100:110] = True
    out = eng.generate(ids, max_new_tokens=12, top_k=50, allowed=mask)
    assert ((out[:, 10:] >= 100) & (out[:, 10:] < 110)).all()

    def even_then_odd(tokens):                                              # a grammar: the next token's parity alternates
        m = torch.zeros(2, 1000, dtype=torch.bool, device=DEV)
        m[:, tokens.shape[1] % 2::2] = True
        return m

    out = eng.generate(ids, max_new_tokens=9, top_k=50, allowed=even_then_odd, attn_cache=True)
    assert torch.equal(out[:, 10:] % 2, (torch.arange(10, 19, device=DEV) % 2).expand(2, -1))
    with pytest.raises(ValueError, match="outside the vocabulary"):
        eng.generate(ids, max_new_tokens=2, logit_bias={1000: 1.0})
    from neuratensor_b200 import native
    assert native.device_error_flags(0) == 0


def test_long_contexts_with_scaled_frequencies():
    """The frequency forms by their formulas, and a rotation with them at a far position."""
    from neuratensor_b200 import native, rotary_frequencies
    D, s = 64, 8.0
    i = torch.arange(0, D, 2, dtype=torch.float64) / D
    plain, m = rotary_frequencies(D)
    assert m == 1.0 and torch.equal(plain, (10000.0 ** -i).float())
    lin, m = rotary_frequencies(D, scaling="linear", factor=s)
    assert m == 1.0 and torch.equal(lin, (10000.0 ** -i / s).float())
    base, m = rotary_frequencies(D, scaling="base", factor=s)
    assert m == 1.0 and base[0] == 1.0 and abs(base[-1].item() * s / plain[-1].item() - 1) < 1e-6
    parts, m = rotary_frequencies(D, scaling="by_parts", factor=s, trained_len=2048)
    assert m == 1.0 + 0.1 * math.log(s) and torch.equal(parts[:8], plain[:8])      # 2048 F / 2 pi >= 32 there
    assert torch.allclose(parts[-3:], plain[-3:] / s)                               # and <= 1 here
    for bad in (dict(dim=3), dict(scaling="other"), dict(factor=0.5), dict(scaling="by_parts", slow=40.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**{**dict(dim=D), **bad})
    x = torch.randn(1, 5, 2, D, device=DEV)
    pos = torch.arange(10 ** 6, 10 ** 6 + 5, device=DEV)
    y = native.rotary(x, pos, parts.to(DEV), mscale=m)
    want = m * rotate64(x, pos[None], parts.to(DEV))
    mag = m * (x.abs() + torch.cat([x[..., D // 2:], x[..., :D // 2]], -1).abs()).double()
    close(y, want, U32, 8 * U32 * mag)


@pytest.mark.parametrize("top_k", [1, 50])
def test_generate_refuses_a_step_without_tokens(top_k):
    """A function whose mask runs empty at the third token: refused on the host, and the device goes on."""
    from neuratensor_b200 import InferenceEngine, NeuraTensorModel, native
    torch.manual_seed(12)
    eng = InferenceEngine(NeuraTensorModel(config()), device=DEV, dtype=BF16)
    ids = torch.randint(0, 1000, (2, 10))

    def closing(tokens):
        m = torch.ones(2, 1000, dtype=torch.bool, device=DEV)
        m[1] = tokens.shape[1] < 12
        return m

    with pytest.raises(ValueError, match="leaves no token"):
        eng.generate(ids, max_new_tokens=5, top_k=top_k, allowed=closing)
    assert eng.generate(ids, max_new_tokens=2, top_k=top_k, allowed=closing).shape == (2, 12)
    assert native.device_error_flags(0) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_negative_repetition_per_occurrence_is_the_loop(dtype):
    from neuratensor_b200 import native
    torch.manual_seed(13)
    x = torch.randn(2, 50, device=DEV).to(dtype)
    tokens = torch.randint(0, 50, (2, 120), device=DEV)
    want, r = x.clone(), -1.07
    for b in range(2):
        for tok in tokens[b].tolist():
            v = want[b, tok]
            want[b, tok] = v / r if v > 0 else v * r
    assert torch.equal(native.logits_process(x, tokens=tokens, repetition=r, each=True), want)


@pytest.mark.parametrize("r", [1.05, 1.07, 1.1, 1.15, 1.3, 0.9])
def test_repetition_per_occurrence_for_usual_penalties(r):
    """Bit for bit the loop in float32, where 1 / r rounded from float64 is not 1 / float32(r) (not for the last two)."""
    from neuratensor_b200 import native
    torch.manual_seed(14)
    x = torch.randn(2, 50, device=DEV)
    tokens = torch.randint(0, 50, (2, 120), device=DEV)
    want = x.clone()
    for b in range(2):
        for tok in tokens[b].tolist():
            v = want[b, tok]
            want[b, tok] = v / r if v > 0 else v * r
    assert torch.equal(native.logits_process(x, tokens=tokens, repetition=r, each=True), want)
