"""Generation with an attention memory, from call to call (B200)."""
import pytest
import torch

from test_gpu_generate_memory import config
from test_gpu_step_ops import BF16, DEV, E4M3, F32, close

pytestmark = pytest.mark.gpu


def steps(model, ids, tokens, graph):
    """Logits of the prompt's last position and of each of `tokens` [n, B], with a memory, captured or not."""
    from neuratensor_b200 import AttentionCache
    dtype = model.lm_head.weight.dtype
    with torch.no_grad():
        if graph:
            g = model.decode_graph(ids.shape[0], ids.device, dtype, 1024)
            cache = g.attn_cache
            cache.reset()
        else:
            cache = AttentionCache(model.config, ids.shape[0], 1024, DEV)
        logits, states, _ = model.forward_device(ids, last_only=True, attn_cache=cache)
        out = [logits[:, -1].clone()]
        if graph:
            g.load_states(states)
        for tok in tokens:
            if graph:
                out.append(g.step(tok[:, None]).clone())
            else:
                logits, states, _ = model.forward_device(tok[:, None], states, attn_cache=cache)
                out.append(logits[:, -1].clone())
    return torch.stack(out)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("how", ["replaced", "written"])
def test_captured_step_follows_the_frequencies(dtype, how):
    """Frequencies that change between two calls are the ones of the next call, captured or not."""
    from neuratensor_b200 import NeuraTensorModel, rotary_frequencies
    torch.manual_seed(21)
    model = NeuraTensorModel(config()).to(DEV).to(dtype).eval()
    ids, tokens = torch.randint(0, 1000, (2, 25), device=DEV), torch.randint(0, 1000, (6, 2), device=DEV)
    before = steps(model, ids, tokens, True)
    assert torch.equal(before, steps(model, ids, tokens, False))
    for factor in (4.0, 16.0):
        f, _ = rotary_frequencies(64, scaling="linear", factor=factor, device=DEV)
        for a in model.attn_layers.values():
            if how == "replaced":
                a.rope.inv_freq = f.clone()
            else:
                a.rope.inv_freq.copy_(f)
        torch.cuda.empty_cache()
        held = [torch.full((32,), 1e3, device=DEV) for _ in range(64)]          # whatever was freed is someone else's now
        after = steps(model, ids, tokens, True)
        assert torch.equal(after, steps(model, ids, tokens, False))
        assert not torch.equal(after[1:], before[1:])
        before = after
        del held


def test_a_longer_prompt_finds_the_same_captured_step():
    """On a model without tables, too: the step that is captured for the first call serves the next ones."""
    from neuratensor_b200 import NeuraTensorModel
    torch.manual_seed(22)
    model = NeuraTensorModel(config()).to(DEV).to(BF16).eval()
    graphs = []
    with torch.no_grad():
        for prompt in (5, 130, 60):
            ids = torch.randint(0, 1000, (2, prompt), device=DEV)
            out = model.generate(ids, max_new_tokens=20, top_k=1, attn_cache=True)[0]
            graphs.append(model.decode_graph(2, ids.device, BF16, 1024))
            cold, _ = model.generate(ids, max_new_tokens=20, top_k=1, attn_cache=True, use_graph=False)
            assert torch.equal(out, cold)
    assert graphs[0] is graphs[1] is graphs[2]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_carried_cache_holds_what_one_sequence_would(dtype):
    """Two calls on one cache against the same tokens run one after the other on a fresh one: codes, scales and
    lengths are equal, and every greedy token has its row's largest logit."""
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    torch.manual_seed(23)
    model = NeuraTensorModel(config()).to(DEV).to(dtype).eval()
    ids, more = torch.randint(0, 1000, (2, 50), device=DEV), torch.randint(0, 1000, (2, 20), device=DEV)
    carried, fresh = (AttentionCache(model.config, 2, 200, DEV, page=16) for _ in range(2))
    with torch.no_grad():
        first, states = model.generate(ids, max_new_tokens=30, top_k=1, attn_cache=carried)
        second, _ = model.generate(more, max_new_tokens=7, top_k=1, attn_cache=carried, states=states)
        assert first.shape == (2, 80) and second.shape == (2, 27)
        states = None
        for whole, prompt in ((first, 50), (second, 20)):
            logits, states, _ = model.forward_device(whole[:, :prompt], states, last_only=True, attn_cache=fresh)
            for t in range(prompt, whole.shape[1]):
                row, tok = logits[:, -1], whole[:, t:t + 1]
                assert torch.equal(row.gather(1, tok)[:, 0], row.amax(-1))
                logits, states, _ = model.forward_device(tok, states, attn_cache=fresh)
    assert carried.filled == fresh.filled == 107 and torch.equal(carried.lengths, fresh.lengths)
    for a, b in zip(carried.layers.values(), fresh.layers.values()):
        for p, q in zip(a, b):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8)) and (p.dtype == E4M3 or p.abs().max() > 0)


@pytest.mark.parametrize("prompt,seq,capacity", [(12, 20, 32), (16, 16, 32), (300, 200, 500)])
def test_a_captured_chunk_may_fill_its_cache(prompt, seq, capacity):
    """step_graph for chunks of several tokens: the capture itself takes no room, and a replay up to the last token
    of the cache is the chunk launched kernel by kernel."""
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    torch.manual_seed(24)
    model = NeuraTensorModel(config()).to(DEV).to(BF16).eval()
    ids = torch.randint(0, 1000, (2, prompt + seq), device=DEV)
    with torch.no_grad():
        g = model.step_graph(2, seq, ids.device, BF16, cache_tokens=capacity)
        cache = AttentionCache(model.config, 2, capacity + 1, DEV, max_step=seq)
        out = []
        for c in (g.attn_cache, cache):
            _, states, _ = model.forward_device(ids[:, :prompt], attn_cache=c)
            if c is cache:
                out.append(model.forward_device(ids[:, prompt:], states, attn_cache=c)[0])
            else:
                g.load_states(states)
                out.append(g.replay(ids[:, prompt:]).clone())
        assert g.attn_cache.filled == prompt + seq
    assert torch.equal(*out)
    assert g.attn_cache.lengths.tolist() == [prompt + seq] * 2


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,dm", [(1, 128), (8, 640), (64, 2048), (37, 256)])
def test_attention_output_against_definition(dtype, M, dm):
    from neuratensor_b200 import native
    torch.manual_seed(25)
    o, x = (torch.randn(M, dm, device=DEV).to(dtype) for _ in range(2))
    W = (torch.randn(dm, dm, device=DEV) / dm ** 0.5).to(dtype)
    acc = o.double() @ W.double().t()
    terms = o.double().abs() @ W.double().abs().t()
    y = native.attention_output(o, W, x)
    # dm products summed in float32, one rounding to the type, the residual's sum rounded once more
    u = torch.finfo(dtype).eps / 2
    tol = dm * 2.0 ** -24 * terms + u * (acc.abs() + dm * 2.0 ** -24 * terms)
    close(y, acc + x.double(), u, (1 + u) * tol)
    part = native.attention_output(o.view(1, M, dm)[:, :1], W, x.view(1, M, dm)[:, :1])
    assert part.shape == (1, 1, dm)
    for bad in (dict(o=o[:, :64]), dict(x=x.double()), dict(W_o=W[:64])):
        with pytest.raises(ValueError):
            native.attention_output(**{**dict(o=o, W_o=W, x=x), **bad})


def test_a_step_with_memory_calls_no_library_product():
    """Eager and on the device: no matrix product of torch's runs in a layer with a memory."""
    from neuratensor_b200 import AttentionCache
    from neuratensor_b200.core.model import SlidingWindowAttention
    attn = SlidingWindowAttention(128, 2, 40).to(DEV).to(BF16)
    cache = AttentionCache(config(), 2, 60, DEV)
    layer = next(iter(cache.layers))
    with torch.no_grad():
        cache.advance(9)
        attn.forward_cached(torch.randn(2, 9, 128, device=DEV).to(BF16), cache, layer)
        cache.advance(1)
        x = torch.randn(2, 1, 128, device=DEV).to(BF16)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
            attn.forward_cached(x, cache, layer)
    assert not {e.key for e in prof.key_averages()} & {"aten::linear", "aten::matmul", "aten::mm", "aten::addmm", "aten::bmm"}
