"""Beam search through ``generate`` (B200): against a search written out here that runs every beam from scratch."""
import gc
import weakref

import pytest
import torch

from neuratensor_b200 import ModelConfig, NeuraTensorModel
from neuratensor_b200.core.cache import AttentionCache, BeamCache

pytestmark = pytest.mark.gpu

DEV = "cuda"


def make(dtype, vocab=211, attn=True, window=8, seed=0, layers=4, tied=False):
    """Tied, the likeliest token is the last one again; with weights of its own for the logits every step is a choice."""
    torch.manual_seed(seed)
    model = NeuraTensorModel(ModelConfig(vocab_size=vocab, d_model=128, n_layers=layers, d_state=16, max_seq_len=256, tie_weights=tied,
                                         attn_every=2 if attn else 0, attn_heads=2, attn_window=window))
    with torch.no_grad():
        model.embedding.weight.mul_(60)                 # logits that tell tokens apart
        if not tied:
            model.lm_head.weight.copy_(0.2 * torch.randn(vocab, 128))
    return model.to(DEV).to(dtype).eval()


@torch.no_grad()
def search(model, ids, new, K, alpha, stop, cache):
    """(tokens, sums) of the best beams: every step runs all beams from their prompts on; sums in float64.

    A beam stays in its place where it goes on, since the blocks' choice of their sparse path looks at all rows of a call."""
    P, T = ids.shape
    pad = stop[0] if stop else 0

    def last_logits(rows):                              # rows: token lists behind the prompts, all of one length
        R = len(rows)
        if not rows[0]:
            return model.forward_device(ids, None, last_only=True)[0][:, -1].double()
        c = AttentionCache(model.config, P, T + new + 1, DEV, max_step=1) if cache else None
        _, states, _ = model.forward_device(ids, None, last_only=True, attn_cache=c)
        K = R // P
        if cache:                                       # the prompts' memory for every beam
            wide = AttentionCache(model.config, R, T + new + 1, DEV, max_step=1)
            for name, layer in c.layers.items():
                for a, b in zip(layer, wide.layers[name]):
                    a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
                    b.view(P, K, c.ring, *a.shape[1:]).copy_(a.view(P, 1, c.ring, *a.shape[1:]))
            wide.lengths += T
            wide.filled = T
            c = wide
        st = [type(s)(membrane=s.membrane.repeat_interleave(K, 0), ssm_state=s.ssm_state.repeat_interleave(K, 0)) for s in states]
        for i in range(len(rows[0])):
            tok = torch.tensor([[r[i]] for r in rows], device=DEV)
            logits, st, _ = model.forward_device(tok, st, attn_cache=c)
        return logits[:, -1].double()

    def cands(logits, beam, sums, beams, done, lens):
        out = []
        p = torch.log_softmax(logits, -1)
        for k in range(beams):
            if done[k]:
                out.append((sums[k] / max(lens[k], 1) ** alpha, k, pad, sums[k]))
                continue
            v, i = torch.sort(p[beam + k], descending=True, stable=True)
            out += [((sums[k] + a) / (lens[k] + 1) ** alpha, k, t, sums[k] + a) for a, t in zip(v[:K].tolist(), i[:K].tolist())]
        return sorted(out, key=lambda c: (-c[0], c[1]))[:K]

    first = last_logits([[]])
    rows, sums, done, lens = [], [], [], []
    for p in range(P):
        for _, _, t, s in cands(first, p, [0.0], 1, [False], [0]):
            rows.append([t])
            sums.append(float(torch.tensor(s, dtype=torch.float32)))
            done.append(t in stop)
            lens.append(1)
    for _ in range(1, new):
        logits = last_logits(rows)
        nr, ns, nd, nl = ([None] * (P * K) for _ in range(4))
        for p in range(P):
            a = p * K
            left = []
            for _, k, t, s in cands(logits, a, sums[a:a + K], K, done[a:a + K], lens[a:a + K]):
                new_beam = (rows[a + k] + [t], float(torch.tensor(s, dtype=torch.float32)), done[a + k] or t in stop,
                            lens[a + k] + (not done[a + k]))
                if nr[a + k] is None:
                    nr[a + k], ns[a + k], nd[a + k], nl[a + k] = new_beam
                else:
                    left.append(new_beam)
            for r in range(a, a + K):
                if nr[r] is None:
                    nr[r], ns[r], nd[r], nl[r] = left.pop(0)
        rows, sums, done, lens = nr, ns, nd, nl
    best = [max(range(p * K, p * K + K), key=lambda r: (sums[r] / max(lens[r], 1) ** alpha, -r)) for p in range(P)]
    return torch.tensor([rows[b] for b in best], device=DEV), [sums[b] for b in best]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P,T,new,K,alpha,stops,cache,window", [
    (1, 1, 1, 2, 0.0, 0, False, 8), (2, 5, 9, 3, 0.0, 0, False, 8), (3, 20, 8, 4, 0.7, 3, True, 8), (2, 40, 10, 5, 1.0, 40, True, 16),
    (1, 33, 12, 2, 0.0, 0, True, 3), (2, 7, 20, 4, 0.5, 25, True, 64)])
@pytest.mark.parametrize("tied", [False, True])
def test_search_is_the_search_from_scratch(dtype, P, T, new, K, alpha, stops, cache, window, tied):
    model = make(dtype, window=window, tied=tied)
    g = torch.Generator(device=DEV).manual_seed(T)
    ids = torch.randint(0, 211, (P, T), device=DEV, generator=g)
    stop = list(range(5, 5 + stops))
    want, _ = search(model, ids, new, K, alpha, stop, cache)
    for graph in (True, False, True):
        out, states = model.generate(ids, max_new_tokens=new, num_beams=K, length_penalty=alpha, stop_tokens=stop or None,
                                     attn_cache=cache, use_graph=graph)
        assert torch.equal(out[:, :T], ids)
        assert torch.equal(out[:, T:], want), graph
        assert len(states) == 4 and states[0].membrane.shape == (P, 256)
    from neuratensor_b200 import native
    assert native.device_error_flags(0) == 0


def test_states_continue_the_best_beam():
    """The states returned are those behind the best beam's tokens but the last."""
    model = make(torch.float32, attn=False)
    ids = torch.randint(0, 211, (1, 6), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    out, states = model.generate(ids, max_new_tokens=5, num_beams=3)
    with torch.no_grad():
        _, st, _ = model.forward_device(ids, None)
        for i in range(6, out.shape[1] - 1):
            _, st, _ = model.forward_device(out[:, i:i + 1], st)
    for a, b in zip(st, states):
        # a beam of three rows and one row alone: float32 sums in another order
        assert torch.allclose(a.membrane, b.membrane, rtol=1e-4, atol=1e-5) and torch.allclose(a.ssm_state, b.ssm_state, rtol=1e-4, atol=1e-5)


def test_a_captured_step_follows_the_weights():
    model = make(torch.bfloat16)
    ids = torch.randint(0, 211, (2, 9), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    a, _ = model.generate(ids, max_new_tokens=6, num_beams=3, attn_cache=True)
    with torch.no_grad():
        model.embedding.weight.copy_(model.embedding.weight.flip(0))
        model.attn_layers["1"].rope.inv_freq.mul_(0.5)
    b, _ = model.generate(ids, max_new_tokens=6, num_beams=3, attn_cache=True)
    c, _ = model.generate(ids, max_new_tokens=6, num_beams=3, attn_cache=True, use_graph=False)
    assert torch.equal(b, c) and not torch.equal(a, b)
    engine_out, _ = model.generate(ids.repeat(2, 1), max_new_tokens=6, num_beams=2, attn_cache=True)
    assert engine_out.shape == (4, 15)


@pytest.mark.parametrize("T,window,steps", [(70, 40, 60), (5, 1000, 40)])
def test_memory_of_a_search_counts_its_pages(T, window, steps):
    """Pages in use are those of the tables, none is lost over many forks, and no more than the window needs."""
    model = make(torch.bfloat16, window=window)
    P, K = 2, 5
    cache = BeamCache(model.config, P, K, T + steps + 2, DEV, page=16)
    g = torch.Generator(device=DEV).manual_seed(3)
    cache.begin(T)
    with torch.no_grad():
        _, states, _ = model.forward_device(torch.randint(0, 211, (P, T), device=DEV, generator=g), None, last_only=True,
                                            attn_cache=cache.prompt_rows())
        cache.filled = T
        states = [type(s)(membrane=s.membrane.repeat_interleave(K, 0), ssm_state=s.ssm_state.repeat_interleave(K, 0)) for s in states]
        rows = torch.arange(P * K, device=DEV, dtype=torch.int32) // K * K
        for _ in range(steps):
            cache.fork(rows)
            used = torch.bincount(cache.table[cache.table >= 0].long(), minlength=cache.refs.numel())
            assert torch.equal(used.int(), cache.refs)
            logits, states, _ = model.forward_device(torch.randint(0, 211, (P * K, 1), device=DEV, generator=g), states, attn_cache=cache)
            assert logits.isfinite().all()
            rows = (torch.randint(0, K, (P, K), device=DEV, generator=g) + K * torch.arange(P, device=DEV)[:, None]).view(-1).int()
    from neuratensor_b200 import native
    assert native.device_error_flags(0) == 0
    assert (cache.table >= 0).sum(1).max() <= window // 16 + 2 and cache.lengths.tolist() == [T + steps] * (P * K)


def test_through_the_engine():
    from neuratensor_b200 import InferenceEngine
    model = make(torch.bfloat16)
    engine = InferenceEngine(model, dtype=torch.bfloat16)
    ids = torch.randint(0, 211, (2, 11), generator=torch.Generator().manual_seed(4))
    out = engine.generate(ids, max_new_tokens=7, num_beams=4, length_penalty=0.6, stop_tokens=[3, 9], attn_cache=True)
    want, _ = model.generate(ids.to(DEV), max_new_tokens=7, num_beams=4, length_penalty=0.6, stop_tokens=[3, 9], attn_cache=True)
    assert torch.equal(out, want) and out.shape == (2, 18)
    sampled = engine.generate(ids, max_new_tokens=7, top_k=1, attn_cache=True)          # and sampling goes on beside it
    assert sampled.shape == (2, 18)
    with pytest.raises(ValueError, match="AttentionCache"):
        engine.generate(ids, max_new_tokens=3, num_beams=2, attn_cache=AttentionCache(model.config, 2, 64, DEV))


def test_models_and_their_captured_steps_go_together_and_captures_bear_collections():
    """A step does not keep its model, so both go without the garbage collector; and one that destroys another graph does
    not come in a capture."""
    ids = torch.zeros(1, 4, dtype=torch.int64, device=DEV)
    for capture in (lambda m: m.generate(ids, max_new_tokens=3, num_beams=2, attn_cache=True),
                    lambda m: m.generate(ids, max_new_tokens=3, top_k=1, attn_cache=True)):
        old = gc.get_threshold()
        gc.disable()
        try:
            dead = make(torch.bfloat16)
            capture(dead)
            gone = weakref.ref(dead)
            cycle = [list(dead.__dict__.get("_beam_steps", {}).values()) + list(dead.__dict__.get("_step_graphs", {}).values())]
            del dead
            assert gone() is None
            cycle.append(cycle)                         # its graphs are left to the collector
            del cycle
            live = make(torch.bfloat16)
            gc.set_threshold(1, 1, 1)                   # from here on every allocation may collect
            gc.enable()
            capture(live)
        finally:
            gc.set_threshold(*old)
            gc.enable()


def test_a_captured_step_outlives_its_model():
    """A step that is kept while its model goes reads the weights that it was captured with."""
    model = make(torch.bfloat16)
    tok = torch.full((2, 1), 7, dtype=torch.int64, device=DEV)
    graph = model.decode_graph(2, torch.device(DEV), torch.bfloat16)
    graph.load_states(None)                             # capturing leaves the states where its own steps took them
    want = graph.step(tok).clone()
    del model
    gc.collect()
    junk = [torch.full((1 << 16,), 1e4, device=DEV) for _ in range(64)]                 # what was freed is written over
    graph.load_states(None)
    assert torch.equal(graph.step(tok), want) and len(graph.states()) == 4
    del junk
