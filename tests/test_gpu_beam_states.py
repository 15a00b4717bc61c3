"""The states that a beam search leaves (B200): of a beam that ended, those ahead of its stop token."""
import pytest
import torch

from test_gpu_beam_search import DEV, make

pytestmark = pytest.mark.gpu

STOP = list(range(25))


def prompts():
    return torch.randint(0, 211, (6, 9), device=DEV, generator=torch.Generator(device=DEV).manual_seed(31))


def run(model, ids, new, **more):
    """The best beams' tokens, their states, and where each ended."""
    out, states = model.generate(ids, max_new_tokens=new, num_beams=3, length_penalty=1.0, stop_tokens=STOP, **more)
    tokens = out[:, ids.shape[1]:]
    ends = [next(i for i, t in enumerate(row) if t in STOP) for row in tokens.tolist()]
    return tokens, [t for s in states for t in (s.membrane, s.ssm_state)], ends


@pytest.mark.parametrize("dtype,cache", [(torch.float32, False), (torch.bfloat16, True)])
def test_states_do_not_depend_on_what_follows(dtype, cache):
    """How many pads follow, and whether the steps are captured."""
    model = make(dtype, window=16)
    runs = [run(model, prompts(), new, attn_cache=cache, use_graph=graph) for new in (40, 45, 61) for graph in (True, False)]
    tokens, states, ends = runs[0]
    assert len(set(ends)) > 2 and max(ends) < 30          # at different steps, long before the last
    for t, s, e in runs[1:]:
        assert torch.equal(t[:, :40], tokens) and (t[:, 40:] == 0).all()
        assert all(torch.equal(a, b) for a, b in zip(states, s))


@pytest.mark.parametrize("attn,cache", [(False, False), (True, False), (True, True)])
def test_states_do_not_depend_on_when_the_others_end(attn, cache):
    """Nor on when the host looks whether all have ended: a prompt among others and alone."""
    model = make(torch.float32, attn=attn, window=16)
    ids = prompts()
    tokens, states, ends = run(model, ids, 40, attn_cache=cache)
    assert len(set(ends)) > 2
    for p in range(6):
        t, s, _ = run(model, ids[p:p + 1], 40, attn_cache=cache)
        assert torch.equal(t[0], tokens[p])
        # eighteen rows and three: float32 sums in another order
        assert all(torch.allclose(a[0], b[p], rtol=1e-4, atol=1e-5) for a, b in zip(s, states))


def test_states_of_ended_beams_are_those_ahead_of_the_stop_token():
    model = make(torch.float32, attn=False)
    ids = prompts()
    tokens, states, ends = run(model, ids, 40)
    assert len(set(ends)) > 2
    for p, end in enumerate(ends):
        with torch.no_grad():
            _, st, _ = model.forward_device(ids[p:p + 1], None)
            for t in tokens[p, :end].tolist():
                _, st, _ = model.forward_device(torch.tensor([[t]], device=DEV), st)
        for a, b in zip([t for s in st for t in (s.membrane, s.ssm_state)], states):
            # eighteen rows and one row alone: float32 sums in another order
            assert torch.allclose(a[0], b[p], rtol=1e-4, atol=1e-5)


def test_a_first_token_that_stops_leaves_the_prompts_states():
    model = make(torch.float32, attn=False)
    ids = prompts()
    out, states = model.generate(ids, max_new_tokens=20, num_beams=3, stop_tokens=list(range(211)))
    assert (out[:, 10:] == 0).all()
    with torch.no_grad():
        _, want, _ = model.forward_device(ids, None)
    for a, b in zip(want, states):
        assert torch.equal(a.membrane, b.membrane) and torch.equal(a.ssm_state, b.ssm_state)


def test_the_engine_goes_on_from_them():
    """A second call that carries the states on gives a prompt what it gives when the prompt has run alone."""
    from neuratensor_b200 import InferenceEngine
    engine = InferenceEngine(make(torch.float32, attn=False), dtype=torch.float32)
    first, then = prompts(), prompts()[:, :4].flip(0)
    how = dict(num_beams=3, length_penalty=1.0, stop_tokens=STOP)
    engine.generate(first, max_new_tokens=40, **how)
    both = engine.generate(then, max_new_tokens=6, num_beams=3, reset_state=False)
    for p in range(6):
        engine.generate(first[p:p + 1], max_new_tokens=40, **how)
        assert torch.equal(both[p:p + 1], engine.generate(then[p:p + 1], max_new_tokens=6, num_beams=3, reset_state=False))
