"""Generation with and without torch.inference_mode on one model (B200): a step captured in either serves both."""
import contextlib

import pytest
import torch

from test_gpu_beam_search import DEV, make

pytestmark = pytest.mark.gpu

KINDS = {"beams": dict(num_beams=3, stop_tokens=[3, 9]), "beams with a memory": dict(num_beams=2, attn_cache=True),
         "uncaptured beams": dict(num_beams=3, attn_cache=True, use_graph=False), "sampling": dict(top_k=1),
         "sampling with a memory": dict(top_k=1, attn_cache=True)}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("first", [True, False])
def test_calls_in_inference_mode_and_out_of_it(kind, first):
    model = make(torch.bfloat16)
    ids = torch.randint(0, 211, (2, 9), device=DEV, generator=torch.Generator(device=DEV).manual_seed(41))
    outs, states = [], []
    for inference in (first, not first, first, not first):
        with torch.inference_mode() if inference else contextlib.nullcontext():
            torch.manual_seed(1)
            out, st = model.generate(ids, max_new_tokens=7, **KINDS[kind])
            outs.append(out)
            states.append(st)
    assert all(torch.equal(outs[0], o) for o in outs)
    for st in states:
        assert all(torch.equal(a.membrane, b.membrane) and torch.equal(a.ssm_state, b.ssm_state) for a, b in zip(states[0], st))
    # and states of one kind of call go on in the other
    for inference, st in ((True, states[0]), (False, states[1]), (True, states[1]), (False, states[0])):
        with torch.inference_mode() if inference else contextlib.nullcontext():
            torch.manual_seed(2)
            outs.append(model.generate(ids, max_new_tokens=5, states=st, **KINDS[kind])[0])
    assert all(torch.equal(outs[4], o) for o in outs[4:])
