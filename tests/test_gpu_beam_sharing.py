"""Beam search whose attention reads what the beams share once (B200): windows and batches long enough for it.

In a window of up to a thousand keys every beam reads its own, which is faster; the tests of the search itself stay
below that."""
import pytest
import torch

from neuratensor_b200 import ModelConfig, NeuraTensorModel
from neuratensor_b200.core.cache import BeamCache
from test_gpu_beam_search import search
from test_gpu_step_ops import BF16, DEV, F32, attention64, close, half

pytestmark = pytest.mark.gpu

WINDOW = 1200


def make(dtype, heads=2):
    torch.manual_seed(0)
    model = NeuraTensorModel(ModelConfig(vocab_size=211, d_model=64 * heads, n_layers=2, d_state=16, max_seq_len=2048, tie_weights=False,
                                         attn_every=2, attn_heads=heads, attn_window=WINDOW))
    with torch.no_grad():
        model.embedding.weight.mul_(60)
        model.lm_head.weight.copy_(0.2 * torch.randn(211, 64 * heads))
    return model.to(DEV).to(dtype).eval()


def prompts(P, T):
    return torch.randint(0, 211, (P, T), device=DEV, generator=torch.Generator(device=DEV).manual_seed(T))


# eight rows a prompt, taken together with the rests in one kernel, and forty, on tcgen05
@pytest.mark.parametrize("P,K", [(8, 8), (2, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1150, 1290])
def test_attention_of_every_step_against_its_definition(monkeypatch, dtype, P, K, T):
    from neuratensor_b200 import native
    native.device_error_flags(0)
    L, attend, seen = native.load(), BeamCache.attend, []

    def checked(self, layer, q, lengths):
        o = attend(self, layer, q, lengths)
        B, _, H, D = q.shape
        blocks, code = self.table.shape[1], 0 if q.dtype == F32 else 1
        # it is one that shares, by its workspace, over what all beams have of the prompt
        assert L.nt_kv_attention_shared_workspace_bytes(code, B, P, 1, H, H, D, self.page, blocks, self.window) != \
            L.nt_kv_attention_workspace_bytes(B, 1, H, H, D, self.page, blocks, self.window)
        seen.append(self.shared.tolist())
        want, tol = attention64(q, self.layers[layer], self.table, lengths, [1] * B, self.window, self.page)
        close(o, want, half(q.dtype), tol)
        return o

    monkeypatch.setattr(BeamCache, "attend", checked)
    out, _ = make(dtype).generate(prompts(P, T), max_new_tokens=5, num_beams=K, attn_cache=True, use_graph=False)
    assert out.shape == (P, T + 5) and len(seen) == 4
    assert all(s >= T // 32 * 32 for shared in seen for s in shared)
    assert native.device_error_flags(0) == 0


@pytest.mark.parametrize("P,K,T", [(8, 8, 1150), (2, 40, 1290)])
def test_search_is_the_search_from_scratch(P, K, T):
    model = make(F32)
    ids = prompts(P, T)
    want, _ = search(model, ids, 5, K, 0.6, [3, 9], True)
    for graph in (True, False, True):
        out, _ = model.generate(ids, max_new_tokens=5, num_beams=K, length_penalty=0.6, stop_tokens=[3, 9], attn_cache=True, use_graph=graph)
        assert torch.equal(out[:, T:], want), graph


@pytest.mark.parametrize("P,K", [(8, 8), (2, 40)])
def test_captured_steps_share_as_uncaptured_ones_do(P, K):
    model = make(BF16)
    ids = prompts(P, 1180)
    outs = [model.generate(ids, max_new_tokens=40, num_beams=K, attn_cache=True, use_graph=graph) for graph in (True, False)]
    assert torch.equal(outs[0][0], outs[1][0])
    for a, b in zip(outs[0][1], outs[1][1]):
        assert torch.equal(a.membrane, b.membrane) and torch.equal(a.ssm_state, b.ssm_state)
