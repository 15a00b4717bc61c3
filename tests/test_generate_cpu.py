"""What the model keeps between calls of generate, without a GPU."""
import copy

import pytest
import torch


def config(**kw):
    from neuratensor_b200 import ModelConfig
    return ModelConfig(**{**dict(vocab_size=70, d_model=128, n_layers=4, d_state=16, max_seq_len=64, attn_every=2,
                                 attn_heads=2, attn_window=8), **kw})


@pytest.mark.parametrize("how", ["replaced", "written"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tables_follow_the_frequencies(how, dtype):
    from neuratensor_b200 import RotaryEmbedding
    rope, x = RotaryEmbedding(64), torch.zeros(1, 9, 64, dtype=dtype)
    before = rope(x)[0]
    assert rope(x)[0].data_ptr() == before.data_ptr()               # kept as long as nothing changes
    f = rope.inv_freq / 8
    if how == "replaced":
        rope.inv_freq = f
    else:
        rope.inv_freq.copy_(f)
    cos, sin = rope(x)
    ang = torch.outer(torch.arange(9.0), f).repeat(1, 2)
    assert torch.equal(cos, ang.cos().to(dtype)) and torch.equal(sin, ang.sin().to(dtype))
    assert rope(x)[0].data_ptr() == cos.data_ptr()


def test_moved_and_copied_tables_stay():
    """A cast or a copy of the module takes its tables along, as it does for the reference's."""
    from neuratensor_b200 import RotaryEmbedding
    rope, x = RotaryEmbedding(64), torch.zeros(1, 9, 64, dtype=torch.bfloat16)
    table = rope(x.float())[0]
    other = copy.deepcopy(rope)
    assert torch.equal(other(x.float())[0], table)
    rope = rope.to(torch.bfloat16)
    assert torch.equal(rope(x)[0], table.to(torch.bfloat16))
    rope.inv_freq.mul_(0.5)
    assert not torch.equal(rope(x)[0], table.to(torch.bfloat16))


def test_a_captured_step_is_told_of_new_frequencies():
    """A captured step holds the frequencies that it was captured with; only one without a cache reads the tables."""
    from neuratensor_b200 import NeuraTensorModel
    from neuratensor_b200.core.rotary import Seen
    from neuratensor_b200.inference.decode import StepGraph
    model = NeuraTensorModel(config()).to(torch.bfloat16)
    step = object.__new__(StepGraph)                                # as one is behind its capture
    step.model, step.frequencies = model, [Seen(a.rope.inv_freq) for a in model.attn_layers.values()]
    rope = list(model.attn_layers.values())[-1].rope
    for T in (9, 20):                                               # tables, and longer ones
        with_cache, without = model._graph_signature(1024), model._graph_signature(0)
        rope(torch.zeros(1, T, 64, dtype=torch.bfloat16))
        assert model._graph_signature(1024) == with_cache and model._graph_signature(0) != without
        assert step.frequencies_hold()
    for change in (lambda: rope.inv_freq.mul_(0.5), lambda: setattr(rope, "inv_freq", rope.inv_freq.clone())):
        change()
        assert not step.frequencies_hold()
        step.frequencies = [Seen(a.rope.inv_freq) for a in model.attn_layers.values()]
        assert step.frequencies_hold()


def test_a_copied_model_does_not_go_by_the_original_buffers():
    """What a copy keeps of its frequencies is its own: no later tensor can pass for the original's."""
    from neuratensor_b200 import RotaryEmbedding
    rope, x = RotaryEmbedding(64), torch.zeros(1, 9, 64)
    rope(x)
    other = copy.deepcopy(rope)
    assert other._made_from.tensor is other.inv_freq and other._made_from.tensor is not rope.inv_freq
    f = rope.inv_freq / 3
    other.inv_freq = f
    assert torch.equal(other(x)[0][1], torch.cat([f, f]).cos())


def test_generate_refuses_a_cache_without_room():
    """Before anything runs, and the cache stays where it was."""
    from neuratensor_b200 import AttentionCache, NeuraTensorModel
    model = NeuraTensorModel(config())
    cache = AttentionCache(model.config, 2, 32, "cpu", page=16)
    cache.filled = 20
    ids = torch.zeros(2, 3, dtype=torch.int64)
    for kw in (dict(max_new_tokens=10), dict(max_new_tokens=1000), dict(input_ids=torch.zeros(2, 13, dtype=torch.int64), stop_tokens=[1])):
        with pytest.raises(ValueError, match="do not fit"):
            model.generate(**{**dict(input_ids=ids, attn_cache=cache), **kw})
    with pytest.raises(ValueError, match="for 2 sequences"):
        model.generate(ids[:1], max_new_tokens=1, attn_cache=cache)
    for kw in (dict(max_new_tokens=9), dict(max_new_tokens=1000, stop_tokens=[1]),        # 20 + 3 + 9 = 32; ends where it stops
               dict(input_ids=torch.zeros(2, 100, dtype=torch.int64), max_new_tokens=1)):
        with pytest.raises((RuntimeError, ValueError)) as e:                              # no GPU here, or 64 of 100 tokens that do not fit
            model.generate(**{**dict(input_ids=ids, attn_cache=cache), **kw})
        assert ("CUDA" in str(e.value)) == ("input_ids" not in kw)
        cache.filled, cache.lengths = 20, cache.lengths * 0


def test_attention_output_status():
    """Statuses and messages of the entry point that need no GPU."""
    import ctypes

    from neuratensor_b200 import build, native
    build.build()
    L, X = native.load(), ctypes.c_void_p(4096)

    def call(dtype=1, M=2, dm=64, o=X, W=X, x=X, out=X):
        return L.nt_attention_output(dtype, M, dm, o, W, x, out, None), L.nt_last_error().decode()

    assert call(M=0, o=None)[0] == 0
    for bad, status, text in ((dict(dtype=2), 2, "dtype"), (dict(M=-1), 1, "sizes"), (dict(dm=0), 1, "sizes"),
                              (dict(o=None), 1, "null"), (dict(W=None), 1, "null"), (dict(x=None), 1, "null"),
                              (dict(out=None), 1, "null"), (dict(dm=60), 1, "multiple of 8"),
                              (dict(o=ctypes.c_void_p(4104)), 1, "alignment")):
        rc, said = call(**bad)
        assert rc == status and text in said
    with pytest.raises(RuntimeError, match="CUDA"):
        native.attention_output(*[torch.zeros(64, 64)] * 3)
