"""A beam search of a model that is not on a GPU: refused like sampling, whatever is asked for."""
import pytest
import torch

from neuratensor_b200 import ModelConfig, NeuraTensorModel


@pytest.mark.parametrize("more", [dict(), dict(use_graph=False), dict(attn_cache=True), dict(max_new_tokens=1), dict(num_beams=1)])
def test_generate_on_the_cpu_says_that_it_runs_on_cuda(more):
    model = NeuraTensorModel(ModelConfig(vocab_size=70, d_model=128, n_layers=2, d_state=16, max_seq_len=64, attn_every=2,
                                         attn_heads=2, attn_window=8))
    with pytest.raises(RuntimeError, match="on CUDA"):
        model.generate(torch.zeros(2, 3, dtype=torch.int64), **{**dict(max_new_tokens=2, num_beams=2), **more})
