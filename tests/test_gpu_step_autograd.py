"""The generation-step operators among differentiated ones (B200)."""
import pytest
import torch

from test_gpu_step_ops import BF16, DEV, F32, U32, close, freqs, gen, make_cache, nat, rotary64  # noqa: F401

pytestmark = pytest.mark.gpu


def calls(nat, x):  # noqa: F811
    """One call of each operator that writes what it is given, on x [2, 3, 4, 64] or as many numbers of it."""
    rows = x.view(2, -1)
    tokens = torch.zeros(2, 3, device=DEV, dtype=torch.int64)
    return {"rotary": lambda: nat.rotary(x, torch.arange(3, device=DEV), freqs(64), out=x),
            "rotary into": lambda: nat.rotary(torch.ones_like(x), torch.arange(3, device=DEV), freqs(64), out=x),
            "logits": lambda: nat.logits_process(rows, tokens=tokens, repetition=2.0, out=rows),
            "logits into": lambda: nat.logits_process(torch.ones_like(rows), tokens=tokens, repetition=2.0, out=rows)}


@pytest.mark.parametrize("which", ["rotary", "rotary into", "logits", "logits into"])
def test_a_saved_tensor_that_is_written_is_known(nat, which):  # noqa: F811
    """torch's own in-place operations raise in a backward pass that saved what they wrote; so do these."""
    w = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(60), requires_grad=True)
    x = w * 2
    loss = (x * x).sum()                                     # saves x
    with torch.no_grad():
        calls(nat, x)[which]()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_saved_cache_that_is_written_is_known(nat):  # noqa: F811
    cache, table = make_cache(1, 2, 3, 16, 64, 61)
    w = torch.ones(4, 3, device=DEV, requires_grad=True)
    n = torch.ones(1, device=DEV, dtype=torch.int32)
    k = torch.randn(1, 1, 3, 64, device=DEV, generator=gen(62))
    for i in (1, 3):
        loss = (w * cache[i]).sum()
        versions = [t._version for t in cache]
        nat.kv_append(k, k, *cache, table, n)
        assert all(t._version > v for t, v in zip(cache, versions))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    versions = [t._version for t in cache]
    nat.kv_attention(k, *cache, table, n)
    assert [t._version for t in cache] == versions


@pytest.mark.parametrize("which", ["rotary into", "logits into"])
def test_writing_a_tensor_that_requires_grad_is_refused(nat, which):  # noqa: F811
    x = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(63), requires_grad=True)
    before = x.detach().clone()
    with pytest.raises(RuntimeError, match="requires grad"):
        calls(nat, x)[which]()
    assert torch.equal(x, before)
    with torch.no_grad():
        calls(nat, x)[which]()                               # as torch's own allow it
    assert not torch.equal(x, before)


def test_a_cache_that_requires_grad_is_refused(nat):  # noqa: F811
    cache, table = make_cache(1, 2, 3, 16, 64, 64)
    k, n = torch.ones(1, 1, 3, 64, device=DEV), torch.ones(1, device=DEV, dtype=torch.int32)
    cache[1].requires_grad_()
    with pytest.raises(RuntimeError, match="requires grad"):
        nat.kv_append(k, k, *cache, table, n)


def test_inference_tensors_are_written(nat):  # noqa: F811
    """They have no version; writing them is as before, captured too."""
    with torch.inference_mode():
        x = torch.ones(2, 3, 4, 64, device=DEV)
        for call in calls(nat, x).values():
            call()
        cache, table = make_cache(1, 2, 3, 16, 64, 65)
        k, n = torch.ones(1, 1, 3, 64, device=DEV), torch.ones(1, device=DEV, dtype=torch.int32)
        nat.kv_append(k, k, *cache, table, n)
        assert cache[0][table[0, 0].long(), :, 0].float().eq(256).all()          # 1 / 2^-8
