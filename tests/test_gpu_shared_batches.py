"""Attention over shared beginnings for more sequences than even shares take (B200): which of its forms a call takes, and what
each computes, against the definition in float64."""
import random

import pytest
import torch

from test_gpu_shared_attention import attention64, close, ints, setup, wide
from test_gpu_step_ops import BF16, DEV, F32, gen, half

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0


def test_which_calls_share(nat):
    """By the workspace, which is that of the attention without sharing where nothing is shared."""
    L = nat.load()

    def shares(B, groups, T=1, G=1, H=8):
        sizes = (B, T, H * G, H, 128, 32, 256, -1)
        return (L.nt_kv_attention_shared_workspace_bytes(1, B, groups, *sizes[1:]) != L.nt_kv_attention_workspace_bytes(*sizes))

    assert shares(512, 256) and shares(512, 128) and shares(512, 64)
    assert not shares(600, 300) and not shares(600, 150)
    assert shares(640, 80) and shares(640, 20) and shares(4096, 512) and not shares(4104, 513)
    assert shares(600, 150, G=16) and not shares(600, 600)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups,K,H,G,longest,tail,window", [
    (70, 8, 2, 1, 1500, 60, None), (65, 9, 1, 3, 300, 200, None), (20, 32, 2, 1, 2000, 30, 1100), (300, 2, 2, 1, 200, 30, None),
    (129, 4, 1, 4, 400, 70, None), (510, 8, 1, 1, 90, 20, None)])
def test_many_sequences(nat, dtype, groups, K, H, G, longest, tail, window):
    P, D = 32, 128
    rng = random.Random(groups + K)
    shared = [rng.choice([rng.randint(0, longest), rng.randint(0, longest) // P * P, 0]) for _ in range(groups)]
    shared[0] = longest
    lengths = [shared[b // K] + rng.randint(0, tail) for b in range(groups * K)]
    counts = [0 if rng.random() < 0.1 or n == 0 else 1 for n in lengths]
    cache, table = setup(groups, K, H, P, D, shared, lengths, 95 + groups)
    table = wide(table, P)
    q = torch.randn(groups * K, 1, H * G, D, device=DEV, generator=gen(96)).to(dtype)
    args = (q, *cache, table, ints(lengths), ints(shared))
    o = nat.kv_attention_shared(*args, counts=ints(counts), window=window)
    want, tol = attention64(q, cache, table, lengths, counts, window, P)
    close(o, want, half(dtype), tol)
    assert torch.equal(o, nat.kv_attention_shared(*args, counts=ints(counts), window=window))
