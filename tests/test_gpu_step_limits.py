"""The generation-step operators at the ends of their ranges (B200)."""
import math

import pytest
import torch

from test_gpu_step_ops import BF16, DEV, E4M3, F32, U32, attention64, close, gen, half, make_cache, nat  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,G,D,P,lengths,window", [
    (1, 1, 64, 16, [2, 3, 4, 6, 300], 3), (1, 1, 128, 32, [2, 3, 5, 8, 40], None), (1, 4, 128, 64, [3000, 2, 900], 2),
    (4, 2, 64, 16, [5, 7, 333, 40], 4)])
def test_bf16_attention_is_float32_rounded_once(nat, T, G, D, P, lengths, window):  # noqa: F811
    """Every output lies between the roundings of what float32 arithmetic may give: with few keys and a
    score of one product that is one number, or two neighbours.  Weights of 11 bits fall outside."""
    B, H = len(lengths), 10
    cache, table = make_cache(B, -(-max(lengths) // P), H, P, D, 70)
    g = gen(71)
    for c, s in ((cache[0], cache[1]), (cache[2], cache[3])):
        c.copy_(torch.randn(c.shape, device=DEV, generator=g).to(E4M3))
        s.fill_(1.0)
    q = torch.zeros(B, T, H * G, D, device=DEV)
    q[..., 5] = 1 + torch.rand(B, T, H * G, device=DEV, generator=g)
    q = q.to(BF16)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    o = nat.kv_attention(q, *cache, table, n, window=window, scale=0.5).double()
    want, tol = attention64(q.float(), cache, table, lengths, [T] * B, window, P, scale=0.5)     # the bound of float32
    low, high = (want - tol).to(BF16).double(), (want + tol).to(BF16).double()
    assert ((o >= low) & (o <= high)).all(), f"{((o < low) | (o > high)).double().mean().item():.2g} of the outputs are outside"
