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


def large_cache(B, blocks, H, P, D, seed, code):
    """Random finite codes, keys of about one, values of up to `code` times the pages' scales of 1."""
    cache, table = make_cache(B, blocks, H, P, D, seed)
    g = gen(seed + 1)
    cache[0].copy_(torch.randn(cache[0].shape, device=DEV, generator=g).to(E4M3))
    cache[2].copy_((code * (2 * torch.rand(cache[2].shape, device=DEV, generator=g) - 1)).to(E4M3))
    cache[1].fill_(1.0)
    cache[3].fill_(1.0)
    return cache, table


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,G,D,P,lengths,window", [
    (1, 1, 10, 1, 64, 16, [257], 256),                    # one CTA a head
    (2, 1, 8, 4, 128, 64, [5000, 300], None),             # even shares
    (2, 2, 3, 8, 64, 32, [2900, 1500], None)])            # chunks of row tiles
def test_attention_over_the_largest_values(nat, dtype, B, T, H, G, D, P, lengths, window):  # noqa: F811
    """The mean of values of up to 448 * 2^119, the last scale whose codes are all finite, is finite: every sum of
    them on the way must be, too."""
    cache, table = large_cache(B, -(-max(lengths) // P), H, P, D, 80, 448)
    q = torch.randn(B, T, H * G, D, device=DEV, generator=gen(82)).to(dtype)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    plain = nat.kv_attention(q, *cache, table, n, window=window)
    want, tol = attention64(q, cache, table, lengths, [T] * B, window, P)
    close(plain, want, half(dtype), tol)
    for e in (100, 119):
        cache[3].fill_(2.0 ** e)
        o = nat.kv_attention(q, *cache, table, n, window=window)
        assert torch.equal(o.double(), plain.double() * 2.0 ** e)      # a power of two on every value is one on the result


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("e", [-80, -100, -112, -120])
def test_attention_of_the_smallest_queries(nat, dtype, e):  # noqa: F811
    """Queries of 2^e with a scale of 2^-e have the scores of ordinary ones: a power of two on the query and its
    inverse on the scale change no rounding while every number is normal."""
    B, T, H, G, D, P, lengths = 2, 2, 2, 2, 64, 16, [100, 33]
    cache, table = large_cache(B, 7, H, P, D, 85, 1)
    q = torch.randn(B, T, H * G, D, device=DEV, generator=gen(86))
    q = (torch.where(q.abs() < 2.0 ** -5, torch.zeros_like(q), q)).to(dtype)          # 2^-125 and above, or zero
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    want, tol = attention64(q, cache, table, lengths, [T] * B, None, P, scale=0.25)
    plain = nat.kv_attention(q, *cache, table, n, scale=0.25)
    close(plain, want, half(dtype), tol)
    o = nat.kv_attention((q.double() * 2.0 ** e).to(dtype), *cache, table, n, scale=0.25 * 2.0 ** -e)
    # q is split into f16 as before or, below 2^-113, from 2^7 on instead of 2^13: f16 still ends at 2^-31 of its largest
    close(o, want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_subnormal_queries(nat, dtype):  # noqa: F811
    B, T, H, G, D, P, lengths = 1, 1, 4, 1, 64, 16, [50]
    cache, table = large_cache(B, 4, H, P, D, 87, 1)
    q = (torch.randint(-100, 100, (B, T, H, D), device=DEV, generator=gen(88)).double() * 2.0 ** -133).to(dtype)
    assert q.abs().max() > 0
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    want, tol = attention64(q, cache, table, lengths, [T], None, P, scale=2.0 ** 124)
    close(nat.kv_attention(q, *cache, table, n, scale=2.0 ** 124), want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,G,D,P,low,high,window", [
    (3, 1, 2, 16, 64, 16, 100, 1500, None), (520, 1, 1, 1, 64, 16, 1, 1500, None), (150, 1, 2, 1, 64, 32, 900, 1500, 1000),
    (2, 1, 3, 1, 128, 64, 1200, 1500, 1300), (3, 9, 2, 2, 64, 32, 60, 1500, None)])
def test_attention_in_chunks_of_every_sequence_and_head(nat, dtype, B, T, H, G, D, P, low, high, window):  # noqa: F811
    """Spans over several chunks, whose partial rows lie apart by sequence, head and row tile
    (test_step_chunks_cpu.py checks that these sizes are split)."""
    g = gen(90)
    lengths = torch.randint(low, high + 1, (B,), device=DEV, generator=g)
    lengths[-1] = high
    cache, table = large_cache(B, -(-high // P), H, P, D, 91, 1)
    scale = 2.0 ** torch.randint(-2, 3, cache[1].shape, device=DEV, generator=g).float()
    cache[1].copy_(scale / 4)
    cache[3].copy_(scale)
    q = torch.randn(B, T, H * G, D, device=DEV, generator=g).to(dtype)
    o = nat.kv_attention(q, *cache, table, lengths, window=window)
    n = lengths.tolist()
    want, tol = attention64(q, cache, table, n, [min(T, x) for x in n], window, P)
    close(o, want, half(dtype), tol)
    again = nat.kv_attention(q, *cache, table, lengths, window=window)
    assert torch.equal(o, again)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,G", [(3, 1), (2, 2), (1, 4), (6, 1), (3, 2), (5, 3)])
@pytest.mark.parametrize("window", [20, None])
def test_a_nan_reaches_the_rows_that_see_it(nat, dtype, T, G, window):  # noqa: F811
    """With the second halves of the weights in columns of their own (four rows or fewer) and as a second product;
    over pages whose scales are 2^60 apart, which take a product of their own, too."""
    P, D, H, n = 16, 64, 2, 100
    for spread in (0, 60):
        cache, table = large_cache(1, 7, H, P, D, 95, 1)
        q = torch.randn(1, T, H * G, D, device=DEV, generator=gen(96)).to(dtype)
        if spread:
            cache[3][table[0, ::2].long()] = 2.0 ** -spread
        lengths = torch.tensor([n], device=DEV, dtype=torch.int32)
        want, tol = attention64(q, cache, table, [n], [T], window, P)
        close(nat.kv_attention(q, *cache, table, lengths, window=window), want, half(dtype), tol)
        for key in (99, 98, 97, 96, 81, 79, 78, 77, 40):
            page, slot = int(table[0, key // P]), key % P
            for side in (0, 2):
                codes = cache[side].view(torch.uint8)
                kept = codes[page, 0, slot].clone()
                codes[page, 0, slot, 7] = 0x7f                       # one NaN, of head 0
                o = nat.kv_attention(q, *cache, table, lengths, window=window)
                codes[page, 0, slot] = kept
                for t in range(T):
                    p = n - T + t
                    sees = key <= p and (window is None or key >= p - window)
                    bad = torch.zeros(H * G, D, dtype=torch.bool, device=DEV)
                    if sees:
                        bad[:G, 7 if side else slice(None)] = True
                    assert torch.equal(o[0, t].isnan(), bad)
                    close(o[0, t][~bad], want[0, t][~bad], half(dtype), tol[0, t][~bad])
