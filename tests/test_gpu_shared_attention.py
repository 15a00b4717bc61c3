"""Attention over caches whose sequences share their beginnings (B200), against its definition in float64.

The tolerances are those of the attention over a cache without sharing: half a step of the output
type, and what float32 scores, weights and sums leave (``attention64``).
"""
import random

import pytest
import torch

from test_gpu_step_ops import BF16, DEV, E4M3, F32, U32, attention64, close, fill, gen, half, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0      # every test clears what it provokes


def setup(groups, K, H, P, D, shared, lengths, seed, spread=0.7, own=0.3, spare_blocks=2):
    """A cache whose rows b of group b // K agree on the first shared[group] positions: in the same pages where
    whole blocks are shared (some rows have copies of them), in copies of their own behind that."""
    B = groups * K
    blocks = -(-max(lengths + [1]) // P) + spare_blocks
    cache, table = make_cache(B, blocks, H, P, D, seed)
    fill(cache, table, lengths, H, P, D, seed + 1, spread)
    rng = random.Random(seed)
    for b in range(B):
        # the longest row of a group has all that is shared
        lead = max(range(b // K * K, b // K * K + K), key=lambda r: lengths[r])
        if lead == b:
            continue
        for j in range(-(-min(shared[b // K], lengths[b]) // P)):
            src, dst = int(table[lead, j]), int(table[b, j])
            if (j + 1) * P <= min(shared[b // K], lengths[b]) and rng.random() >= own:
                table[b, j] = src
                continue
            k = min(P, shared[b // K] - j * P)              # slots behind keep their own
            for c, s in ((cache[0], cache[1]), (cache[2], cache[3])):
                s[dst] = s[src]
                c.view(torch.uint8)[dst, :, :k] = c.view(torch.uint8)[src, :, :k]
    return cache, table


def wide(table, P, tokens=1 << 18):
    """The table with room for `tokens`, as one has that is made for the longest sequence: from a thousand keys and
    some megabytes on that a call can reach, what is shared is read once, below that by every row."""
    more = torch.full((table.shape[0], tokens // P), -1, device=DEV, dtype=torch.int32)
    return torch.cat([table, more], 1)


def ints(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,D", [(16, 64), (32, 128), (64, 64), (16, 128)])
@pytest.mark.parametrize("K,T,H,G,shared,behind,counts,window", [
    (1, 1, 1, 1, [0], [1], None, None),
    (4, 1, 2, 1, [256], [9, 9, 9, 9], None, None),
    (4, 1, 3, 1, [300, 129], [40] * 8, None, 256),
    (3, 2, 1, 4, [500, 0, 16], [2, 30, 77, 5, 2, 100, 3, 3, 3], None, None),
    (5, 3, 2, 2, [257], [3, 60, 9, 200, 3], [3, 1, 0, 2, 3], None),
    (2, 1, 1, 8, [1000, 700, 33], [1, 400, 17, 1, 5, 5], None, 500),
    (8, 5, 1, 7, [400], [5, 6, 7, 8, 9, 10, 64, 65], [5, 5, 0, 4, 5, 1, 2, 5], 100),
    (64, 1, 1, 4, [700], [1 + 3 * i for i in range(64)], None, None),
    (3, 1, 2, 1, [128, 127, 15], [1] * 9, None, 0),
    (7, 4, 1, 11, [130], [4] * 7, None, 129),
    (1, 1, 1, 16, [600, 90], [1, 2], None, None),
    (2, 1, 2, 1, [1500, 2200], [1, 90, 33, 700], None, 1024),
    (4, 2, 1, 4, [1400], [2, 300, 5, 47], [2, 1, 0, 2], 1100),
    (8, 5, 1, 7, [1600], [5, 6, 7, 8, 9, 10, 64, 65], [5, 5, 0, 4, 5, 1, 2, 5], 1030),
    (3, 12, 1, 1, [1700], [12, 40, 20], None, 1200)])
@pytest.mark.parametrize("roomy", [False, True])
def test_against_definition(nat, dtype, P, D, K, T, H, G, shared, behind, counts, window, roomy):
    groups = len(shared)
    lengths = [shared[b // K] + n for b, n in enumerate(behind)]
    cache, table = setup(groups, K, H, P, D, shared, lengths, 50 + K)
    if roomy:
        table = wide(table, P)
    B = groups * K
    cnt = counts if counts else [T] * B
    q = (1.5 * torch.randn(B, T, H * G, D, device=DEV, generator=gen(60))).to(dtype)
    for b, c in enumerate(cnt):
        q[b, c:] = float("nan")                              # padding rows
    args = (q, *cache, table, ints(lengths))
    o = nat.kv_attention_shared(*args, ints(shared), counts=None if counts is None else ints(cnt), window=window)
    want, tol = attention64(q, cache, table, lengths, cnt, window, P)
    close(o, want, half(dtype), tol)
    for b, c in enumerate(cnt):
        assert (o[b, c:] == 0).all()
    assert torch.equal(o, nat.kv_attention_shared(*args, ints(shared), counts=None if counts is None else ints(cnt), window=window))
    # nothing shared is the attention without sharing
    o = nat.kv_attention_shared(*args, ints([0] * groups), counts=None if counts is None else ints(cnt), window=window)
    close(o, want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups,K,H,G,longest,tail,window", [
    (40, 3, 2, 1, 900, 50, None), (3, 20, 4, 1, 5000, 300, None), (1, 33, 1, 4, 20000, 30, None), (100, 2, 1, 1, 300, 400, 64),
    (2, 5, 16, 1, 2000, 64, 512), (1, 300, 1, 1, 700, 20, None), (30, 4, 1, 1, 3000, 700, 1024), (2, 60, 1, 4, 2500, 400, 1500),
    (260, 2, 1, 1, 200, 30, None), (520, 33, 1, 1, 40, 9, None)])
def test_many_ragged_groups(nat, dtype, groups, K, H, G, longest, tail, window):
    """Shares of the work that begin and end inside groups, groups without keys, idle and bad sequences."""
    P, D = 32, 64
    rng = random.Random(groups)
    shared = [rng.choice([rng.randint(0, longest), rng.randint(0, longest) // P * P, 0]) for _ in range(groups)]
    shared[-1] = longest
    lengths = [shared[b // K] + rng.randint(0, tail) for b in range(groups * K)]
    counts = [0 if rng.random() < 0.1 or n == 0 else 1 for n in lengths]
    cache, table = setup(groups, K, H, P, D, shared, lengths, 70 + groups, spare_blocks=5)
    table = wide(table, P)
    q = torch.randn(groups * K, 1, H * G, D, device=DEV, generator=gen(71)).to(dtype)
    n, c = ints(lengths), ints(counts)
    o = nat.kv_attention_shared(q, *cache, table, n, ints(shared), counts=c, window=window)
    want, tol = attention64(q, cache, table, lengths, counts, window, P)
    close(o, want, half(dtype), tol)
    assert nat.device_error_flags(0) == 0
    n[0], c[0] = table.shape[1] * P + 1, 1                  # past the table
    n[-1], c[-1] = 3, 2                                     # more than T
    o = nat.kv_attention_shared(q, *cache, table, n, ints(shared), counts=c, window=window)
    assert nat.device_error_flags(0) == 8
    assert (o[0] == 0).all() and (o[-1] == 0).all()
    close(o[1:-1], want[1:-1], half(dtype), tol[1:-1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_counts_and_bad_pages(nat, dtype):
    """Less than is shared may be said, nothing where it is negative; more than a sequence has is what it has; a bad page is
    not seen and flagged."""
    P, D, H, K = 16, 64, 2, 3
    lengths, shared = [200, 210, 190, 64, 64, 64], [180, 48]
    cache, table = setup(2, K, H, P, D, shared, lengths, 80)
    table = wide(table, P)
    q = torch.randn(6, 1, H, D, device=DEV, generator=gen(81)).to(dtype)
    want, tol = attention64(q, cache, table, lengths, [1] * 6, None, P)
    for fewer in ([-1, 48], [180, -5], [17, 15]):
        close(nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(fewer)), want, half(dtype), tol)
    table[:3] = table[0].clone()                            # the same pages to the end: all is shared, the new token too
    want, tol = attention64(q, cache, table, lengths, [1] * 6, None, P)
    o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints([210, 48]))
    close(o, want, half(dtype), tol)
    assert nat.device_error_flags(0) == 0
    table[:, 2] = 10 ** 6
    o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(shared))
    assert nat.device_error_flags(0) == 8
    keep = torch.cat([table[:, :2], table[:, 3:]], 1)
    want, tol = attention64(q, cache, keep, [n - P for n in lengths], [1] * 6, None, P)
    close(o, want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,K", [(64, 4), (128, 4), (64, 40), (128, 40)])
def test_extreme_scales_and_scores(nat, dtype, D, K):
    """Pages whose scales are far apart, sharp and flat rows, tiny and large queries, a scale of its own, values near the largest."""
    P, H, shared = 16, 2, [700]
    lengths = [700 + 9 * b for b in range(1, K + 1)]
    cache, table = setup(1, K, H, P, D, shared, lengths, 82)
    table = wide(table, P)
    first = table[max(range(K), key=lambda r: lengths[r])].long()
    for j, f in ((3, 2.0 ** -60), (5, 2.0 ** 30), (20, 2.0 ** -30), (41, 2.0 ** 12)):
        for b in range(K):
            page = int(table[b, j])
            cache[3][page] = cache[3][first[j]] if page != int(first[j]) else cache[3][page]
        for page in {int(table[b, j]) for b in range(K)}:
            cache[3][page] *= f
    for page in {int(table[b, 7]) for b in range(K)}:
        cache[1][page] *= 2.0 ** -40
    for mag, scale in ((1.0, None), (60.0, None), (1e-30, 1e30), (3.0, 0.01), (2.0, -0.3), (400.0, 1.0)):
        q = (mag * torch.randn(K, 1, H, D, device=DEV, generator=gen(83))).to(dtype)
        o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(shared), scale=scale)
        want, tol = attention64(q, cache, table, lengths, [1] * K, None, P, scale)
        close(o, want, half(dtype), tol)
    # finite values, however large, give finite outputs
    cache[2].view(torch.uint8)[:] = cache[2].view(torch.uint8) & 0xf7            # no NaN codes in the slots behind
    cache[3][:] = 2.0 ** 118
    q = (0.1 * torch.randn(K, 1, H, D, device=DEV, generator=gen(84))).to(dtype)
    o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(shared))
    want, tol = attention64(q, cache, table, lengths, [1] * K, None, P)
    close(o, want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", [3, 20])
def test_not_finite(nat, dtype, K):
    """A NaN reaches exactly the rows that see it; a query that is not finite only its own row."""
    P, D, H, T, shared, window = 16, 64, 1, 2, [1300], 1200
    lengths = ([1310, 1330, 1302] * K)[:K]
    for where, key in (("v", 150), ("k", 150), ("v", 1299), ("v", 108), ("k", 120), ("v", 101), ("k", 129), ("v", 5), ("k", 700)):
        cache, table = setup(1, K, H, P, D, shared, lengths, 85, own=0.0)
        table = wide(table, P)
        q = torch.randn(K, T, H, D, device=DEV, generator=gen(86)).to(dtype)
        clean, tol = attention64(q, cache, table, lengths, [T] * K, window, P)
        for b in range(K):
            cache[0 if where == "k" else 2].view(torch.uint8)[int(table[b, key // P]), 0, key % P, 5] = 0xff
        o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(shared), window=window)
        for b in range(K):
            for t in range(T):
                p = lengths[b] - T + t
                sees = p - window <= key <= p
                bad = o[b, t, 0].isnan()
                want = torch.arange(D, device=DEV) == 5 if where == "v" else torch.ones(D, device=DEV, dtype=torch.bool)
                assert torch.equal(bad, want & sees), (where, key, b, t)
                d = ((o[b, t, 0].double() - clean[b, t, 0]).abs() - half(dtype) * clean[b, t, 0].abs() - tol[b, t, 0])[~bad]
                assert d.numel() == 0 or d.max() <= 0
    cache, table = setup(1, K, H, P, D, shared, lengths, 87)
    table = wide(table, P)
    for v in (float("nan"), float("inf"), -float("inf")):
        q = torch.randn(K, T, H, D, device=DEV, generator=gen(88)).to(dtype)
        want, tol = attention64(q, cache, table, lengths, [T] * K, window, P)
        q[1, 0, 0, 3] = v
        o = nat.kv_attention_shared(q, *cache, table, ints(lengths), ints(shared), window=window)
        assert o[1, 0].isnan().any()
        o[1, 0], want[1, 0] = 0, 0
        close(o, want, half(dtype), tol)


@pytest.mark.parametrize("K", [4, 36])
def test_layouts_streams_and_graphs(nat, K):
    groups, T, H, D, P = 2, 1, 4, 64, 16
    shared, lengths = [300, 150], ([301, 333, 340, 309] * K)[:K] + ([151, 152, 153, 160] * K)[:K]
    cache, table = setup(groups, K, H, P, D, shared, lengths, 89)
    table = wide(table, P)
    B = groups * K
    qkv = torch.randn(B, T, 3 * H, D, device=DEV, generator=gen(90)).to(BF16)
    q = qkv[:, :, :H]
    n, s = ints(lengths), ints(shared)
    want = nat.kv_attention_shared(q.contiguous(), *cache, table, n, s)
    ref, tol = attention64(q, cache, table, lengths, [1] * B, None, P)
    close(want, ref, half(BF16), tol)
    assert torch.equal(nat.kv_attention_shared(q, *cache, table, n, s), want)
    odd = torch.zeros(B, T, H, D + 1, device=DEV, dtype=BF16)[..., 1:].copy_(q)
    assert torch.equal(nat.kv_attention_shared(odd, *cache, table, n, s.long()), want)
    assert torch.equal(nat.kv_attention_shared(q.transpose(2, 3).contiguous().transpose(2, 3), *cache, table, n, s), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = nat.kv_attention_shared(q, *cache, table, n, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nat.kv_attention_shared(q, *cache, table, n, s))
        graphs.append(g)
    for g in graphs:
        g.replay()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    n -= ints(([1, 20, 0, 9] * K)[:K] + ([0, 0, 1, 3] * K)[:K])
    s.copy_(ints([288, 0]))
    want = nat.kv_attention_shared(q, *cache, table, n, s)
    for _ in range(3):
        graphs[0].replay()
        assert torch.equal(outs[0], want)


@pytest.mark.parametrize("K,G", [(2, 2), (40, 4)])
def test_long_cache_past_32_bits(nat, K, G):
    """Pages whose byte offset passes 2^32."""
    H, P, D, n = 8, 64, 128, 4000
    per = H * P * D
    total = (2 ** 32) // per + 80
    kc, vc = (torch.empty(total, H, P, D, device=DEV, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.ones(total, H, device=DEV) for _ in range(2))
    table = (total - 1 - torch.randperm(70, device=DEV, generator=gen(27)))[None].int().expand(K, 70).contiguous()
    g = gen(28)
    k, v = (torch.randn(1, n, H, D, device=DEV, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(K, 1, G * H, D, device=DEV, generator=g)
    cache = [kc.view(E4M3), ks, vc.view(E4M3), vs]
    nat.kv_append(k, v, *cache, table[:1], ints([n]))
    o = nat.kv_attention_shared(q, *cache, table, ints([n] * K), ints([n - 1]))
    low = [(c.view(torch.uint8)[total - 80:] if c.dim() == 4 else c[total - 80:]) for c in cache]
    low = [low[0].view(E4M3), low[1], low[2].view(E4M3), low[3]]
    rows = [0, K - 1]
    want, tol = attention64(q[rows], low, table[rows] - (total - 80), [n, n], [1, 1], None, P)
    close(o[rows], want, U32, tol)


def test_refusals(nat):
    B, T, H, D, P = 4, 1, 2, 64, 16
    cache, table = make_cache(B, 2, H, P, D, 29)
    x, n, s = torch.zeros(B, T, H, D, device=DEV, dtype=BF16), ints([1] * B), ints([0, 0])
    good = dict(q=x, k_codes=cache[0], k_scale=cache[1], v_codes=cache[2], v_scale=cache[3], table=table, lengths=n, shared=s)
    for bad in (dict(q=x[0]), dict(k_codes=cache[0][:, :, ::2]), dict(k_codes=cache[0].view(torch.int8)), dict(k_scale=cache[1].double()),
                dict(table=table.long()), dict(table=table[:1]), dict(lengths=n[:1]), dict(counts=n[:1]), dict(window=-1),
                dict(shared=ints([0, 0, 0])), dict(shared=ints([])), dict(shared=ints([[0, 0]])), dict(q=x[:, :, :1].expand(B, T, 3, D))):
        with pytest.raises(ValueError):
            nat.kv_attention_shared(**{**good, **bad})
    for bad in (dict(q=x.half()), dict(shared=s.float()), dict(lengths=n.float())):
        with pytest.raises(TypeError):
            nat.kv_attention_shared(**{**good, **bad})
    for shape in ((4, H, 8, D), (4, H, 48, D), (4, H, P, 96)):
        c, sc = torch.zeros(shape, device=DEV, dtype=torch.uint8), torch.zeros(shape[:2], device=DEV)
        y = torch.zeros(B, T, H, shape[3], device=DEV)
        with pytest.raises(nat.NativeError):
            nat.kv_attention_shared(y, c, sc, c.clone(), sc.clone(), table, n, s)
    with pytest.raises(RuntimeError, match="no backward"):
        nat.kv_attention_shared(**{**good, "q": x.clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_attention_shared(**{**good, "shared": s.cpu()})
    assert nat.kv_attention_shared(**{**good, "window": 2 ** 63 - 1}).shape == (B, T, H, D)
    assert nat.kv_attention_shared(**{**good, "q": x[:, :0]}).shape == (B, 0, H, D)
    assert nat.kv_attention_shared(x[:0], *cache, table[:0], n[:0], s).shape == (0, T, H, D)
