"""The operators of a generation step with an attention memory (B200): rotary positions, the
8-bit cache, attention over it, penalties on logits.

Each is compared with its definition in float64, written out here.  Tolerances
are counted from the roundings: half a step of the output type (``eps / 2``)
relative to the value, plus what float32 arithmetic leaves, stated at each test.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
U32 = 2.0 ** -24                       # half a step of float32
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0      # every test clears what it provokes


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def close(got, want, rtol, atol):
    """|got - want| <= rtol |want| + atol elementwise, equal where not finite."""
    got, want = got.double(), want.double()
    fin = want.isfinite()
    assert torch.equal(got.isfinite(), fin)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    over = ((got - want).abs() - rtol * want.abs() - atol)[fin]
    assert over.numel() == 0 or over.max().item() <= 0, f"off by {over.max().item():.3g} over the tolerance"


# --------------------------------------------------------------------------- #
#  rotary                                                                      #
# --------------------------------------------------------------------------- #

def rotary64(x, pos, freq, layout, m, inverse=False):
    x = x.double()
    R = 2 * freq.numel()
    a = pos.double()[..., None, None] * freq.double()
    c, s = m * a.cos(), m * a.sin() * (-1 if inverse else 1)
    y = x.clone()
    i1, i2 = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1] = x1 * c - x2 * s
    y[..., i2] = x2 * c + x1 * s
    mag = torch.zeros_like(x)
    mag[..., i1] = mag[..., i2] = abs(m) * (x1.abs() + x2.abs())
    return y, mag


# float32: the angle in turns is rounded once (pi 2^-24 radians at most), sincospi is good to
# 2 half steps, the product with mscale, two products and a sum round once each: 8 half steps of
# float32 relative to |x1| + |x2| cover them.
ROT = 8 * U32


def freqs(R, base=10000.0):
    return (base ** -(torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)).float()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,D,R,first", [
    (1, 1, 1, 64, 64, 0), (64, 1, 32, 128, 128, 8191), (2, 37, 5, 64, 32, 5), (3, 7, 20, 128, 122, 100000),
    (1, 1, 3, 6, 2, 7), (1, 1, 1, 7, 4, -50), (2, 300, 1, 80, 80, 3000000), (5, 3, 40, 72, 48, 2 ** 31), (1, 3, 2, 600, 600, 1)])
def test_rotary_against_definition(nat, layout, dtype, B, T, H, D, R, first):
    g = gen(1)
    x = torch.randn(B, T, H, D, device=DEV, generator=g).to(dtype)
    pos = first + torch.randint(0, 50, (B, T), device=DEV, generator=g)
    f, m = freqs(R), 1.3
    y = nat.rotary(x, pos, f, layout=layout, mscale=m)
    want, mag = rotary64(x, pos, f, layout, m)
    close(y, want, half(dtype), ROT * mag)
    assert torch.equal(y[..., R:], x[..., R:])
    back = nat.rotary(x, pos, f, layout=layout, mscale=m, inverse=True)
    want, mag = rotary64(x, pos, f, layout, m, inverse=True)
    close(back, want, half(dtype), ROT * mag)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_strides_shared_positions_and_in_place(nat, dtype):
    B, T, H, D = 3, 33, 4, 64
    qkv = torch.randn(B, T, 3 * H, D, device=DEV, generator=gen(2)).to(dtype)
    pos, f = torch.arange(T, device=DEV, dtype=torch.int32), freqs(D)
    view = qkv[:, :, :2 * H]
    want = nat.rotary(view.contiguous(), pos.long().expand(B, T).contiguous(), f)
    assert torch.equal(nat.rotary(view, pos, f), want)
    # heads outside tokens, odd offsets that no 16-byte vector fits
    byhead = view.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(nat.rotary(byhead, pos, f), want)
    wide = torch.zeros(B, T, 2 * H, D + 3, device=DEV, dtype=dtype)
    wide[..., 1:D + 1] = view
    assert torch.equal(nat.rotary(wide[..., 1:D + 1], pos, f), want)
    got = nat.rotary(wide[..., 1:D + 1], pos, f, out=wide[..., 1:D + 1])
    assert got.data_ptr() == wide[..., 1:].data_ptr() and torch.equal(got, want)
    assert wide[..., 0].abs().max() == 0 and wide[..., D + 1:].abs().max() == 0
    rest = qkv[:, :, 2 * H:].clone()
    nat.rotary(view, pos, f, out=view)
    assert torch.equal(qkv[:, :, :2 * H], want) and torch.equal(qkv[:, :, 2 * H:], rest)
    one = view[:, :1].expand(B, T, 2 * H, D)                      # a broadcast input
    assert torch.equal(nat.rotary(one, pos, f), nat.rotary(one.contiguous(), pos, f))
    assert nat.rotary(view[:, :0], pos[:0], f).shape == (B, 0, 2 * H, D)


def test_rotary_rejoins_the_module_tables(nat):
    """Positions 0..T-1 with the module's frequencies are apply_rotary on its float32 tables."""
    from neuratensor_b200.core.model import RotaryEmbedding, apply_rotary
    T, H, D = 65, 3, 64
    rope = RotaryEmbedding(D).to(DEV)
    x = torch.randn(2, T, H, D, device=DEV, generator=gen(3))
    cos, sin = rope(x.transpose(1, 2))
    want = apply_rotary(x.transpose(1, 2), cos, sin).transpose(1, 2)
    y = nat.rotary(x, torch.arange(T, device=DEV), rope.inv_freq)
    # the tables round the angle to float32: T * 2^-24 radians at most, beside the arithmetic above on both sides
    mag = x.abs().double() + torch.cat([x[..., D // 2:], x[..., :D // 2]], -1).abs()
    close(y, want, 0.0, (2 * ROT + T * U32) * mag)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(nat, layout):
    B, T, H, D, R = 2, 9, 3, 64, 40
    g = gen(4)
    x = torch.randn(B, T, H, D, device=DEV, generator=g, requires_grad=True)
    dy = torch.randn(B, T, H, D, device=DEV, generator=g)
    pos, f, m = torch.randint(0, 5000, (B, T), device=DEV, generator=g), freqs(R), 0.9
    y = nat.rotary(x, pos, f, layout=layout, mscale=m)
    (gx,) = torch.autograd.grad(y, x, dy)
    want, mag = rotary64(dy, pos, f, layout, m, inverse=True)
    close(gx, want, U32, ROT * mag)
    # against differences: the map is linear, so one difference of any size is the derivative
    d = torch.randn(B, T, H, D, device=DEV, generator=g)
    with torch.no_grad():
        num = ((nat.rotary(x + d, pos, f, layout=layout, mscale=m).double() -
                nat.rotary(x, pos, f, layout=layout, mscale=m).double()) * dy).sum()
    terms = (dy.abs() * (x.abs() + d.abs() + 1)).double().sum()
    assert abs(num - (gx.double() * d).sum()) <= 4 * ROT * terms
    # a broadcast input gets the sum over what it was broadcast to
    one = torch.randn(B, 1, H, D, device=DEV, generator=g, requires_grad=True)
    (g1,) = torch.autograd.grad(nat.rotary(one.expand(B, T, H, D), pos, f, layout=layout, mscale=m), one, dy)
    # torch adds the T gradients in float32: T - 1 roundings, each of a partial sum of at most sum |gradient|,
    # which is at most sum |dy| for the copied dimensions and sum of mag for the turned ones
    close(g1, want.sum(1, keepdim=True), U32, ROT * mag.sum(1, keepdim=True) +
          T * U32 * (mag + dy.abs()).sum(1, keepdim=True))
    assert not nat.rotary(x.detach(), pos, f).requires_grad
    with pytest.raises(RuntimeError, match="no backward"):
        nat.rotary(x, pos, f, out=torch.empty_like(x))


def test_rotary_captured_with_its_gradient(nat):
    B, T, H, D = 2, 5, 3, 64
    x = torch.randn(B, T, H, D, device=DEV, generator=gen(50), requires_grad=True)
    dy = torch.randn(B, T, H, D, device=DEV, generator=gen(51))
    pos, f = torch.arange(T, device=DEV), freqs(D)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = nat.rotary(x, pos, f)
        (gx,) = torch.autograd.grad(y, x, dy)
    for first in (0, 700, 123456):
        pos.copy_(first + torch.arange(T, device=DEV))
        g.replay()
        want, mag = rotary64(x.detach(), pos.expand(B, T), f, "half", 1.0)
        close(y.detach(), want, U32, ROT * mag)
        want, mag = rotary64(dy, pos.expand(B, T), f, "half", 1.0, inverse=True)
        close(gx, want, U32, ROT * mag)


def test_rotary_refusals(nat):
    x, p, f = torch.zeros(2, 3, 4, 64, device=DEV), torch.zeros(2, 3, device=DEV, dtype=torch.int64), freqs(64)
    for bad in (dict(x=x[0]), dict(layout="pairs"), dict(inv_freq=f.double()), dict(inv_freq=freqs(66)),
                dict(positions=p[:, :2]), dict(out=x[:, :, :, :32]), dict(out=x[:1].expand(2, 3, 4, 64)),
                dict(inv_freq=f[:0])):
        with pytest.raises(ValueError):
            nat.rotary(**{**dict(x=x, positions=p, inv_freq=f), **bad})
    with pytest.raises(TypeError):
        nat.rotary(x.half(), p, f)
    with pytest.raises(TypeError):
        nat.rotary(x, p.float(), f)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.rotary(x.cpu(), p, f)


# --------------------------------------------------------------------------- #
#  the cache                                                                   #
# --------------------------------------------------------------------------- #

def make_cache(B, blocks, H, P, D, seed=0, spare=2):
    """A pool with stale contents, NaN codes among them, and shuffled pages."""
    g = gen(seed)
    n = B * blocks + spare
    kc, vc = (torch.randint(0, 256, (n, H, P, D), device=DEV, generator=g, dtype=torch.uint8).view(E4M3) for _ in range(2))
    ks, vs = (2.0 ** torch.randint(-6, 6, (n, H), device=DEV, generator=g).float() for _ in range(2))
    table = torch.randperm(n, device=DEV, generator=g)[:B * blocks].view(B, blocks).int()
    return [kc, ks, vc, vs], table


def scale64(amax):
    return 2.0 ** max(-126, math.ceil(math.log2(amax / 448) - 1e-12)) if amax > 0 else 2.0 ** -126


def e4m3(y):
    """Round a float64 tensor to e4m3, saturating; the torch cast rounds float32 to nearest even
    and the inputs here (code or bf16/float32 value times a power of two) are exact in float32."""
    return y.clamp(-448, 448).float().to(E4M3)


def append64(x, codes, scale, table, lengths, counts, P):
    codes, scale = codes.view(torch.uint8).clone().view(E4M3), scale.clone()
    for b in range(x.shape[0]):
        n, c = int(lengths[b]), int(counts[b])
        first = n - c
        for blk in range(first // P, -(-n // P) if c else 0):
            lo, hi = max(first, blk * P), min(n, blk * P + P)
            if hi <= lo:
                continue
            page = int(table[b, blk])
            for h in range(x.shape[2]):
                y = x[b, lo - first:hi - first, h].double()
                fin = y[y.isfinite()].abs()
                s, k = scale64(fin.max().item() if fin.numel() else 0.0), lo - blk * P
                if k:
                    old = scale[page, h].item()
                    s = max(s, old)
                    if s > old:
                        codes[page, h, :k] = e4m3(codes[page, h, :k].double() * (old / s))
                codes[page, h, k:hi - blk * P] = e4m3(y / s)
                scale[page, h] = s
    return codes, scale


def same_codes(a, b):
    """Equal bytes, any NaN code for any NaN code."""
    a, b = a.view(torch.uint8), b.view(torch.uint8)
    nan = ((a & 127) == 127) & ((b & 127) == 127)
    return bool(((a == b) | nan).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P", [16, 32, 64])
@pytest.mark.parametrize("B,T,H,D,lengths,counts", [
    (1, 1, 1, 64, [1], None), (3, 1, 4, 128, [17, 64, 130], None),
    (4, 70, 3, 64, [70, 71, 100, 133], [70, 1, 0, 69]), (2, 129, 2, 128, [129, 200], [129, 65]),
    (2, 16, 1, 64, [64, 63], None)])
def test_kv_append_bit_exact(nat, dtype, P, B, T, H, D, lengths, counts):
    g = gen(5)
    cache, table = make_cache(B, 13, H, P, D, 6)
    lengths = torch.tensor(lengths, device=DEV)
    cnt = torch.tensor(counts if counts else [T] * B, device=DEV)
    kv = torch.randn(B, T, 2, H, D, device=DEV, generator=g) * torch.exp(3 * torch.randn(B, T, 2, H, 1, device=DEV, generator=g))
    kv = kv.to(dtype)
    for b, c in enumerate(cnt.tolist()):
        kv[b, c:] = float("nan")                              # padding may hold anything
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = [append64(x, c, s, table, lengths, cnt, P) for x, c, s in ((k, cache[0], cache[1]), (v, cache[2], cache[3]))]
    nat.kv_append(k, v, *cache, table, lengths, counts=None if counts is None else cnt)
    for (codes, scale), (c, s) in zip(want, ((cache[0], cache[1]), (cache[2], cache[3]))):
        assert same_codes(c, codes)
        assert torch.equal(s, scale)


def test_kv_append_one_by_one_is_append_at_once(nat):
    """Growing scales re-encode by powers of two: a page filled token by token holds what it would hold
    filled at once, as long as no code falls among e4m3's subnormals (values within 2^7 of each other do not)."""
    B, T, H, D, P = 2, 40, 3, 64, 16
    g = gen(7)
    x = (1 + torch.rand(B, T, H, D, device=DEV, generator=g)) * torch.where(torch.rand(B, T, H, D, device=DEV, generator=g) < 0.5, -1.0, 1.0)
    x = (x * 2.0 ** torch.linspace(0, 6, T, device=DEV)[None, :, None, None].floor()).to(BF16)
    a, table = make_cache(B, 3, H, P, D, 8)
    b = [t.clone() for t in a]
    full = torch.full((B,), T, device=DEV, dtype=torch.int32)
    nat.kv_append(x, x.neg(), *a, table, full)
    for t in range(T):
        nat.kv_append(x[:, t:t + 1], x[:, t:t + 1].neg(), *b, table, torch.full_like(full, t + 1))
    for p, q in zip(a, b):
        assert same_codes(p, q) if p.dtype == E4M3 else torch.equal(p, q)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kv_append_special_values(nat, dtype):
    """Zeros, infinities, NaN, the largest and smallest numbers."""
    P, D = 16, 64
    cache, table = make_cache(1, 6, 1, P, D, 9)
    x = torch.zeros(1, 6 * P, 1, D, device=DEV)
    tiny = torch.finfo(dtype).tiny
    x[0, P, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0])
    x[0, 2 * P, 0, :3] = torch.tensor([torch.finfo(dtype).max, 1.0, -1e30])
    x[0, 3 * P, 0, :3] = torch.tensor([tiny, -tiny / 4, tiny / 128])
    x[0, 4 * P:, 0] = float("inf")
    x[0, 5 * P:, 0] = 448.0
    x = x.to(dtype)
    n = torch.tensor([6 * P], device=DEV)
    want = append64(x, cache[0], cache[1], table, n, n, P)
    nat.kv_append(x, x, *cache, table, n)
    assert same_codes(cache[0], want[0]) and torch.equal(cache[1], want[1])
    pages = table[0].long()
    assert cache[0].view(torch.uint8)[pages[0]].abs().max() == 0          # a zero page is zero, at the smallest scale
    assert cache[1][pages[0]].item() == 2.0 ** -126
    assert cache[1][pages[5]].item() == 1.0
    c = cache[0][pages[1], 0, 0, :4].float().tolist()
    assert c[0] == 448 and c[1] == -448 and math.isnan(c[2]) and c[3] == 3.0 / cache[1][pages[1]].item()


def test_kv_append_strides_and_untouched_slots(nat):
    B, T, H, D, P = 2, 21, 3, 64, 16
    qkv = torch.randn(B, T, 3 * H, D, device=DEV, generator=gen(10)).to(BF16)
    a, table = make_cache(B, 3, H, P, D, 11)
    b, before = [t.clone() for t in a], [t.clone() for t in a]
    n = torch.tensor([21, 40], device=DEV, dtype=torch.int32)
    k, v = qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    nat.kv_append(k, v, *a, table, n)
    odd = torch.zeros(B, T, H, D + 1, device=DEV, dtype=BF16)[..., 1:]
    odd.copy_(k)
    nat.kv_append(odd, v.transpose(1, 2).contiguous().transpose(1, 2), b[0].view(torch.uint8), b[1], b[2].view(torch.uint8), b[3], table, n)
    for p, q in zip(a, b):
        assert torch.equal(p.view(torch.uint8) if p.dtype == E4M3 else p, q.view(torch.uint8) if q.dtype == E4M3 else q)
    # what no new token reaches is as it was: other pages, slots behind the last token
    used = set(table[0, :2].tolist()) | set(table[1, 1:3].tolist())
    for p, q in zip(a, before):
        p, q = (t.view(torch.uint8) if t.dtype == E4M3 else t for t in (p, q))
        for page in range(p.shape[0]):
            if page not in used:
                assert torch.equal(p[page], q[page])
        if p.dim() == 4:
            assert torch.equal(p[table[0, 1].item(), :, 5:], q[table[0, 1].item(), :, 5:])
            assert torch.equal(p[table[1, 2].item(), :, 8:], q[table[1, 2].item(), :, 8:])


def test_kv_bad_sequences_and_pages_are_skipped_and_flagged(nat):
    B, T, H, D, P = 5, 4, 2, 64, 16
    cache, table = make_cache(B, 2, H, P, D, 12)
    before = [t.clone() for t in cache]
    x = torch.randn(B, T, H, D, device=DEV, generator=gen(13)).to(BF16)
    lengths = torch.tensor([4, 3, 33, 4, 20], device=DEV, dtype=torch.int32)       # 3 < count 4; 33 past the table
    counts = torch.tensor([4, 4, 4, 5, 4], device=DEV, dtype=torch.int32)          # 5 > T
    table[4, 1] = cache[0].shape[0]                                                # a page that is not there
    table[0, 1] = -1                                                               # never reached
    nat.kv_append(x, x, *cache, table, lengths, counts=counts)
    assert nat.device_error_flags(0) == 8
    for p, q in zip(cache, before):
        p, q = (t.view(torch.uint8) if t.dtype == E4M3 else t for t in (p, q))
        changed = {i for i in range(p.shape[0]) if not torch.equal(p[i], q[i])}
        assert changed == {table[0, 0].item()}
    cache[0].view(torch.uint8)[:] = 0x38
    cache[2].view(torch.uint8)[:] = 0x38
    q = torch.randn(B, T, H, D, device=DEV, generator=gen(14)).to(BF16)
    o = nat.kv_attention(q, *cache, table, lengths, counts=counts)
    assert nat.device_error_flags(0) == 8
    assert o[1:4].abs().max() == 0
    assert o[0].isfinite().all() and o[0].abs().min() > 0
    assert o[4].isfinite().all() and o[4].abs().min() > 0                          # keys of the bad page are not seen
    want = attention64(q[4:], cache, table[4:, :1], torch.tensor([16]), torch.tensor([1]), None, P)[0]
    close(o[4:, :1], want[:, :1], half(BF16), 2.0 ** -11 * want[:, :1].abs())


# --------------------------------------------------------------------------- #
#  attention over the cache                                                    #
# --------------------------------------------------------------------------- #

def attention64(q, cache, table, lengths, counts, window, P, scale=None):
    """(output, bound): the bound is what float32 scores and weights may be off by."""
    kc, ks, vc, vs = cache
    B, T, Hq, D = q.shape
    H = kc.shape[1]
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, T, Hq, D, device=DEV, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n, c = int(lengths[b]), int(counts[b])
        pages = table[b, :-(-n // P)].long()
        k, v = ((x.view(torch.uint8)[pages].view(E4M3).double() * s[pages].double()[:, :, None, None]).transpose(0, 1)
                .reshape(H, -1, D)[:, :n] for x, s in ((kc, ks), (vc, vs)))
        for t in range(c):
            p = n - c + t
            lo = 0 if window is None else max(0, p - window)
            for h in range(Hq):
                kk, vv, qq = k[h // G, lo:p + 1], v[h // G, lo:p + 1], q[b, t, h].double()
                sc = scale * (kk @ qq)
                w = torch.softmax(sc, 0)
                out[b, t, h] = w @ vv
                # scores: D products summed in float32, three factors multiplied on; weights: exp2 to 2^-22;
                # sums over n keys; float32 q and weights as f16 pairs (2^-22), bf16 outputs from f16 weights (2^-12)
                es = abs(scale) * (kk.abs() @ qq.abs()).max() * (D + 8) * U32
                rel = 2 * (es + 2.0 ** -21 + (p - lo + 33) / 16 * U32 + (2.0 ** -12 if q.dtype == BF16 else 2.0 ** -21))
                tol[b, t, h] = rel * (w @ vv.abs())
    return out, tol


def fill(cache, table, lengths, H, P, D, seed, spread=0.7):
    """Random codes and scales in the pages in use; slots past each length stay stale."""
    g = gen(seed)
    for c, s in ((cache[0], cache[1]), (cache[2], cache[3])):
        x = torch.randn(c.shape, device=DEV, generator=g) * torch.exp(spread * torch.randn(c.shape[0], H, 1, D, device=DEV, generator=g))
        amax = x.abs().amax((2, 3))
        sc = 2.0 ** torch.ceil(torch.log2(amax / 448))
        for b, n in enumerate(lengths):
            for blk in range(-(-n // P)):
                page, k = int(table[b, blk]), min(P, n - blk * P)
                s[page] = sc[page]
                c[page, :, :k] = (x[page, :, :k] / sc[page][:, None, None]).to(E4M3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,D", [(16, 64), (32, 128), (64, 64)])
@pytest.mark.parametrize("T,H,G,lengths,counts,window", [
    (1, 1, 1, [1], None, None), (1, 3, 1, [1, 15, 16, 17, 300], None, None), (1, 2, 4, [257, 33, 2, 64], None, 256),
    (5, 2, 1, [5, 9, 0, 200, 77], [5, 3, 0, 1, 5], None), (3, 1, 7, [3, 100, 515], [3, 2, 3], 40),
    (1, 1, 8, [700], None, 0), (20, 1, 2, [20, 333], [20, 17], 11), (1, 1, 16, [90], None, None),
    (2, 1, 1, [1500], None, 1000)])
def test_kv_attention_against_definition(nat, dtype, P, D, T, H, G, lengths, counts, window):
    B = len(lengths)
    cache, table = make_cache(B, 1536 // P, H, P, D, 15)
    fill(cache, table, lengths, H, P, D, 16)
    q = (1.5 * torch.randn(B, T, H * G, D, device=DEV, generator=gen(17))).to(dtype)
    cnt = counts if counts else [T] * B
    for b, c in enumerate(cnt):
        q[b, c:] = float("nan")                              # padding rows
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    o = nat.kv_attention(q, *cache, table, n, counts=None if counts is None else torch.tensor(cnt, device=DEV, dtype=torch.int32),
                         window=window)
    want, tol = attention64(q, cache, table, lengths, cnt, window, P)
    close(o, want, half(dtype), tol)
    for b, c in enumerate(cnt):
        assert (o[b, c:] == 0).all()


@pytest.mark.parametrize("B,H,G,longest,window", [(70, 2, 1, 900, None), (520, 1, 2, 200, None), (300, 4, 1, 60, None), (9, 1, 8, 1300, None),
                                                  (150, 2, 1, 700, 33), (2, 1, 1, 1536, None)])
def test_kv_attention_many_ragged_sequences(nat, B, H, G, longest, window):
    """Shares of the work that begin and end inside sequences, sequences without keys between them, batches
    of every size that the plan tells apart; twice the same bits, and bad sequences flagged and zero."""
    P, D = 16, 64
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lengths[-1] = longest
    counts = [min(1, n) for n in lengths]
    counts[B // 2] = 0
    cache, table = make_cache(B, 96, H, P, D, 40)
    fill(cache, table, lengths, H, P, D, 41)
    q = torch.randn(B, 1, H * G, D, device=DEV, generator=gen(42)).to(BF16)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    c = torch.tensor(counts, device=DEV, dtype=torch.int32)
    o = nat.kv_attention(q, *cache, table, n, counts=c, window=window)
    want, tol = attention64(q, cache, table, lengths, counts, window, P)
    close(o, want, half(BF16), tol)
    assert torch.equal(o, nat.kv_attention(q, *cache, table, n, counts=c, window=window))
    assert nat.device_error_flags(0) == 0
    n[0], c[0] = 97 * P, 1                                   # past the table
    n[1], c[1] = 3, 2                                        # more than T
    o2 = nat.kv_attention(q, *cache, table, n, counts=c, window=window)
    assert nat.device_error_flags(0) == 8
    assert (o2[:2] == 0).all()
    close(o2[2:], want[2:], half(BF16), tol[2:])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kv_attention_extreme_scales_and_scores(nat, dtype):
    """Pages whose scales are 2^60 apart, sharp and flat rows, tiny and large queries, a scale of its own."""
    P, D, H, n = 16, 64, 2, 200
    cache, table = make_cache(1, 16, H, P, D, 18)
    fill(cache, table, [n], H, P, D, 19)
    cache[3][table[0, 3].long()] *= 2.0 ** -60
    cache[3][table[0, 5].long()] *= 2.0 ** 30
    cache[1][table[0, 7].long()] *= 2.0 ** -40
    for mag, scale in ((1.0, None), (60.0, None), (1e-30, 1e30), (1e-42 if dtype == F32 else 1e-38, 1.0), (3.0, 0.01), (2.0, -0.3)):
        q = (mag * torch.randn(1, 1, H, D, device=DEV, generator=gen(20))).to(dtype)
        o = nat.kv_attention(q, *cache, table, torch.tensor([n], device=DEV), scale=scale)
        want, tol = attention64(q, cache, table, [n], [1], None, P, scale)
        close(o, want, half(dtype), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kv_attention_not_finite(nat, dtype):
    """A NaN reaches exactly the rows that see it: keys behind a row's position or before its window do not."""
    P, D, H, n, T, window = 16, 64, 1, 100, 3, 20
    for where, key in (("v", 99), ("v", 98), ("v", 77), ("v", 79), ("k", 99), ("k", 78), ("v", 40), ("k", 90)):
        cache, table = make_cache(1, 7, H, P, D, 21)
        fill(cache, table, [n], H, P, D, 22)
        q = torch.randn(1, T, H, D, device=DEV, generator=gen(23)).to(dtype)
        clean, tol = attention64(q, cache, table, [n], [T], window, P)
        codes = cache[0 if where == "k" else 2].view(torch.uint8)
        codes[int(table[0, key // P]), 0, key % P, 5] = 0xff
        o = nat.kv_attention(q, *cache, table, torch.tensor([n], device=DEV), window=window)
        sees = torch.tensor([97 + t - window <= key <= 97 + t for t in range(T)], device=DEV)
        bad = o[0, :, 0].isnan()
        # a row that sees a NaN key is NaN, one that sees a NaN value is NaN in that dimension
        want = sees[:, None] & (torch.arange(D, device=DEV) == 5 if where == "v" else torch.ones(D, device=DEV, dtype=torch.bool))
        assert torch.equal(bad, want), (where, key)
        d = ((o.double() - clean).abs() - half(dtype) * clean.abs() - tol)[0, :, 0][~bad]
        assert d.numel() == 0 or d.max() <= 0
    q = torch.randn(1, 2, H, D, device=DEV, generator=gen(23)).to(dtype)
    q[0, 0, 0, 3] = float("nan")
    o = nat.kv_attention(q, *cache, table, torch.tensor([50], device=DEV))
    assert o[0, 0].isnan().all() and o[0, 1].isfinite().all()


def test_kv_attention_strided_q_other_stream_and_graph(nat):
    B, T, H, D, P = 4, 1, 4, 64, 16
    lengths = [40, 1, 300, 77]
    cache, table = make_cache(B, 20, H, P, D, 24)
    fill(cache, table, lengths, H, P, D, 25)
    qkv = torch.randn(B, T, 3 * H, D, device=DEV, generator=gen(26)).to(BF16)
    q = qkv[:, :, :H]
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    want = nat.kv_attention(q.contiguous(), *cache, table, n)
    assert torch.equal(nat.kv_attention(q, *cache, table, n), want)
    odd = torch.zeros(B, T, H, D + 1, device=DEV, dtype=BF16)[..., 1:].copy_(q)
    assert torch.equal(nat.kv_attention(odd, *cache, table, n), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = nat.kv_attention(q, *cache, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want)
    # two captured graphs, each with its own workspace, replayed in turn and again after the lengths moved
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nat.kv_attention(q, *cache, table, n))
        graphs.append(g)
    for g in graphs:
        g.replay()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    # a table wide enough that the work is shared between CTAs and joined by a second kernel
    wide = torch.cat([table, table.flip(1), table, table.flip(1), table], 1)
    first = nat.kv_attention(q, *cache, wide, n)
    close(first, *(lambda w, t: (w, half(BF16), t))(*attention64(q, cache, table, lengths, [1] * B, None, P)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        joined = nat.kv_attention(q, *cache, wide, n)
    for _ in range(3):
        joined.zero_()
        g.replay()
        assert torch.equal(joined, first)
    n -= torch.tensor([1, 0, 37, 60], device=DEV, dtype=torch.int32)
    want = nat.kv_attention(q, *cache, table, n)
    graphs[0].replay()
    assert torch.equal(outs[0], want)


def test_kv_attention_long_cache_past_32_bits(nat):
    """Pages whose byte offset passes 2^32, a sequence long enough to be split, against the definition."""
    H, P, D, n = 8, 64, 128, 4000
    per = H * P * D
    total = (2 ** 32) // per + 80
    kc, vc = (torch.empty(total, H, P, D, device=DEV, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.ones(total, H, device=DEV) for _ in range(2))
    table = (total - 1 - torch.randperm(70, device=DEV, generator=gen(27)))[None].int()
    g = gen(28)
    k, v = (torch.randn(1, n, H, D, device=DEV, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(1, 1, 2 * H, D, device=DEV, generator=g)
    cache = [kc.view(E4M3), ks, vc.view(E4M3), vs]
    length = torch.tensor([n], device=DEV)
    nat.kv_append(k, v, *cache, table, length)
    o = nat.kv_attention(q, *cache, table, length)
    low = [(c.view(torch.uint8)[total - 80:] if c.dim() == 4 else c[total - 80:]) for c in cache]
    low = [low[0].view(E4M3), low[1], low[2].view(E4M3), low[3]]
    want, tol = attention64(q, low, table - (total - 80), [n], [1], None, P)
    close(o, want, U32, tol)


def test_kv_refusals(nat):
    B, T, H, D, P = 2, 1, 2, 64, 16
    cache, table = make_cache(B, 2, H, P, D, 29)
    x, n = torch.zeros(B, T, H, D, device=DEV, dtype=BF16), torch.ones(B, device=DEV, dtype=torch.int32)
    good = dict(k=x, v=x, k_codes=cache[0], k_scale=cache[1], v_codes=cache[2], v_scale=cache[3], table=table, lengths=n)
    for bad in (dict(k=x[0]), dict(v=x[:, :, :1]), dict(v=x.float()), dict(k_codes=cache[0][:, :, ::2]),
                dict(k_codes=cache[0].view(torch.int8)), dict(k_scale=cache[1].double()), dict(v_scale=cache[3][:1]),
                dict(table=table.long()), dict(table=table[:1]), dict(table=table.t().contiguous().t()),
                dict(lengths=n[:1]), dict(counts=n[:1]), dict(v_codes=cache[0])):
        with pytest.raises(ValueError):
            nat.kv_append(**{**good, **bad})
    with pytest.raises(TypeError):
        nat.kv_append(**{**good, "k": x.half(), "v": x.half()})
    with pytest.raises(TypeError):
        nat.kv_append(**{**good, "lengths": n.float()})
    with pytest.raises(RuntimeError, match="no backward"):
        nat.kv_append(**{**good, "k": x.clone().requires_grad_()})
    for shape in ((4, H, 8, D), (4, H, 48, D), (4, H, P, 96)):         # pages and head dims that are not built
        c = torch.zeros(shape, device=DEV, dtype=torch.uint8)
        s = torch.zeros(shape[:2], device=DEV)
        y = torch.zeros(B, T, H, shape[3], device=DEV)
        with pytest.raises(nat.NativeError):
            nat.kv_append(y, y, c, s, c.clone(), s.clone(), table, n)
        with pytest.raises(nat.NativeError):
            nat.kv_attention(y, c, s, c.clone(), s.clone(), table, n)
    with pytest.raises(ValueError):
        nat.kv_attention(x[:, :, :1].expand(B, T, 3, D), *cache, table, n)
    with pytest.raises(ValueError):
        nat.kv_attention(x, *cache, table, n, window=-1)
    with pytest.raises(RuntimeError, match="no backward"):
        nat.kv_attention(x.clone().requires_grad_(), *cache, table, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_attention(x, *cache, table, n.cpu())
    assert nat.kv_attention(x, *cache, table, n, window=2 ** 63 - 1).shape == (B, T, H, D)     # as good as none
    assert nat.kv_attention(x[:, :0], *cache, table, n).shape == (B, 0, H, D)
    assert nat.kv_attention(x[:0], *cache, table[:0], n[:0]).shape == (0, T, H, D)


# --------------------------------------------------------------------------- #
#  logits                                                                      #
# --------------------------------------------------------------------------- #

def logits64(x, tokens=None, lengths=None, prompts=None, rep=None, fq=None, ps=None, ids=None, bias=None, allowed=None):
    """(result, bound in float32 half steps of the largest intermediate)."""
    x = x.double().clone()
    B, V = x.shape
    mag = x.abs().clone()
    for b in range(B):
        get = lambda p, none: none if p is None else (float(p[b]) if isinstance(p, torch.Tensor) else p)  # noqa: E731
        row = x[b]
        n = 0 if tokens is None else (tokens.shape[1] if lengths is None else int(lengths[b]))
        hist = tokens[b, :n] if n else torch.zeros(0, dtype=torch.int64, device=DEV)
        made = hist[(0 if prompts is None else int(prompts[b])):]
        hist, made = (t[(t >= 0) & (t < V)] for t in (hist, made))
        seen = torch.bincount(hist, minlength=V) > 0
        times = torch.bincount(made, minlength=V).double()
        r = get(rep, 1.0)
        row = torch.where(seen, torch.where(row > 0, row / r, row * r), row)
        row = row - get(fq, 0.0) * times - get(ps, 0.0) * (times > 0)
        mag[b] += row.abs() + abs(get(fq, 0.0)) * times + abs(get(ps, 0.0))
        if ids is not None:
            last = {i: j for j, i in enumerate(ids[b].tolist()) if 0 <= i < V}
            for i, j in last.items():
                row[i] += float(bias[b, j])
                mag[b, i] += abs(float(bias[b, j]))
        if allowed is not None:
            w = allowed[b if allowed.shape[0] > 1 else 0].long()[torch.arange(V, device=DEV) // 32]
            row = torch.where((w >> (torch.arange(V, device=DEV) % 32)) & 1 == 1, row, -math.inf)
        x[b] = row
    return x, mag


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V,L,N", [(1, 1, 1, 1), (3, 33, 5, 4), (2, 1000, 0, 0), (5, 32000, 300, 40), (2, 50001, 1000, 7),
                                     (3, 131072, 64, 300), (1, 401000, 500, 50), (2, 777, 40000, 3)])
def test_logits_against_definition(nat, dtype, B, V, L, N):
    g = gen(30)
    x = (3 * torch.randn(B, V, device=DEV, generator=g)).to(dtype)
    x[0, 0] = 0.0
    tokens = torch.randint(0, max(1, V // 3 + 1), (B, L), device=DEV, generator=g) - (1 if V > 40 else 0)    # -1 among them
    lengths = torch.randint(0, L + 1, (B,), device=DEV, generator=g)
    prompts = (lengths * torch.rand(B, device=DEV, generator=g)).long()
    rep, fq = 1 + torch.rand(B, device=DEV, generator=g), torch.rand(B, device=DEV, generator=g)
    ids = torch.randint(-1, V, (B, N), device=DEV, generator=g)
    if N > 2:
        ids[:, N - 1] = ids[:, 0]                               # the same index twice: the last holds
    bias = 5 * torch.randn(B, N, device=DEV, generator=g)
    mask = torch.rand(B, V, device=DEV, generator=g) < 0.8
    if B > 1:
        mask[1] = False                                         # nothing allowed
    allowed = nat.pack_allowed(mask)
    kw = dict(tokens=tokens, lengths=lengths)
    for case in (dict(repetition=rep, **kw), dict(frequency=fq, presence=0.5, prompt_lengths=prompts, **kw),
                 dict(bias_ids=ids, bias=bias), dict(allowed=allowed),
                 dict(repetition=1.3, frequency=fq, presence=-0.2, prompt_lengths=prompts, bias_ids=ids, bias=bias, allowed=allowed, **kw),
                 dict(tokens=tokens, repetition=1.0 / 3), dict()):
        want, mag = logits64(x, case.get("tokens"), case.get("lengths"), case.get("prompt_lengths"), case.get("repetition"),
                             case.get("frequency"), case.get("presence"), case.get("bias_ids"), case.get("bias"), case.get("allowed"))
        y = nat.logits_process(x, **case)
        # 1/r, the product, g*f + p, two sums: 6 half steps of the largest intermediate; what nothing touches is equal
        close(y, want, half(dtype), 6 * U32 * mag)
        same = (want == x.double())
        assert torch.equal(y[same], x[same])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_each_is_generates_loop(nat, dtype):
    """Per occurrence, with a rounding each: bit for bit the loop over the tokens."""
    B, V, L, r = 3, 500, 60, 1.17
    g = gen(31)
    x = (3 * torch.randn(B, V, device=DEV, generator=g)).to(dtype)
    tokens = torch.randint(0, 25, (B, L), device=DEV, generator=g)
    want = x.clone()
    for b in range(B):
        for tok in tokens[b].tolist():
            v = want[b, tok]
            want[b, tok] = v / r if v > 0 else v * r
    assert torch.equal(nat.logits_process(x, tokens=tokens, repetition=r, each=True), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_layouts_and_not_finite(nat, dtype):
    B, V, L = 4, 1003, 20
    g = gen(32)
    full = (3 * torch.randn(B, 2, V + 5, device=DEV, generator=g)).to(dtype)
    x = full[:, 1, 2:V + 2]                                     # the last position of a longer output, at an odd offset
    x[0, 3], x[1, 4], x[2, 5], x[3, 6] = float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min
    tokens = torch.randint(0, 30, (B, L), device=DEV, generator=g)
    tokens[:, :4] = torch.tensor([3, 4, 5, 6], device=DEV)
    mask = torch.ones(B, V, device=DEV, dtype=torch.bool)
    mask[0, 3] = mask[3, 6] = False                             # a masked NaN and a masked lowest value
    kw = dict(tokens=tokens, repetition=2.0, frequency=0.25, allowed=nat.pack_allowed(mask))
    want = nat.logits_process(x.contiguous(), **kw)
    ref, mag = logits64(x, tokens, None, None, 2.0, 0.25, None, None, None, nat.pack_allowed(mask))
    ref = ref.clamp(min=-math.inf)
    lowest = torch.finfo(dtype).min
    assert want[0, 3] == -math.inf and want[3, 6] == -math.inf and want[1, 4] == math.inf and want[2, 5] == -math.inf
    fin = ref.isfinite() & (ref.abs() < -lowest)
    close(want[fin], ref[fin], half(dtype), (6 * U32 * mag)[fin])
    assert torch.equal(nat.logits_process(x, **kw), want)
    rest = full.clone()
    got = nat.logits_process(x, out=x, **kw)                    # in place
    assert got.data_ptr() == x.data_ptr() and torch.equal(x, want)
    assert torch.equal(full[:, 0], rest[:, 0]) and torch.equal(full[:, 1, :2], rest[:, 1, :2]) and torch.equal(full[:, 1, V + 2:], rest[:, 1, V + 2:])
    one = nat.pack_allowed(mask[:1])                            # one grammar for the batch
    assert torch.equal(nat.logits_process(want, allowed=one), nat.logits_process(want, allowed=one.expand(B, -1).contiguous()))
    wide = torch.randint(0, V, (L, B), device=DEV, generator=g).t()
    assert torch.equal(nat.logits_process(want, tokens=wide, repetition=1.5), nat.logits_process(want, tokens=wide.contiguous(), repetition=1.5))


def test_logits_graph_and_stream(nat):
    B, V, L = 2, 4000, 64
    x = torch.randn(B, V, device=DEV, generator=gen(33)).to(BF16)
    tokens = torch.randint(0, V, (B, L), device=DEV, generator=gen(34))
    n = torch.tensor([10, 64], device=DEV, dtype=torch.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = nat.logits_process(x, tokens=tokens, lengths=n, repetition=1.4)
    for _ in range(3):
        n += torch.tensor([7, -9], device=DEV, dtype=torch.int32)
        g.replay()
        assert torch.equal(y, nat.logits_process(x, tokens=tokens, lengths=n, repetition=1.4))


def test_logits_refusals(nat):
    x, t = torch.zeros(2, 100, device=DEV), torch.zeros(2, 5, device=DEV, dtype=torch.int64)
    n = torch.zeros(2, device=DEV, dtype=torch.int32)
    ids = torch.zeros(2, 3, device=DEV, dtype=torch.int64)
    for bad in (dict(logits=x[0]), dict(tokens=t[:1]), dict(tokens=None, lengths=n), dict(lengths=n[:1]), dict(repetition=0.0),
                dict(repetition=-1.0), dict(repetition=math.inf), dict(repetition=torch.ones(3, device=DEV)), dict(bias_ids=ids),
                dict(bias_ids=ids, bias=torch.zeros(2, 2, device=DEV)), dict(allowed=torch.zeros(2, 3, device=DEV, dtype=torch.int32)),
                dict(allowed=torch.zeros(2, 100, device=DEV, dtype=torch.bool)), dict(each=True, prompt_lengths=n),
                dict(out=x.double()), dict(out=x[:1].expand(2, 100))):
        with pytest.raises(ValueError):
            nat.logits_process(**{**dict(logits=x, tokens=t), **bad})
    with pytest.raises(TypeError):
        nat.logits_process(x.half())
    with pytest.raises(TypeError):
        nat.logits_process(x, tokens=t.float())
    with pytest.raises(RuntimeError, match="no backward"):
        nat.logits_process(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.logits_process(x, tokens=t.cpu())
    assert nat.logits_process(x[:0]).shape == (0, 100)
