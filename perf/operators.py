"""What one step of generation with an attention memory is made of, as cases that can be timed and checked.

Four operators, in the order a step uses them: rotary positions on q and k, new keys and values into a
paged cache of 8-bit codes with a scale for each page and head, attention of the new tokens over that
cache, and penalties, biases and grammar masks on the logits.  ``run`` computes them in plain torch
operations, or, where ``own`` is true, through ``neuratensor_b200.native``.
"""
import math

import torch

own = False


DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TOP = 448.0                 # the largest e4m3 value
SMALLEST = 2.0 ** -126      # the smallest scale of a block


# --------------------------------------------------------------------------------------------------- #
#  Cases                                                                                              #
# --------------------------------------------------------------------------------------------------- #

def listed():
    return [
        # q|k of one token for each of 64 streams of the large preset (16 heads of 128), every stream at its own position
        dict(name="rotary-step", op="rotary", type="bf16", B=64, T=1, heads=32, dim=128, part=128, layout="half",
             first=8192, scale=1.0, view=True, grad=False),
        # q|k of a prompt of the small preset (10 heads of 64), read where the qkv projection left them
        dict(name="rotary-prompt", op="rotary", type="bf16", B=8, T=2048, heads=20, dim=64, part=64, layout="half",
             first=0, scale=1.0, view=True, grad=False),
        # a long document at far positions, half of each head rotated in neighbouring pairs, stretched frequencies, with the gradient
        dict(name="rotary-long", op="rotary", type="f32", B=1, T=32767, heads=24, dim=128, part=64, layout="interleaved",
             first=100000, scale=8.0, view=False, grad=True),
        # one new token for each of 64 streams of the large preset, anywhere in its page
        dict(name="append-step", op="append", type="bf16", B=64, T=1, kv=16, dim=128, page=32, longest=8704, ragged=False),
        # eight ragged prompts of the large preset at once, k and v read where the qkv projection left them
        dict(name="append-prompt", op="append", type="bf16", B=8, T=8192, kv=16, dim=128, page=32, longest=8704, ragged=True),
        # one stream of the small preset shortly after its prompt: latency alone
        dict(name="attention-one", op="attention", type="bf16", B=1, T=1, kv=10, group=1, dim=64, page=16, longest=300,
             window=256, ragged=False),
        # a step of 64 streams of the large preset behind an 8192-token prompt, window 512
        dict(name="attention-step", op="attention", type="bf16", B=64, T=1, kv=16, group=1, dim=128, page=32, longest=8704,
             window=512, ragged=False),
        # a step over long ragged caches without a window, four query heads on each cached head
        dict(name="attention-long", op="attention", type="bf16", B=8, T=1, kv=8, group=4, dim=128, page=64, longest=65536,
             window=-1, ragged=True),
        # a ragged batch that checks drafts of up to five tokens in 32 bits, idle slots among them
        dict(name="attention-draft", op="attention", type="f32", B=24, T=5, kv=10, group=1, dim=64, page=16, longest=2048,
             window=1001, ragged=True),
        # one stream of the presets' vocabulary with a short history and the repetition penalty alone
        dict(name="logits-one", op="logits", type="bf16", B=1, vocab=32000, history=40, biases=0, mask=False, all=False),
        # 64 streams behind an 8192-token prompt and 512 new tokens, every kind of penalty, bias and mask
        dict(name="logits-step", op="logits", type="bf16", B=64, vocab=32000, history=8704, biases=64, mask=True, all=True),
        # a large batch over a large vocabulary in 32 bits
        dict(name="logits-large", op="logits", type="f32", B=250, vocab=131072, history=4000, biases=300, mask=True, all=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "logits"])
    kind = rng.choice(["bf16", "bf16", "f32"])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64])
    if op == "rotary":
        tokens, heads = _log(rng, 1, 32768), _log(rng, 1, 40)
        tokens = max(1, min(tokens, 700000 // heads))
        B = rng.choice([b for b in (1, 2, 3, 8, 24, 64) if b <= tokens])
        part = rng.choice([dim, dim, dim // 2, dim // 4, dim - 6])
        return dict(op=op, type=kind, B=B, T=max(1, tokens // B), heads=heads, dim=dim, part=part,
                    layout=rng.choice(["half", "interleaved"]), first=rng.choice([0, 0, 5000, 100000, 3000000]),
                    scale=rng.choice([1.0, 2.5, 8.0]), view=rng.random() < 0.5, grad=rng.random() < 0.4)
    if op == "append":
        kv, tokens = _log(rng, 1, 32), _log(rng, 1, 32768)
        B = rng.choice([b for b in (1, 2, 5, 8, 17, 64) if b <= tokens])
        T = max(1, tokens // B)
        return dict(op=op, type=kind, B=B, T=T, kv=kv, dim=dim, page=page, longest=T + _log(rng, 1, 2000),
                    ragged=rng.random() < 0.6)
    if op == "attention":
        group, kv = rng.choice([1, 1, 2, 4, 7, 8]), _log(rng, 1, 16)
        longest = _log(rng, 1, 65536)
        B = max(1, min(_log(rng, 1, 64), 4000000 // (longest * kv)))
        T = min(longest, rng.choice([1, 1, 1, 2, 3, 5, 8]))
        return dict(op=op, type=kind, B=B, T=T, kv=kv, group=group, dim=dim, page=page, longest=longest,
                    window=rng.choice([-1, -1, 0, 256, 512, 1001]), ragged=rng.random() < 0.7)
    vocab = rng.choice([32000, 131072, 50001, _log(rng, 1000, 131072)])
    return dict(op=op, type=kind, B=max(1, min(_log(rng, 1, 256), 32000000 // vocab)), vocab=vocab,
                history=rng.choice([0, _log(rng, 1, 8704)]), biases=rng.choice([0, _log(rng, 1, 300)]),
                mask=rng.random() < 0.6, all=rng.random() < 0.7)


# --------------------------------------------------------------------------------------------------- #
#  Inputs                                                                                             #
# --------------------------------------------------------------------------------------------------- #

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV)


def _lengths(g, case):
    """Tokens in the cache after this call and how many of them are new, for each sequence."""
    B, T, longest = case["B"], case["T"], case["longest"]
    if case["ragged"]:
        counts = _randint(g, 1, T + 1, B)
        counts[0] = T
        if B > 4:
            counts[B // 2] = 0                       # an idle slot of the batch
        spread = torch.rand(B, generator=g, device=DEV)
        spread[0] = 1.0                              # and one sequence as long as it gets
        lengths = torch.maximum((spread * longest).long(), counts)
    else:
        counts = torch.full((B,), T, device=DEV)
        lengths = _randint(g, max(T, longest - longest // 16), longest + 1, B)
    return lengths.int(), counts.int()


def _channels(g, *shape):
    """Keys and values as a trained projection leaves them: some channels much larger than others."""
    x = _randn(g, *shape)
    return x.mul_(torch.exp(0.7 * _randn(g, *shape[-2:])))


def _pool(g, case):
    """A pool of pages in use: codes of random keys and values, each page and head with its own scale, the pages of a sequence anywhere."""
    B, kv, P, D = case["B"], case["kv"], case["page"], case["dim"]
    wide = (case["longest"] + case["T"] + P - 1) // P + 1
    n = B * wide + 3
    sides = []
    for _ in range(2):
        codes = torch.empty(n, kv, P, D, device=DEV, dtype=torch.float8_e4m3fn)
        scale = torch.empty(n, kv, device=DEV)
        for a in range(0, n, 4096):
            x = _randn(g, min(4096, n - a), kv, P, D).mul_(torch.exp(0.5 * _randn(g, kv, 1, D)))
            s = _block_scale(x.abs().amax((2, 3)))
            codes[a:a + 4096] = (x / s[:, :, None, None]).to(torch.float8_e4m3fn)
            scale[a:a + 4096] = s
        sides.append((codes, scale))
    table = torch.randperm(n, generator=g, device=DEV)[:B * wide].view(B, wide).int()
    return sides, table


def prepare(case, seed):
    g = _gen(seed)
    t = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "rotary":
        B, T, H, D, R = (case[k] for k in ("B", "T", "heads", "dim", "part"))
        if case["view"]:                              # columns of a wider projection, as q|k lie in q|k|v
            s["x"] = _randn(g, B, T, H + (H + 1) // 2, D).to(t)[:, :, :H]
        else:
            s["x"] = _randn(g, B, T, H, D).to(t)
        s["positions"] = case["first"] + (_randint(g, 0, 512, B, 1) + torch.arange(T, device=DEV))
        i = torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R
        f = 10000.0 ** -i
        ramp = ((i * R / 2 - R / 8) / (R / 4)).clamp(0, 1)      # slow dimensions stretched, fast ones kept
        s["inv_freq"] = (f * (1 - ramp) + f / case["scale"] * ramp).float()
        s["mscale"] = 1.0 + 0.1 * math.log(case["scale"])
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = _randn(g, B, T, H, D).to(t)
    elif case["op"] == "append":
        B, T, kv, D = (case[k] for k in ("B", "T", "kv", "dim"))
        qkv = _channels(g, B, T, 3 * kv, D).to(t)
        s["k"], s["v"] = qkv[:, :, kv:2 * kv], qkv[:, :, 2 * kv:]
        s["lengths"], s["counts"] = _lengths(g, case)
        s["sides"], s["table"] = _pool(g, case)
    elif case["op"] == "attention":
        s["lengths"], s["counts"] = _lengths(g, case)
        s["sides"], s["table"] = _pool(g, case)
        s["q"] = (1.5 * _randn(g, case["B"], case["T"], case["kv"] * case["group"], case["dim"])).to(t)
    else:
        B, V, L = case["B"], case["vocab"], case["history"]
        s["logits"] = (2.5 * _randn(g, B, V)).to(t)
        s["tokens"] = (V * torch.rand(B, L, generator=g, device=DEV) ** 3).long().clamp_(0, V - 1)   # few tokens make most of a text
        s["lengths"] = _randint(g, L // 2, L + 1, B).int()
        s["prompts"] = (s["lengths"] * torch.rand(B, generator=g, device=DEV)).int()
        s["repetition"] = 1.0 + 0.5 * torch.rand(B, generator=g, device=DEV)
        if case["all"]:
            s["frequency"] = 0.3 * torch.rand(B, generator=g, device=DEV)
            s["presence"] = torch.rand(B, generator=g, device=DEV) - 0.3
        if case["biases"]:
            s["bias_ids"] = _randint(g, 0, V, B, case["biases"])
            s["bias_ids"][:, case["biases"] // 2 + 1:] = -1          # requests have fewer than the widest
            s["bias"] = 4 * _randn(g, B, case["biases"])
        if case["mask"]:
            words = _randint(g, -2 ** 31, 2 ** 31, B, (V + 31) // 32) & _randint(g, -2 ** 31, 2 ** 31, B, (V + 31) // 32)
            words[::3] = -1                                          # a third of the requests has no grammar
            s["allowed"] = words.int()
    return s


# --------------------------------------------------------------------------------------------------- #
#  The operators: plain forms, and the framework's calls                                              #
# --------------------------------------------------------------------------------------------------- #

def run(s):
    return {"rotary": _rotary, "append": _append, "attention": _attention, "logits": _logits}[s["case"]["op"]](s)


def _pairs(y, R, layout):
    return (y[..., :R // 2], y[..., R // 2:R]) if layout == "half" else (y[..., 0:R:2], y[..., 1:R:2])


def _rotate(x, cos, sin, R, layout):
    x1, x2 = (a.float() for a in _pairs(x, R, layout))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y1, y2 = _pairs(y, R, layout)
    y1.copy_(x1 * cos - x2 * sin)
    y2.copy_(x2 * cos + x1 * sin)
    y[..., R:] = x[..., R:]
    return y


def _rotary(s):
    case = s["case"]
    if own:
        from neuratensor_b200 import native
        y = native.rotary(s["x"], s["positions"], s["inv_freq"], layout=case["layout"], mscale=s["mscale"])
        return (y, torch.autograd.grad(y, s["x"], s["dy"])[0]) if case["grad"] else y
    x = s["x"].detach()
    angle = s["positions"].double()[..., None, None] * s["inv_freq"].double()
    cos, sin = (s["mscale"] * angle.cos()).float(), (s["mscale"] * angle.sin()).float()
    y = _rotate(x, cos, sin, case["part"], case["layout"])
    return (y, _rotate(s["dy"], cos, -sin, case["part"], case["layout"])) if case["grad"] else y


def _block_scale(amax):
    """The smallest power of two that brings `amax` to 448 or below, 2^-126 at least."""
    m, e = torch.frexp(amax)
    e = (e - 9 + (m > 0.875)).clamp(-126, 127)
    e = torch.where(amax > 0, e, -126)
    return ((e + 127).int() << 23).view(torch.float32)


def _append(s):
    (kc, ks), (vc, vs) = s["sides"]
    if own:
        from neuratensor_b200 import native
        native.kv_append(s["k"], s["v"], kc, ks, vc, vs, s["table"], s["lengths"], counts=s["counts"])
        return kc, ks, vc, vs
    P, T = s["case"]["page"], s["case"]["T"]
    lengths, counts = s["lengths"].long(), s["counts"].long()
    start = lengths - counts
    blocks = start[:, None] // P + torch.arange((T + P - 2) // P + 1, device=start.device)
    here = (blocks * P < lengths[:, None]) & (counts > 0)[:, None]
    pages = s["table"].long().gather(1, blocks.clamp(max=s["table"].shape[1] - 1))
    at = blocks[..., None] * P + torch.arange(P, device=start.device)          # [B, blocks, P] positions
    row = at - start[:, None, None]
    new = ((row >= 0) & (row < counts[:, None, None]))[..., None, None]
    old = (here[..., None] & (row < 0))[..., None, None]
    seq = torch.arange(start.numel(), device=start.device)[:, None, None]
    _write(s["k"], kc, ks, pages, seq, row.clamp(0, T - 1), new, old)
    _write(s["v"], vc, vs, pages, seq, row.clamp(0, T - 1), new, old)
    return kc, ks, vc, vs


def _write(x, codes, scale, pages, seq, row, new, old):
    x = x[seq, row].float()                                                     # [B, blocks, P, heads, D]
    amax = torch.where(new & x.isfinite(), x.abs(), 0.0).amax((2, 4))
    before = scale[pages]                                                       # [B, blocks, heads]
    now = torch.maximum(_block_scale(amax), torch.where(old.any(2)[..., 0], before, SMALLEST))
    held = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float().transpose(2, 3)
    kept = torch.where(old, held * (before / now)[:, :, None, :, None], held)
    fresh = (x / now[:, :, None, :, None]).clamp(-TOP, TOP)
    out = torch.where(new, fresh, kept).to(torch.float8_e4m3fn).transpose(2, 3).contiguous()
    codes.view(torch.uint8)[pages] = out.view(torch.uint8)
    scale[pages] = torch.where(new.any(2)[..., 0], now, before)


def _attention(s):
    (kc, ks), (vc, vs) = s["sides"]
    case = s["case"]
    window = case["window"]
    if own:
        from neuratensor_b200 import native
        return native.kv_attention(s["q"], kc, ks, vc, vs, s["table"], s["lengths"], counts=s["counts"],
                                   window=window if window >= 0 else None)
    B, T, kv, G, D, P = (case[k] for k in ("B", "T", "kv", "group", "dim", "page"))
    lengths, counts = s["lengths"].long(), s["counts"].long()
    span = case["longest"] if window < 0 else min(case["longest"], window + T)
    at = lengths[:, None] - span + torch.arange(span, device=DEV)               # the last `span` positions
    block = at.clamp(min=0) // P
    page = s["table"].long().gather(1, block)
    slot = at.clamp(min=0) % P
    k = kc.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float().mul_(ks[page][..., None])
    v = vc.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float().mul_(vs[page][..., None])
    pos = (lengths - counts)[:, None] + torch.arange(T, device=DEV)
    see = (at[:, None] >= 0) & (at[:, None] <= pos[..., None]) & (torch.arange(T, device=DEV) < counts[:, None])[..., None]
    if window >= 0:
        see &= at[:, None] >= pos[..., None] - window
    see = see[:, None, :, None]                                                 # [B, 1, T, 1, span]
    q = s["q"].float().view(B, T, kv, G, D).transpose(1, 2).reshape(B, kv, T * G, D)
    w = (q @ k.permute(0, 2, 3, 1)).view(B, kv, T, G, span).mul_(1.0 / math.sqrt(D))
    w = torch.where(see, w, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    o = w.view(B, kv, T * G, span) @ v.transpose(1, 2)
    o = o.view(B, kv, T, G, D) / torch.where(total > 0, total, 1.0)
    return o.transpose(1, 2).reshape(B, T, kv * G, D).to(s["q"].dtype)


def _logits(s):
    if own:
        from neuratensor_b200 import native
        return native.logits_process(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                                     repetition=s["repetition"], frequency=s.get("frequency"), presence=s.get("presence"),
                                     bias_ids=s.get("bias_ids"), bias=s.get("bias"), allowed=s.get("allowed"))
    x = s["logits"].float()
    B, V = x.shape
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    live = at < s["lengths"][:, None]
    made = live & (at >= s["prompts"][:, None])
    seen = torch.zeros(B, V, device=x.device).scatter_add_(1, s["tokens"], live.float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    if "frequency" in s:
        times = torch.zeros(B, V, device=x.device).scatter_add_(1, s["tokens"], made.float())
        x = x - (s["frequency"][:, None] * times + s["presence"][:, None] * (times > 0))
    if "bias" in s:                                                             # of equal ids the last one holds
        ids = s["bias_ids"]
        order = torch.arange(1, ids.shape[1] + 1, device=x.device).expand(B, -1)
        last = torch.zeros(B, V + 1, device=x.device, dtype=torch.int64)
        last.scatter_reduce_(1, torch.where(ids < 0, V, ids), order, "amax")
        last = last[:, :V]
        x = torch.where(last > 0, x + s["bias"].gather(1, (last - 1).clamp(min=0)), x)
    if "allowed" in s:
        bit = (s["allowed"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bit.view(B, -1)[:, :V] != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


# --------------------------------------------------------------------------------------------------- #
#  What a pass cannot do without                                                                      #
# --------------------------------------------------------------------------------------------------- #

def _seen(case):
    """Keys that the rows of one sequence read, over the batch, as the lengths are drawn on average."""
    longest, T, window = case["longest"], case["T"], case["window"]
    reach = longest if window < 0 else min(longest, window + T)
    if not case["ragged"]:
        return case["B"] * reach
    mean = longest / 2 if window < 0 else reach * (1 - reach / (2 * longest))
    return int(reach + (case["B"] - 1) * mean)


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "rotary":
        n = case["B"] * case["T"] * case["heads"]
        once = 2 * n * case["dim"] * size + case["B"] * case["T"] * 8
        return {"bytes": once * (2 if case["grad"] else 1), "flops": 3 * n * case["part"] * (2 if case["grad"] else 1)}
    if case["op"] == "append":
        n = int(case["B"] * case["T"] * (0.5 if case["ragged"] and case["T"] > 1 else 1.0)) * case["kv"] * case["dim"] * 2
        return {"bytes": n * (size + 1), "flops": 3 * n}
    if case["op"] == "attention":
        keys = _seen(case) * case["kv"]
        rows = case["B"] * case["T"] * case["kv"] * case["group"]
        return {"bytes": int(2 * keys * case["dim"] * (1 + 4 / (case["page"] * case["dim"]))) + 2 * rows * case["dim"] * size,
                "flops": 4 * keys * case["group"] * case["T"] * case["dim"]}
    n = case["B"] * case["vocab"]
    return {"bytes": 2 * n * size + (n // 8 if case["mask"] else 0) + case["B"] * (6 * case["history"] + 12 * case["biases"]),
            "flops": n * (6 if case["all"] else 2)}


# --------------------------------------------------------------------------------------------------- #
#  The definitions in 64 bits                                                                         #
# --------------------------------------------------------------------------------------------------- #

def exact(case, seed):
    if case["op"] == "append" and case["B"] * case["T"] * case["kv"] > 1 << 17:
        return None                                   # its blocks are walked one by one here
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](s, case)


def _exact_rotary(s, case):
    """Each pair as a complex number times m e^(i a)."""
    R, H = case["part"], case["heads"]
    angle = s["positions"].double()[:, :, None] * s["inv_freq"].double()
    turn = torch.polar(torch.full_like(angle, s["mscale"]), angle)[:, :, None]

    def by(x, turn):
        x = x.detach().double()
        head = x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else x[..., :R].unflatten(-1, (R // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
        y = y.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else y.flatten(-2)
        return torch.cat([y, x[..., R:]], -1)

    y = by(s["x"], turn)
    return (y, by(s["dy"], turn.conj())) if case["grad"] else y


def _exact_append(s, case):
    """Block by block: the scale by its exponent, the codes as the nearest of the 8-bit values."""
    P = case["page"]
    out = []
    lengths, counts, table = s["lengths"].tolist(), s["counts"].tolist(), s["table"].tolist()
    grid = torch.arange(256, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = grid[grid.isfinite()].sort().values
    mid = (grid[1:] + grid[:-1]) / 2
    powers = torch.tensor([2.0 ** e for e in range(-126, 128)], device=DEV, dtype=torch.float64)

    def nearest(y):
        y = y.clamp(-TOP, TOP)
        i = torch.searchsorted(mid, y.contiguous())
        tie = (i < mid.numel()) & (mid[i.clamp(max=mid.numel() - 1)] == y)
        low, high = grid[i], grid[(i + 1).clamp(max=grid.numel() - 1)]
        odd = lambda g: (g.to(torch.float8_e4m3fn).view(torch.uint8) & 1) == 1    # noqa: E731
        return torch.where(tie & odd(low), high, low)

    for x, (codes, scale) in zip((s["k"], s["v"]), s["sides"]):
        values, scales = codes.double(), scale.double()
        for b in range(case["B"]):
            first = lengths[b] - counts[b]
            for blk in range(first // P, (lengths[b] + P - 1) // P if counts[b] else 0):
                lo, hi = max(first, blk * P), min(lengths[b], (blk + 1) * P)
                if hi <= lo:
                    continue
                page = table[b][blk]
                y = x[b, lo - first:hi - first].double().transpose(0, 1)         # [heads, new, D]
                top = y.abs().amax((1, 2))
                now = powers[torch.searchsorted(TOP * powers, top.contiguous())]
                held = lo - blk * P
                if held > 0:
                    before = scales[page]
                    now = torch.maximum(now, before)
                    values[page, :, :held] = nearest(values[page, :, :held] * (before / now)[:, None, None])
                values[page, :, held:held + hi - lo] = nearest(y / now[:, None, None])
                scales[page] = now
        out += [values, scales]
    return tuple(out)


def _exact_attention(s, case):
    """Sequence by sequence over its own keys."""
    (kc, ks), (vc, vs) = s["sides"]
    P, T, kv, G, D, window = (case[k] for k in ("page", "T", "kv", "group", "dim", "window"))
    out = torch.zeros(case["B"], T, kv * G, D, device=DEV, dtype=torch.float64)
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        if not c:
            continue
        pages = s["table"][b, :(n + P - 1) // P].long()
        low = 0 if window < 0 else max(0, n - c - window)
        pages, base = pages[low // P:], low // P * P
        both = []
        for codes, scale in ((kc, ks), (vc, vs)):
            y = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * scale.double()[pages][:, :, None, None]
            both.append(y.transpose(0, 1).reshape(kv, -1, D)[:, :n - base])
        k, v = both
        at = base + torch.arange(n - base, device=DEV)
        for t in range(c):
            p = n - c + t
            keep = at <= p if window < 0 else (at <= p) & (at >= p - window)
            q = s["q"][b, t].double().view(kv, G, D)
            w = torch.einsum("hgd,hjd->hgj", q, k[:, keep]) / math.sqrt(D)
            out[b, t] = torch.einsum("hgj,hjd->hgd", torch.softmax(w, -1), v[:, keep]).reshape(kv * G, D)
    return out


def _exact_logits(s, case):
    x = s["logits"].double()
    B, V = x.shape
    for b in range(B):
        n, p = int(s["lengths"][b]), int(s["prompts"][b])
        row = x[b]
        seen = torch.bincount(s["tokens"][b, :n], minlength=V) > 0
        r = s["repetition"][b].double()
        row = torch.where(seen, torch.where(row > 0, row / r, row * r), row)
        if case["all"]:
            times = torch.bincount(s["tokens"][b, p:n], minlength=V).double()
            row = row - s["frequency"][b].double() * times - s["presence"][b].double() * (times > 0)
        if case["biases"]:
            held = {i: j for j, i in enumerate(s["bias_ids"][b].tolist()) if i >= 0}
            if held:
                row[torch.tensor(list(held), device=DEV)] += s["bias"][b].double()[torch.tensor(list(held.values()), device=DEV)]
        if case["mask"]:
            word = s["allowed"][b].long()[torch.arange(V, device=DEV) // 32]
            row = torch.where((word >> (torch.arange(V, device=DEV) % 32)) & 1 == 1, row, -math.inf)
        x[b] = row
    return x
