"""What a step of a beam search over a paged attention memory is made of, as cases that can be timed and checked.

Four operators, in the order a step uses them: the choice of the best continuations over beams and vocabulary,
the block states moved to the chosen beams, the pages of the attention cache forked for them (with the copies that
this takes), and attention in which the beams of a prompt read the prefix that they share once.  ``run`` computes
them in plain torch operations, or, where ``own`` is true, through ``neuratensor_b200.native``.
"""
import math

import torch

own = False


DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------------- #
#  Cases                                                                                              #
# --------------------------------------------------------------------------------------------------- #

def listed():
    return [
        # the four beams of one prompt over the presets' vocabulary: latency
        dict(name="select-one", op="select", type="bf16", B=1, K=4, n=4, vocab=32000, alpha=0.0, finished=False, stay=False),
        # four beams for each of 16 prompts, some finished, ranked by length, children in their parents' slots
        dict(name="select-step", op="select", type="bf16", B=16, K=4, n=4, vocab=32000, alpha=0.7, finished=True, stay=True),
        # twice as many candidates as beams, wide beams over a large vocabulary in 32 bits
        dict(name="select-large", op="select", type="f32", B=16, K=16, n=32, vocab=131072, alpha=0.0, finished=False, stay=False),
        # membranes and states of the small preset's 12 blocks for the beams of one prompt
        dict(name="reorder-one", op="reorder", type="bf16", B=1, K=4, keep=3, blocks=12, inner=1280, states=32),
        # those of the large preset's 28 blocks for 16 prompts of four beams, of which one in four gives way
        dict(name="reorder-step", op="reorder", type="bf16", B=16, K=4, keep=3, blocks=28, inner=4096, states=128),
        # in 32 bits, eight beams of which half give way, rows of an odd length
        dict(name="reorder-odd", op="reorder", type="f32", B=5, K=8, keep=4, blocks=20, inner=1153, states=17),
        # the small preset's two attention layers, one prompt of four beams, a window of 256
        dict(name="fork-one", op="fork", B=1, K=4, keep=3, layers=2, kv=10, dim=64, page=32, longest=300, window=256, tokens=1),
        # the large preset's four attention layers, 16 prompts of four beams behind 8192 tokens, window 512
        dict(name="fork-step", op="fork", B=16, K=4, keep=3, layers=4, kv=16, dim=128, page=32, longest=8704, window=512, tokens=1),
        # 64 samples of each of four long prompts without a window, eight heads; drafts of five tokens
        dict(name="fork-long", op="fork", B=4, K=64, keep=40, layers=1, kv=8, dim=128, page=64, longest=40000, window=-1, tokens=5),
        # the beams of one prompt of the small preset within its window: latency
        dict(name="shared-one", op="shared", type="bf16", groups=1, K=4, T=1, kv=10, group=1, dim=64, page=32, prefix=288, tail=40,
             window=256, ragged=False),
        # four beams for each of 16 prompts of the large preset, window 512
        dict(name="shared-step", op="shared", type="bf16", groups=16, K=4, T=1, kv=16, group=1, dim=128, page=32, prefix=8192,
             tail=128, window=512, ragged=False),
        # 64 samples that share a long prompt, four query heads on each cached head, of different lengths behind it
        dict(name="shared-long", op="shared", type="bf16", groups=1, K=64, T=1, kv=8, group=4, dim=128, page=64, prefix=65536,
             tail=600, window=-1, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "reorder", "fork", "shared", "shared"])
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "select":
        K = rng.choice([1, 2, 3, 4, 5, 8, 16, 29])
        vocab = rng.choice([32000, 131072, 50001, _log(rng, 500, 131072)])
        stay = rng.random() < 0.4
        return dict(op=op, type=kind, B=max(1, min(_log(rng, 1, 64), 32000000 // (vocab * K))), K=K,
                    n=K if stay else rng.choice([K, 2 * K, K + 1]), vocab=vocab, alpha=rng.choice([0.0, 0.6, 1.0]),
                    finished=rng.random() < 0.5, stay=stay)
    K = rng.choice([2, 3, 4, 5, 8, 16])
    if op == "reorder":
        B, inner, states = _log(rng, 1, 32), rng.choice([192, 576, 1280, 2304, 4096, 1153]), rng.choice([8, 16, 32, 64, 128, 17])
        size = 2 if kind == "bf16" else 4
        blocks = max(1, min(rng.choice([4, 6, 12, 20, 28]), 1600000000 // (B * K * inner * (states + 1) * size)))
        return dict(op=op, type=kind, B=B, K=K, keep=rng.randint(1, K), blocks=blocks, inner=inner, states=states)
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64])
    if op == "fork":
        K = rng.choice([K, K, 32, 64])
        B, kv, longest = _log(rng, 1, 16), rng.choice([4, 8, 10, 16]), _log(rng, 20, 30000)
        window = rng.choice([-1, 256, 512, 1001])
        held = B * ((longest if window < 0 else min(longest, window + page)) + 3 * K * page)
        layers = max(1, min(rng.choice([1, 2, 4]), 1500000000 // (held * kv * dim * 2)))
        return dict(op=op, B=B, K=K, keep=rng.randint(1, K), layers=layers, kv=kv, dim=dim, page=page, longest=longest, window=window,
                    tokens=rng.choice([1, 1, 1, 4, 5]))
    T = rng.choice([1, 1, 1, 2, 3, 5])
    group, kv = rng.choice([1, 1, 2, 4, 7]), _log(rng, 1, 16)
    K = max(1, min(rng.choice([K, K, 1, 24, 64]), 256 // (T * group)))
    prefix, tail = _log(rng, 1, 60000), _log(rng, T, 600)
    groups = max(1, min(_log(rng, 1, 32), 520000 // (prefix * kv), 300000 // (tail * kv * K)))
    return dict(op=op, type=kind, groups=groups, K=K, T=T, kv=kv, group=group, dim=dim, page=page, prefix=prefix, tail=tail,
                window=rng.choice([-1, -1, 0, 256, 512, 1001]), ragged=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------- #
#  Inputs                                                                                             #
# --------------------------------------------------------------------------------------------------- #

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV)


def _codes(g, n, kv, P, D):
    """Pages of random keys or values as 8-bit codes, each page and head with its own power of two."""
    codes = torch.empty(n, kv, P, D, device=DEV, dtype=torch.float8_e4m3fn)
    scale = torch.empty(n, kv, device=DEV)
    for a in range(0, n, 4096):
        x = _randn(g, min(4096, n - a), kv, P, D).mul_(torch.exp(0.5 * _randn(g, kv, 1, D)))
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448.0)))
        codes[a:a + 4096] = (x / s[:, :, None, None]).to(torch.float8_e4m3fn)
        scale[a:a + 4096] = s
    return codes, scale


def _survivors(g, B, K, keep):
    """The row that each row goes on from: `keep` beams of an item stay where they are, the others follow one of them."""
    order = torch.argsort(_rand(g, B, K), 1)
    stay, follow = order[:, :keep], _randint(g, 0, keep, B, K)
    rows = stay.gather(1, follow)
    rows.scatter_(1, stay, stay)
    return (rows + K * torch.arange(B, device=DEV)[:, None]).int()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "select":
        B, K, V = case["B"], case["K"], case["vocab"]
        s["logits"] = (2.5 * _randn(g, B * K, V)).to(TYPES[case["type"]])
        s["scores"] = -2.0 * _randint(g, 1, 40, B, 1) - 3.0 * _rand(g, B, K)
        s["lengths"] = _randint(g, 1, 400, B, 1).expand(B, K).int().contiguous()
        if case["finished"]:
            s["finished"] = _rand(g, B, K) < 0.2
            s["finished"][:, 0] = False
    elif case["op"] == "reorder":
        R, t = case["B"] * case["K"], TYPES[case["type"]]
        s["tensors"] = []
        for _ in range(case["blocks"]):
            s["tensors"].append(_randn(g, R, case["inner"]).to(t))
            s["tensors"].append(_randn(g, R, case["inner"], case["states"]).to(t))
        s["rows"] = _survivors(g, case["B"], case["K"], case["keep"]).view(-1)
    elif case["op"] == "fork":
        _prepare_fork(s, case, g)
    else:
        _prepare_shared(s, case, g)
    return s


def _prepare_fork(s, case, g):
    """Beams of B prompts some steps behind them: the pages of a prompt shared, those since their last common step their own."""
    B, K, P, longest, window, tokens = (case[k] for k in ("B", "K", "page", "longest", "window", "tokens"))
    R = B * K
    wide = (longest + tokens + P - 1) // P + 1
    lengths = (longest - _randint(g, 0, max(1, min(longest // 4, 256)), B)).clamp(min=1)
    low = (lengths - window).clamp(min=0) // P if window >= 0 else torch.zeros_like(lengths)
    have = (lengths + P - 1) // P
    block = torch.arange(wide, device=DEV)
    live = ((block >= low[:, None]) & (block < have[:, None]))[:, None].expand(B, K, wide)
    mine = live & (block >= (have - 1 - _randint(g, 0, 2, B).clamp(max=1))[:, None, None])      # the last one or two blocks
    common = (live & ~mine)[:, 0]
    held = int(common.sum()) + int(mine.sum())
    n = B * (wide if window < 0 else min(wide, window // P + 2)) + R * (4 + (tokens + P - 1) // P) + 5
    pages = torch.randperm(n, generator=g, device=DEV).int()
    table = torch.full((B, K, wide), -1, device=DEV, dtype=torch.int32)
    first = int(common.sum())
    shared = torch.full((B, wide), -1, device=DEV, dtype=torch.int32)
    shared[common] = pages[:first]
    table = torch.where(common[:, None], shared[:, None], table)
    table[mine] = pages[first:held]
    s["table"] = table.view(R, wide).contiguous()
    s["lengths"] = lengths[:, None].expand(B, K).reshape(R).int().contiguous()
    flat = s["table"][s["table"] >= 0].long()
    s["refs"] = torch.bincount(flat, minlength=n).int()
    s["rows"] = _survivors(g, B, K, case["keep"]).view(-1)
    s["layers"] = [_codes(g, n, case["kv"], P, case["dim"]) + _codes(g, n, case["kv"], P, case["dim"]) for _ in range(case["layers"])]


def _prepare_shared(s, case, g):
    G, K, T, P, prefix, tail = (case[k] for k in ("groups", "K", "T", "page", "prefix", "tail"))
    B = G * K
    shared = prefix // P * P - _randint(g, 0, prefix // P // 2 + 1 if case["ragged"] else min(2, prefix // P + 1), G) * P
    shared = shared.clamp(min=0)
    if case["ragged"]:
        behind = _randint(g, T, tail + T, G, K)
        counts = _randint(g, 1, T + 1, G, K)
        counts[0, 0] = T
        if B > 4:
            counts[G // 2, K // 2] = 0               # an idle slot of the batch
    else:
        behind = _randint(g, T, tail + T, G, 1).expand(G, K)
        counts = torch.full((G, K), T, device=DEV)
    s["shared"] = shared.int()
    s["lengths"] = (shared[:, None] + behind).reshape(B).int()
    s["counts"] = counts.reshape(B).int()
    wide = (prefix + tail + T + P - 1) // P + 1
    rear = (tail + T + P - 1) // P + 1
    n = G * (prefix // P) + B * rear + 3
    pages = torch.randperm(n, generator=g, device=DEV).int()
    front = pages[:G * (prefix // P)].view(G, 1, -1)
    own_pages = pages[G * (prefix // P):][:B * rear].view(G, K, rear)
    block = torch.arange(wide, device=DEV)
    past = block - (shared // P)[:, None]                                    # [G, wide]
    table = own_pages.gather(2, past.clamp(0, rear - 1)[:, None].expand(G, K, wide))
    if prefix // P:
        lead = front.gather(2, block.clamp(max=prefix // P - 1).expand(G, 1, wide)).expand(G, K, wide)
        table = torch.where((past < 0)[:, None], lead, table)
    s["table"] = table.reshape(B, wide).contiguous()
    s["sides"] = [_codes(g, n, case["kv"], P, case["dim"]) for _ in range(2)]
    s["q"] = (1.5 * _randn(g, B, T, case["kv"] * case["group"], case["dim"])).to(TYPES[case["type"]])


# --------------------------------------------------------------------------------------------------- #
#  The operators: plain forms, and the framework's calls                                              #
# --------------------------------------------------------------------------------------------------- #

def run(s):
    return {"select": _select, "reorder": _reorder, "fork": _fork, "shared": _shared}[s["case"]["op"]](s)


def _in_slots(rows, K):
    """Where each of an item's chosen candidates stands: the first child of a beam in the beam's slot, the others, in
    order, in the slots left."""
    B, n = rows.shape
    at = torch.arange(n, device=rows.device)
    first = (rows[:, :, None] == rows[:, None, :]).int().argmax(2) == at
    taken = ((rows[:, None, :] == at[:, None]) & first[:, None]).any(2)
    nth = (~first).cumsum(1) - 1
    free = torch.argsort(taken.int(), dim=1, stable=True)                        # free slots first, in order
    return torch.where(first, rows, free.gather(1, nth.clamp(min=0)))


def _select(s):
    case = s["case"]
    B, K, n, V = (case[k] for k in ("B", "K", "n", "vocab"))
    done = s.get("finished")
    if own:
        from neuratensor_b200 import native
        return native.beam_select(s["logits"], s["scores"], finished=done, lengths=s["lengths"], length_penalty=case["alpha"], n=n,
                                  pad=0, stay=case["stay"])
    # in 64 bits: candidates of different beams lie next to each other
    x = s["logits"].double().view(B, K, V)
    top = x.amax(2, keepdim=True)
    total = s["scores"].double()[..., None] + (x - (top + torch.log(torch.exp(x - top).sum(2, keepdim=True))))
    length = s["lengths"].double()[..., None] + 1
    if done is not None:
        alone = torch.full_like(total, -math.inf)
        alone[:, :, 0] = s["scores"].double()
        total = torch.where(done[..., None], alone, total)
        length = length - done[..., None].double()
    rank = (total / length.pow(case["alpha"])).view(B, K * V)
    total = total.view(B, K * V)
    least = torch.topk(rank, n, 1).values[:, -1:]
    above, level = rank > least, rank == least
    keep = above | (level & (level.cumsum(1) <= n - above.sum(1, keepdim=True)))     # of equal ones the first
    flat = keep.nonzero()[:, 1].view(B, n)
    flat = flat.gather(1, torch.argsort(rank.gather(1, flat), dim=1, descending=True, stable=True))
    scores, rows, tokens = total.gather(1, flat).float(), flat // V, flat % V
    if case["stay"]:
        at = _in_slots(rows, K)
        scores, rows, tokens = (torch.empty_like(t).scatter_(1, at, t) for t in (scores, rows, tokens))
    return scores, (rows + K * torch.arange(B, device=rows.device)[:, None]).int(), tokens


def _reorder(s):
    if own:
        from neuratensor_b200 import native
        native.reorder_rows(s["tensors"], s["rows"], group=s["case"]["K"])
    else:
        rows = s["rows"].long()
        for t in s["tensors"]:
            t.copy_(t[rows])
    return s["tensors"]


def _fork(s):
    case = s["case"]
    table, refs, lengths, rows = s["table"], s["refs"], s["lengths"], s["rows"]
    P, window, tokens, K = case["page"], case["window"], case["tokens"], case["K"]
    if own:
        from neuratensor_b200 import native
        copies, shared = native.kv_fork(table, refs, lengths, rows, P, tokens=tokens, window=window if window >= 0 else None, group=K)
        native.kv_copy_pages(s["layers"], copies)
        return table, refs, lengths, copies, shared, s["layers"]
    R, wide = table.shape
    parents = rows.long()
    block = torch.arange(wide, device=DEV)
    n = refs.numel()
    length = lengths[parents].long()
    low = (length - window).clamp(min=0) // P if window >= 0 else torch.zeros_like(length)
    have = (length + P - 1) // P
    live = (block >= low[:, None]) & (block < have[:, None])
    now = torch.where(live, table[parents], -1)
    count = refs.clone()
    count.scatter_add_(0, now.clamp(min=0).view(-1).long(), (now >= 0).view(-1).int())
    count.scatter_add_(0, table.clamp(min=0).view(-1).long(), -(table >= 0).view(-1).int())
    # the page that the next token is written to, where it is begun: one row may keep it when only such rows have it
    at = torch.arange(R, device=DEV)
    begun = (length % P != 0)
    tail = now.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0]
    same = begun[:, None] & begun & (tail[:, None] == tail)
    others = same.sum(1) < count[tail.clamp(min=0).long()]
    place = torch.where(parents == at, at, at + R)                           # a row that had it before the others
    keeper = torch.where(same, place, 2 * R).amin(1) == place
    copy = begun & (tail >= 0) & (others | ~keeper)
    # new pages, row by row: the copy, then the blocks of the new tokens that the window will see
    need = (length + tokens + P - 1) // P
    seen = (length + tokens - window).clamp(min=0) // P if window >= 0 else torch.zeros_like(length)
    fresh = (block >= have[:, None]) & (block < need[:, None]) & (block >= seen[:, None])
    fresh |= copy[:, None] & (block == have[:, None] - 1)
    nth = fresh.view(-1).cumsum(0) - 1
    free = torch.argsort((count > 0).int(), stable=True).int()
    given = free[nth.clamp(0, n - 1)].view(R, wide)
    out = torch.where(fresh, given, now)
    count.scatter_add_(0, torch.where(copy, tail, 0).long(), -copy.int())
    count.scatter_add_(0, torch.where(fresh, out, 0).view(-1).long(), fresh.view(-1).int())
    new_tail = out.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0]
    copies = torch.where(copy[:, None], torch.stack([tail, new_tail], 1), -1).int()
    by = out.view(-1, K, wide)
    alike = ((by == by[:, :1]).all(1).int().cumprod(1).sum(1) * P)
    shared = torch.minimum(alike, (length // P * P).view(-1, K).amin(1)).int()
    table.copy_(out)
    refs.copy_(count)
    lengths.copy_(length)
    src, dst = copies[:, 0].long(), copies[:, 1].long()
    src, dst = src[copy], dst[copy]
    for kc, ks, vc, vs in s["layers"]:
        for codes, scale in ((kc, ks), (vc, vs)):
            codes.view(torch.uint8)[dst] = codes.view(torch.uint8)[src]
            scale[dst] = scale[src]
    return table, refs, lengths, copies, shared, s["layers"]


def _values(side, page, slot=None):
    """Cached heads [..., tokens, kv, D] of whole pages [..., blocks], or of a slot of each page."""
    codes, scale = side
    if slot is not None:
        return codes.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float() * scale[page][..., None]
    y = codes.view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * scale[page][..., None, None]
    return y.transpose(-2, -3).flatten(-4, -3)


def _shared(s):
    case = s["case"]
    G, K, T, kv, gq, D, P, window = (case[k] for k in ("groups", "K", "T", "kv", "group", "dim", "page", "window"))
    key_side, value_side = s["sides"]
    if own:
        from neuratensor_b200 import native
        return native.kv_attention_shared(s["q"], *key_side, *value_side, s["table"], s["lengths"], s["shared"], counts=s["counts"],
                                          window=window if window >= 0 else None)
    B = G * K
    lengths, counts, shared = s["lengths"].long(), s["counts"].long(), s["shared"].long()
    pos = (lengths - counts)[:, None] + torch.arange(T, device=DEV)                  # [B, T]
    live = (torch.arange(T, device=DEV) < counts[:, None])[..., None]
    lowest = pos - window if window >= 0 else torch.zeros_like(pos)
    # the shared part, once for all rows of a group: the blocks that a window can reach
    wide = max(1, case["prefix"] // P)
    near = wide if window < 0 else min(wide, (window + case["tail"] + 2 * T) // P + 2)
    block = (shared // P - near)[:, None] + torch.arange(near, device=DEV)
    page = s["table"].view(G, K, -1)[:, 0].long().gather(1, block.clamp(min=0))
    at = (block[..., None] * P + torch.arange(P, device=DEV)).view(G, 1, 1, -1)
    see = (at >= 0) & (at <= pos.view(G, K, T, 1)) & (at >= lowest.view(G, K, T, 1)) & live.view(G, K, T, 1)
    k, v = _values(key_side, page), _values(value_side, page)                        # [G, near * P, kv, D]
    q = s["q"].float().view(G, K, T, kv, gq, D).permute(0, 3, 1, 2, 4, 5).reshape(G, kv, K * T * gq, D)
    w1 = (q @ k.permute(0, 2, 3, 1)).view(G, kv, K, T, gq, -1).mul_(1.0 / math.sqrt(D))
    w1 = torch.where(see[:, None, :, :, None], w1, -math.inf)
    # the rest, row by row
    span = case["tail"] + T
    at = shared.repeat_interleave(K)[:, None] + torch.arange(span, device=DEV)       # [B, span]
    page = s["table"].long().gather(1, (at // P).clamp(max=s["table"].shape[1] - 1))
    k2, v2 = _values(key_side, page, at % P), _values(value_side, page, at % P)
    see = (at[:, None] <= pos[..., None]) & (at[:, None] >= lowest[..., None]) & live
    q2 = s["q"].float().view(B, T, kv, gq, D).transpose(1, 2).reshape(B, kv, T * gq, D)
    w2 = (q2 @ k2.permute(0, 2, 3, 1)).view(B, kv, T, gq, span).mul_(1.0 / math.sqrt(D))
    w2 = torch.where(see[:, None, :, None], w2, -math.inf)
    w2 = w2.view(G, K, kv, T, gq, span).transpose(1, 2)
    top = torch.maximum(w1.amax(-1, keepdim=True), w2.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    w1, w2 = torch.exp(w1 - top), torch.exp(w2 - top)
    total = w1.sum(-1, keepdim=True) + w2.sum(-1, keepdim=True)
    o = (w1.view(G, kv, K * T * gq, -1) @ v.transpose(1, 2)).view(G, kv, K, T, gq, D)
    o = o + (w2.transpose(1, 2).reshape(B, kv, T * gq, span) @ v2.transpose(1, 2)).view(G, K, kv, T, gq, D).transpose(1, 2)
    o = o / torch.where(total > 0, total, 1.0)
    return o.permute(0, 2, 3, 1, 4, 5).reshape(B, T, kv * gq, D).to(s["q"].dtype)


# --------------------------------------------------------------------------------------------------- #
#  What a pass cannot do without                                                                      #
# --------------------------------------------------------------------------------------------------- #

def work(case):
    if case["op"] == "select":
        rows = case["B"] * case["K"] * (0.8 if case["finished"] else 1.0)
        n = int(rows * case["vocab"])
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + case["B"] * (case["K"] * 9 + case["n"] * 16), "flops": 4 * n}
    if case["op"] == "reorder":
        row = case["blocks"] * case["inner"] * (case["states"] + 1) * (2 if case["type"] == "bf16" else 4)
        K, keep = case["K"], case["keep"]
        # each row that gives way is written; a beam that someone follows is read
        followed = keep * (1 - (1 - 1 / keep) ** (K - keep))
        return {"bytes": int(case["B"] * row * (K - keep + followed)), "flops": 0}
    if case["op"] == "fork":
        K, keep, P = case["K"], case["keep"], case["page"]
        R = case["B"] * K
        followed = keep * (1 - (1 - 1 / keep) ** (K - keep))
        side = case["kv"] * (P * case["dim"] + 4)
        wide = (case["longest"] + case["tokens"] + P - 1) // P + 1
        return {"bytes": int(case["B"] * (K - keep + followed) * 2 * side * case["layers"] * (P - 1) / P) + 2 * 4 * R * wide, "flops": 0}
    G, K, T, kv, gq, D, P, window = (case[k] for k in ("groups", "K", "T", "kv", "group", "dim", "page", "window"))
    prefix, tail = case["prefix"] * (0.75 if case["ragged"] else 1.0), case["tail"] / 2 + T
    if window >= 0:
        tail = min(tail, window + T)
        prefix = min(prefix, max(0, window + T - tail))
    keys, rows = G * kv * (prefix + K * tail), G * K * T * kv * gq
    size = 2 if case["type"] == "bf16" else 4
    return {"bytes": int(2 * keys * D * (1 + 4 / (P * D))) + 2 * rows * D * size, "flops": int(4 * rows * (prefix + tail) * D)}


# --------------------------------------------------------------------------------------------------- #
#  The definitions in 64 bits                                                                         #
# --------------------------------------------------------------------------------------------------- #

def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "fork": _exact_fork, "shared": _exact_shared}[case["op"]](s, case)


def _exact_select(s, case):
    """Item by item: the candidates of each beam in order, merged on the host."""
    B, K, n, V, alpha = (case[k] for k in ("B", "K", "n", "vocab", "alpha"))
    out = [[], [], []]
    for b in range(B):
        found = []
        for k in range(K):
            score, length = float(s["scores"][b, k]), int(s["lengths"][b, k])
            if "finished" in s and bool(s["finished"][b, k]):
                found.append((score / length ** alpha, k, 0, score))
                continue
            p = torch.log_softmax(s["logits"][b * K + k].double(), 0)
            values, ids = torch.sort(p, descending=True, stable=True)
            for v, i in zip(values[:n].tolist(), ids[:n].tolist()):
                found.append(((score + v) / (length + 1) ** alpha, k, i, score + v))
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        found = found[:n]
        if case["stay"]:
            slots, later = [None] * K, []
            for f in found:
                if slots[f[1]] is None:
                    slots[f[1]] = f
                else:
                    later.append(f)
            found = [f if f is not None else later.pop(0) for f in slots]
        out[0].append([f[3] for f in found])
        out[1].append([b * K + f[1] for f in found])
        out[2].append([f[2] for f in found])
    return (torch.tensor(out[0], device=DEV, dtype=torch.float64), torch.tensor(out[1], device=DEV, dtype=torch.int32),
            torch.tensor(out[2], device=DEV))


def _exact_reorder(s, case):
    return [torch.stack([t[r] for r in s["rows"].tolist()]) for t in s["tensors"]]


def _exact_fork(s, case):
    """The pool as a host program would keep it."""
    P, K, window, tokens = (case[k] for k in ("page", "K", "window", "tokens"))
    old, lengths, rows, refs = s["table"].tolist(), s["lengths"].tolist(), s["rows"].tolist(), s["refs"].tolist()
    R, wide = len(old), len(old[0])
    new, size = [], []
    for r in rows:
        n = lengths[r]
        low = max(0, n - window) // P if window >= 0 else 0
        new.append([p if low <= j < -(-n // P) else -1 for j, p in enumerate(old[r])])
        size.append(n)
    for step, tables in ((1, new), (-1, old)):
        for t in tables:
            for p in t:
                if p >= 0:
                    refs[p] += step
    ends = {}
    for r in range(R):
        if size[r] % P:
            ends.setdefault(new[r][size[r] // P], []).append(r)
    copied = {}
    for page, at in ends.items():
        keeps = next((r for r in at if rows[r] == r), at[0]) if refs[page] == len(at) else None
        copied.update((r, page) for r in at if r != keeps)
    free = iter([p for p, c in enumerate(refs) if c == 0])
    copies = [[-1, -1] for _ in range(R)]
    for r in range(R):
        if r in copied:
            page = next(free)
            copies[r] = [copied[r], page]
            new[r][size[r] // P] = page
            refs[copied[r]] -= 1
            refs[page] += 1
        for j in range(-(-size[r] // P), -(-(size[r] + tokens) // P)):
            if window < 0 or j >= max(0, size[r] + tokens - window) // P:
                new[r][j] = next(free)
                refs[new[r][j]] += 1
    shared = []
    for a in range(0, R, K):
        j = 0
        while j < min(size[a:a + K]) // P and len({new[r][j] for r in range(a, a + K)}) == 1:
            j += 1
        shared.append(j * P)
    for layer in s["layers"]:
        for t in layer:
            raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
            for src, dst in copies:
                if dst >= 0:
                    raw[dst] = raw[src]
    ints = [torch.tensor(x, device=DEV, dtype=torch.int32) for x in (new, refs, size, copies, shared)]
    return (*ints, [tuple(t.double() for t in layer) for layer in s["layers"]])


def _exact_shared(s, case):
    """Row by row over its own table."""
    (kc, ks), (vc, vs) = s["sides"]
    P, T, kv, gq, D, window = (case[k] for k in ("page", "T", "kv", "group", "dim", "window"))
    B = case["groups"] * case["K"]
    if B * kv * (case["prefix"] + case["tail"]) > 1 << 27:
        return None                                   # every row reads its whole cache here
    out = torch.zeros(B, T, kv * gq, D, device=DEV, dtype=torch.float64)
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        if not c:
            continue
        low = 0 if window < 0 else max(0, n - c - window)
        pages, base = s["table"][b, low // P:(n + P - 1) // P].long(), low // P * P
        both = []
        for codes, scale in ((kc, ks), (vc, vs)):
            y = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * scale.double()[pages][:, :, None, None]
            both.append(y.transpose(0, 1).reshape(kv, -1, D)[:, :n - base])
        k, v = both
        at = base + torch.arange(n - base, device=DEV)
        for t in range(c):
            p = n - c + t
            keep = at <= p if window < 0 else (at <= p) & (at >= p - window)
            q = s["q"][b, t].double().view(kv, gq, D)
            w = torch.einsum("hgd,hjd->hgj", q, k[:, keep]) / math.sqrt(D)
            out[b, t] = torch.einsum("hgj,hjd->hgd", torch.softmax(w, -1), v[:, keep]).reshape(kv * gq, D)
    return out
