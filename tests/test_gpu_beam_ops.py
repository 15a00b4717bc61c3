"""The operators of a beam search (B200): the choice over beams and vocabulary, rows moved to the
chosen beams, pages of the cache forked and copied.

Each is compared with its definition, written out here in float64 or on the host.
"""
import math
import random

import pytest
import torch

from test_gpu_step_ops import BF16, DEV, E4M3, F32, gen, same_codes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0      # every test clears what it provokes


# --------------------------------------------------------------------------- #
#  beam_select                                                                 #
# --------------------------------------------------------------------------- #

# Scores: the sum of exponentials is off by ex2 (2^-22), by the rounding of its argument (arguments above -20 have
# the weight: 20 * 2^-24) and by its order (at most 16 terms a chain a tile, 64 tiles, 16 more in trees: (1024 + 16)
# * 2^-24 at worst); the float32 result by half a step.
LSE = 2.0 ** -22 + 20 * 2.0 ** -24 + 1040 * 2.0 ** -24


def candidates(x, scores, finished, lengths, alpha, pad, b, K, most):
    """[(rank, beam, place of the token among the beam's, token, sum)], best first."""
    out = []
    for k in range(K):
        s = float(scores[b, k])
        if not math.isfinite(s):
            continue
        n = 0 if lengths is None else int(lengths[b, k])
        if finished is not None and bool(finished[b, k]):
            out.append((s / max(n, 1) ** alpha, k, 0, pad, s))
            continue
        row = x[b * K + k].double()
        lse = float(torch.logsumexp(row, 0))
        if not math.isfinite(lse) or bool(row.isnan().any()):
            continue
        values, ids = torch.sort(row, descending=True, stable=True)
        for j, (v, i) in enumerate(zip(values[:most].tolist(), ids[:most].tolist())):
            if v > -math.inf:
                t = s + (v - lse)
                out.append((t / max(n + 1, 1) ** alpha, k, j, i, t))
    return sorted(out, key=lambda c: (-c[0], c[1], c[2]))


def check_select(nat, x, scores, finished=None, lengths=None, alpha=0.0, n=None, pad=0, stay=False, exact_order=False):
    B, K = scores.shape
    n = K if n is None else n
    got, rows, tokens = nat.beam_select(x, scores, finished=finished, lengths=lengths, length_penalty=alpha, n=n, pad=pad, stay=stay)
    assert got.dtype == F32 and rows.dtype == torch.int32 and tokens.dtype == torch.int64
    assert got.shape == rows.shape == tokens.shape == (B, n)
    xc = x.float().cpu()
    for b in range(B):
        want = candidates(xc, scores, finished, lengths, alpha, pad, b, K, n)
        chosen = [(float(s), int(r) - b * K, int(t)) for s, r, t in zip(got[b], rows[b], tokens[b])]
        by = {(c[1], c[3]): c for c in want}
        live = [c for c in chosen if c[0] > -math.inf]
        assert len(live) == min(n, len(want)) and len({c[1:] for c in live}) == len(live)
        ranks = []
        for s, k, t in live:
            c = by[(k, t)]
            assert abs(s - c[4]) <= LSE + 2.0 ** -24 * abs(c[4]) + 2.0 ** -149
            ranks.append((c[0], k, t, chosen.index((s, k, t))))
        # in order, up to what the sums can be off by; and the best there are
        best = [c[0] for c in want[:n]]
        for r, w in zip(sorted((r[0] for r in ranks), reverse=True), best):
            assert abs(r - w) <= 2 * LSE
        if stay:
            places = {}
            for c in sorted(ranks, key=lambda c: (-c[0], c[1], by[(c[1], c[2])][2])):
                places.setdefault(c[1], c[3])
            assert all(at == k for k, at in places.items())          # the best child of a beam is in its place
        else:
            assert [r[3] for r in ranks] == list(range(len(ranks)))
            assert all(a[0] >= z[0] - 2 * LSE for a, z in zip(ranks, ranks[1:]))
            if exact_order:
                assert [(c[1], c[2]) for c in live] == [(c[1], c[3]) for c in want[:n]]
        for at, c in enumerate(chosen):
            if c[0] == -math.inf:
                assert c[2] == pad and (c[1] == at if stay else c[1] == at % K)
    return got, rows, tokens


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,K,V,n,alpha,stay", [
    (1, 1, 1, 1, 0.0, False), (1, 4, 7, 4, 0.0, False), (3, 2, 33, 5, 0.7, False), (2, 5, 1000, 5, 1.0, True), (1, 4, 32000, 8, 0.0, False),
    (5, 8, 5003, 16, 0.6, False), (2, 29, 50001, 29, 0.0, True), (1, 64, 2050, 64, 0.5, False), (70, 3, 257, 3, -1.0, True),
    (1, 1, 131072, 64, 0.0, False), (9, 7, 20011, 1, 0.0, False)])
def test_select_against_definition(nat, dtype, B, K, V, n, alpha, stay):
    g = gen(B * 1000 + K)
    x = (2.5 * torch.randn(B * K, V, device=DEV, generator=g)).to(dtype)
    scores = -50 * torch.rand(B, 1, device=DEV, generator=g) - 3 * torch.rand(B, K, device=DEV, generator=g)
    finished = torch.rand(B, K, device=DEV, generator=g) < 0.3
    lengths = torch.randint(0, 50, (B, K), device=DEV, generator=g)
    x[torch.rand(B * K, V, device=DEV, generator=g) < 0.05] = -math.inf
    check_select(nat, x, scores, finished, lengths, alpha, n, 3 % V, stay)
    check_select(nat, x, scores, None, lengths.int() if alpha else None, alpha, n, 0, stay)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [9, 4000, 40003])
@pytest.mark.parametrize("how", ["constant", "ascending", "descending", "two", "masked", "zeros"])
def test_select_ties_and_adverse_orders(nat, dtype, V, how):
    """Logits in which far more values reach any bound than are wanted; ties go to the lower token and beam."""
    K, n = 3, 8
    at = torch.arange(V, device=DEV).float()
    row = {"constant": torch.full((V,), 1.5, device=DEV), "ascending": at / 8, "descending": -at / 8,
           "two": (at % 2), "masked": torch.where(at % 17 == 16, 2.0, -math.inf) if V > 16 else torch.where(at == 5, 2.0, -math.inf),
           "zeros": torch.where(at % 2 == 0, -0.0, 0.0)}[how]
    x = row.to(dtype).expand(K, V).contiguous()
    scores = torch.tensor([[-1.0, -1.0, -4.0]], device=DEV)
    check_select(nat, x, scores, n=n, exact_order=True)
    check_select(nat, x, scores, n=3, stay=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_beams_that_offer_nothing(nat, dtype):
    """NaN, infinities, nothing but -inf, dead scores; a finished beam's logits do not matter; large and tiny logits."""
    K, V = 8, 4097
    x = torch.randn(2 * K, V, device=DEV, generator=gen(5)).to(dtype)
    scores = -torch.arange(2 * K, device=DEV).float().view(2, K)
    x[0, 4000] = math.nan
    x[1, 7] = math.inf
    x[2] = -math.inf
    x[3, 5:] = -math.inf
    x[4] *= 3e36
    x[5] *= 1e-30
    x[6, ::2] = -3e38
    x[7, 1] = math.nan
    finished = torch.zeros(2, K, dtype=torch.bool, device=DEV)
    finished[0, 7] = True
    scores[1, 0], scores[1, 1], scores[1, 2] = -math.inf, math.nan, math.inf
    for n in (1, 5, 8, 64):
        check_select(nat, x, scores, finished, n=n, pad=11)
    check_select(nat, x, scores, finished, n=K, pad=11, stay=True)
    everything = torch.full((2, K), -math.inf, device=DEV)
    got, rows, tokens = nat.beam_select(x, everything, n=K, pad=11, stay=True)
    assert (got == -math.inf).all() and (tokens == 11).all() and torch.equal(rows.view(-1), torch.arange(2 * K, device=DEV).int())
    x[:K] = math.nan
    finished[0] = True
    got, rows, tokens = check_select(nat, x, scores, finished, n=5, pad=2)
    assert rows[0].tolist() == [0, 1, 2, 3, 4] and got[0].tolist() == [0, -1, -2, -3, -4]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_layouts_stream_and_graph(nat, dtype):
    B, K, V = 2, 3, 5001
    wide = torch.randn(B * K, V + 13, device=DEV, generator=gen(6)).to(dtype)
    scores = -torch.rand(B, K, device=DEV, generator=gen(7))
    want = nat.beam_select(wide[:, 5:5 + V].contiguous(), scores)
    same = lambda o: all(torch.equal(a, z) for a, z in zip(o, want))  # noqa: E731
    assert same(nat.beam_select(wide[:, 5:5 + V], scores))                       # rows of any alignment
    assert same(nat.beam_select(wide[:, 5:5 + V].t().contiguous().t(), scores.t().contiguous().t()))
    x = wide[:, 5:5 + V]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = nat.beam_select(x, scores)
    torch.cuda.current_stream().wait_stream(side)
    assert same(o)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nat.beam_select(x, scores))
        graphs.append(g)
    for g in graphs:
        g.replay()
    assert same(outs[0]) and same(outs[1])
    x.neg_()
    want = nat.beam_select(x, scores)
    graphs[1].replay()
    assert same(outs[1])


def test_select_refusals(nat):
    x, scores = torch.zeros(6, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    for bad in (dict(logits=x[:5]), dict(logits=x[:, :0]), dict(logits=x[0]), dict(scores=scores.double()), dict(scores=scores[0]),
                dict(n=0), dict(n=65), dict(n=2, stay=True), dict(finished=torch.zeros(2, 3, device=DEV)),
                dict(finished=torch.zeros(3, 2, device=DEV, dtype=torch.bool)), dict(length_penalty=1.0),
                dict(length_penalty=math.nan), dict(lengths=torch.zeros(2, device=DEV, dtype=torch.int32)), dict(pad=-1),
                dict(pad=2 ** 31), dict(logits=torch.zeros(130, 4, device=DEV), scores=torch.zeros(2, 65, device=DEV))):
        with pytest.raises(ValueError):
            nat.beam_select(**{**dict(logits=x, scores=scores), **bad})
    with pytest.raises(TypeError):
        nat.beam_select(x.half(), scores)
    with pytest.raises(TypeError):
        nat.beam_select(x, scores, lengths=scores)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.beam_select(x, scores.cpu())
    with pytest.raises(RuntimeError, match="no backward"):
        nat.beam_select(x.clone().requires_grad_(), scores)
    with pytest.raises(RuntimeError, match="no backward"):
        nat.beam_select(x, scores.clone().requires_grad_())
    with pytest.raises(nat.NativeError, match="65535"):
        nat.beam_select(torch.zeros(65536, 1, device=DEV), torch.zeros(65536, 1, device=DEV))
    assert [t.shape for t in nat.beam_select(x[:0], scores[:0])] == [(0, 3)] * 3


# --------------------------------------------------------------------------- #
#  reorder_rows                                                                #
# --------------------------------------------------------------------------- #

MAPS = {"same": lambda g, rng: list(range(g)), "turn": lambda g, rng: [(i + 1) % g for i in range(g)],
        "first": lambda g, rng: [0] * g, "last": lambda g, rng: [g - 1] * g, "swap": lambda g, rng: [i ^ 1 if i ^ 1 < g else i for i in range(g)],
        "any": lambda g, rng: [rng.randrange(g) for _ in range(g)], "holes": lambda g, rng: [rng.choice([-1, i, rng.randrange(g)]) for i in range(g)],
        "stay": lambda g, rng: [i if i % 3 else (1 if g > 1 else 0) for i in range(g)]}


@pytest.mark.parametrize("how", list(MAPS))
@pytest.mark.parametrize("groups,group", [(1, 1), (2, 3), (5, 8), (16, 4), (1, 64), (1, 1024), (3, 333)])
def test_reorder_any_map(nat, how, groups, group):
    rng = random.Random(group)
    R = groups * group
    maps = [MAPS[how](group, rng) for _ in range(groups)]
    rows = torch.tensor([r if r < 0 else r + i * group for i, m in enumerate(maps) for r in m], device=DEV, dtype=torch.int32)
    g = gen(group)
    shapes = [((7, 9), BF16), ((1000,), F32), ((3,), torch.uint8), ((33, 17), F32), ((4, 2048) if R < 400 else (64,), BF16), ((2,), torch.int64), ((), F32), ((0, 5), F32),
              ((5, 3), torch.bool)]
    tensors = [(100 * torch.randn((R, *s), device=DEV, generator=g)).to(t) for s, t in shapes]
    wide = torch.randn(R, 50, device=DEV, generator=g)
    tensors.append(wide[:, 3:40])                        # rows apart, at any alignment
    src = torch.where(rows < 0, torch.arange(R, device=DEV), rows).long()
    want, edge = [t[src] for t in tensors], (wide[:, :3].clone(), wide[:, 40:].clone())
    versions = [t._version for t in tensors]
    nat.reorder_rows(tensors, rows, group=group)
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)
    assert torch.equal(wide[:, :3], edge[0]) and torch.equal(wide[:, 40:], edge[1])
    assert all(t._version > v for t, v in zip(tensors, versions))
    assert nat.device_error_flags(0) == 0


def test_reorder_many_tensors_long_rows_and_whole_batches(nat):
    """More tensors than one launch takes; rows of many pieces; one group by default, int64 rows; a graph."""
    R = 6
    tensors = [torch.randn(R, 30 + i, device=DEV, generator=gen(i)) for i in range(200)]
    tensors.append(torch.randn(R, 70001, device=DEV, generator=gen(999)))
    tensors.append(torch.randn(R, 3, 40000, device=DEV, generator=gen(998)).to(BF16))
    rows = torch.tensor([3, 3, 0, 5, 4, 1], device=DEV)
    want = [t[rows] for t in tensors]
    nat.reorder_rows(tensors, rows)
    assert all(torch.equal(t, w) for t, w in zip(tensors, want))
    rows = rows.int()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nat.reorder_rows(tensors, rows)
    for m in ([1, 0, 3, 2, 5, 4], [2, 2, 2, 3, 4, 2], [0, 1, 2, 3, 4, 5]):
        rows.copy_(torch.tensor(m, device=DEV))
        want = [t[rows.long()] for t in tensors]
        graph.replay()
        assert all(torch.equal(t, w) for t, w in zip(tensors, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = [t.flip(0) for t in tensors]
    with torch.cuda.stream(side):
        nat.reorder_rows(tensors, torch.arange(R - 1, -1, -1, device=DEV))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, w) for t, w in zip(tensors, want))


def test_reorder_refusals(nat):
    t = torch.arange(12.0, device=DEV).view(6, 2)
    rows = torch.arange(6, device=DEV, dtype=torch.int32)
    for bad in (dict(rows=rows.view(2, 3)), dict(group=4), dict(group=0), dict(tensors=[t[:5]]), dict(tensors=[t.t().contiguous().t()]),
                dict(tensors=[t[:1].expand(6, 2)]), dict(tensors=[t[0, 0]]), dict(tensors=[t, t.clone(), t]), dict(rows=torch.zeros(1025, device=DEV, dtype=torch.int32),
                                                                                tensors=[torch.zeros(1025, 1, device=DEV)])):
        with pytest.raises(ValueError):
            nat.reorder_rows(**{**dict(tensors=[t], rows=rows), **bad})
    with pytest.raises(TypeError):
        nat.reorder_rows([t], rows.float())
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.reorder_rows([t], rows.cpu())
    with pytest.raises(RuntimeError, match="requires grad"):
        nat.reorder_rows([t.clone().requires_grad_()], rows)
    before = t.clone()
    nat.reorder_rows([t], torch.tensor([0, 3, 6, -2, 2, 5], device=DEV, dtype=torch.int32), group=3)   # rows of other groups
    assert torch.equal(t, before) and nat.device_error_flags(0) == 8
    nat.reorder_rows([], rows)
    nat.reorder_rows([t[:0]], rows[:0])


# --------------------------------------------------------------------------- #
#  kv_fork, kv_copy_pages                                                      #
# --------------------------------------------------------------------------- #

class Pool:
    """The pages as a host program would keep them."""

    def __init__(self, R, blocks, pages, P, group=None):
        self.R, self.blocks, self.P, self.group = R, blocks, P, group
        self.table = [[-1] * blocks for _ in range(R)]
        self.refs, self.lengths, self.flagged = [0] * pages, [0] * R, False

    def fork(self, parents, tokens, window):
        P, R = self.P, self.R
        size = [0 if p < 0 else self.lengths[p] for p in parents]
        low = [0 if window is None else max(0, n - window) // P for n in size]
        new = [[self.table[p][j] if p >= 0 and low[r] <= j < -(-size[r] // P) else -1 for j in range(self.blocks)]
               for r, p in enumerate(parents)]
        for step, tables in ((1, new), (-1, self.table)):
            for t in tables:
                for p in t:
                    if p >= 0:
                        self.refs[p] += step
        ends = {}
        for r, n in enumerate(size):
            if n % P and new[r][n // P] >= 0:
                ends.setdefault(new[r][n // P], []).append(r)
        copied = {}
        for page, at in ends.items():
            keep = next((r for r in at if parents[r] == r), at[0]) if self.refs[page] == len(at) else None
            copied.update((r, page) for r in at if r != keep)
        free, copies, self.flagged = [p for p, c in enumerate(self.refs) if c == 0], [[-1, -1] for _ in range(R)], False
        for r, n in enumerate(size):
            jobs = [n // P] if r in copied else []
            if parents[r] >= 0:
                first = -(-n // P) if window is None else max(-(-n // P), max(0, n + tokens - window) // P)
                last = -(-(n + tokens) // P)
                if last > self.blocks:
                    self.flagged = True
                jobs += range(first, min(last, self.blocks))
            if r in copied:
                self.refs[copied[r]] -= 1
            for j in jobs:
                new[r][j] = free.pop(0) if free else -1
                if new[r][j] < 0:
                    self.flagged = True
                else:
                    self.refs[new[r][j]] += 1
                    if r in copied and j == n // P:
                        copies[r] = [copied[r], new[r][j]]
        self.table, self.lengths = new, size
        shared = []
        for a in range(0, R, self.group or R):
            rows, j = range(a, a + (self.group or R)), 0
            while j < min(size[r] for r in rows) // P and len({new[r][j] for r in rows}) == 1:
                j += 1
            shared.append(j * P)
        return copies, shared

    def on_device(self):
        wide = torch.full((self.R, self.blocks + 3), 77, device=DEV, dtype=torch.int32)       # rows apart
        table = wide[:, :self.blocks]
        table.copy_(torch.tensor(self.table, device=DEV, dtype=torch.int32).view(self.R, self.blocks))
        ints = lambda v: torch.tensor(v, device=DEV, dtype=torch.int32)  # noqa: E731
        return wide, table, ints(self.refs), ints(self.lengths)


def check_fork(nat, pool, parents, tokens, window, state=None):
    wide, table, refs, lengths = state or pool.on_device()
    copies, shared = nat.kv_fork(table, refs, lengths, torch.tensor(parents, device=DEV, dtype=torch.int32), pool.P, tokens=tokens,
                                 window=window, group=pool.group)
    want_copies, want_shared = pool.fork(parents, tokens, window)
    assert table.tolist() == pool.table and refs.tolist() == pool.refs and lengths.tolist() == pool.lengths
    assert copies.tolist() == want_copies
    assert shared is None if pool.group is None else shared.tolist() == want_shared
    assert (wide[:, pool.blocks:] == 77).all()
    assert nat.device_error_flags(0) == (8 if pool.flagged else 0)
    return wide, table, refs, lengths


@pytest.mark.parametrize("R,group,P,blocks,pages,window", [
    (1, 1, 16, 5, 9, None), (4, 4, 32, 20, 60, None), (12, 3, 16, 40, 300, 70), (64, 4, 64, 30, 700, 200), (200, 50, 16, 50, 5000, None),
    (1024, 8, 32, 9, 9000, None), (6, None, 16, 300, 700, 100)])
def test_fork_over_many_steps(nat, R, group, P, blocks, pages, window):
    """Prompts, beams that follow one another, rows that end and begin again, drafts that are taken back."""
    rng = random.Random(R)
    pool = Pool(R, blocks, pages, P, group)
    state = None
    for step in range(14):
        if step == 0:
            parents, tokens = list(range(R)), rng.randint(1, 2 * P)
        else:
            tokens = rng.choice([1, 1, 2, P // 2, P + 3])
            parents = [rng.choice([r, r, rng.randrange(R)]) for r in range(R)]
            if step % 4 == 3:
                parents[rng.randrange(R)] = -1
        if max(pool.lengths) + tokens > blocks * P:
            break
        state = check_fork(nat, pool, parents, tokens, window, state)
        # the new tokens are written; some sequences write fewer than they have pages for, one goes back by a few
        for r in range(R):
            if parents[r] >= 0 and rng.random() < 0.9:
                pool.lengths[r] += tokens if window is None else min(tokens, window)
            elif pool.lengths[r] > 3 and window is None:
                pool.lengths[r] -= rng.randint(0, 3)
        state[3].copy_(torch.tensor(pool.lengths, device=DEV, dtype=torch.int32))
    used = [0] * pages
    for t in pool.table:
        for p in t:
            if p >= 0:
                used[p] += 1
    assert used == pool.refs


def test_fork_pages_held_elsewhere_and_shared_in_the_middle(nat):
    P = 16
    pool = Pool(3, 6, 30, P, 3)
    check_fork(nat, pool, [0, 1, 2], 40, None)
    pool.lengths = [40, 0, 0]
    check_fork(nat, pool, [0, 0, 0], 1, None)
    pool.refs[pool.table[0][2]] += 1                    # someone else holds the begun page: nobody may write it
    pool.lengths = [41, 41, 41]
    check_fork(nat, pool, [0, 0, 2], 1, None)
    pool.lengths = [20, 41, 20]                         # one row goes back into a block that others have whole
    check_fork(nat, pool, [0, 1, 0], 5, None)
    pool.lengths = [32, 41, 32]                         # at a border nothing is copied
    check_fork(nat, pool, [2, 2, 2], 0, None)


def test_fork_window_lets_pages_go_and_skips_what_it_will_not_see(nat):
    P = 16
    pool = Pool(2, 64, 40, P, 2)
    check_fork(nat, pool, [0, 1], 900, 50)              # a prompt: the pages of its last 50 tokens
    assert sum(p >= 0 for p in pool.table[0]) == 4      # blocks 850 // 16 = 53 to 899 // 16 = 56
    pool.lengths = [900, 900]
    check_fork(nat, pool, [0, 1], 1, 50)
    check_fork(nat, pool, [1, 1], 1, 50)
    pool.lengths = [950, 950]
    check_fork(nat, pool, [1, 1], 1, 50)
    check_fork(nat, pool, [1, 0], 1, 0)                 # a window of the new token alone
    assert sum(c for c in pool.refs) <= 4


def test_fork_runs_out(nat):
    """Too few pages or blocks, bad parents, lengths and pages: empty entries, flagged, nothing else."""
    P = 16
    pool = Pool(4, 4, 6, P, 4)
    check_fork(nat, pool, [0, 1, 2, 3], 17, None)       # eight pages wanted
    assert pool.flagged and pool.table == [[0, 1, -1, -1], [2, 3, -1, -1], [4, 5, -1, -1], [-1] * 4]
    pool.lengths = [17, 17, 0, 0]
    check_fork(nat, pool, [0, 0, 0, 1], 1, None)        # copies of which two find a page
    pool = Pool(2, 3, 50, P, 2)
    check_fork(nat, pool, [0, 1], 49, None)             # past the table
    assert pool.flagged
    table, refs, lengths = pool.on_device()[1:]
    for parents, n in (([5, 1], [3, 3]), ([-2, 1], [3, 3]), ([0, 1], [-1, 3]), ([0, 1], [49, 3])):
        lengths.copy_(torch.tensor(n, device=DEV))
        nat.kv_fork(table, refs, lengths, torch.tensor(parents, device=DEV), P)
        assert nat.device_error_flags(0) == 8
        assert lengths.tolist() == [0, 3]
        refs.copy_(torch.tensor(pool.refs, device=DEV))
        table.copy_(torch.tensor(pool.table, device=DEV))
    table[1, 0] = 50                                    # a page that is not there
    lengths.fill_(3)
    nat.kv_fork(table, refs, lengths, torch.tensor([1, 1], device=DEV), P, tokens=0)
    assert nat.device_error_flags(0) == 8 and table[0, 0] == -1


def test_fork_graph_stream_and_refusals(nat):
    P = 16
    pool = Pool(4, 6, 30, P, 2)
    state = check_fork(nat, pool, [0, 1, 2, 3], 20, None)
    table, refs, lengths = state[1:]
    lengths.fill_(20)
    parents = torch.tensor([1, 1, 2, 2], device=DEV, dtype=torch.int32)
    keep = [t.clone() for t in (table, refs, lengths)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copies, shared = nat.kv_fork(table, refs, lengths, parents, P, group=2)
    pool.lengths = [20] * 4
    for turn in ([1, 1, 2, 2], [0, 0, 3, 3], [1, 0, 3, 2]):
        parents.copy_(torch.tensor(turn, device=DEV))
        graph.replay()
        want = pool.fork(turn, 1, None)
        assert (copies.tolist(), shared.tolist()) == want and table.tolist() == pool.table and refs.tolist() == pool.refs
    for t, k in zip((table, refs, lengths), keep):
        t.copy_(k)
    versions = [t._version for t in (table, refs, lengths)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nat.kv_fork(table, refs, lengths, parents, P)
    torch.cuda.current_stream().wait_stream(side)
    assert all(t._version > v for t, v in zip((table, refs, lengths), versions))
    good = dict(table=table, refs=refs, lengths=lengths, parents=parents, page=P)
    for bad in (dict(table=table.long()), dict(table=table[0]), dict(table=table.t()), dict(refs=refs.long()), dict(refs=refs[::2]),
                dict(lengths=lengths[:3]), dict(lengths=lengths.long()), dict(parents=parents[:3]), dict(page=0), dict(tokens=-1), dict(window=-1),
                dict(group=3), dict(group=0), dict(table=table[:1].expand(4, 6)),
                dict(table=torch.zeros(1025, 1, device=DEV, dtype=torch.int32), lengths=torch.zeros(1025, device=DEV, dtype=torch.int32),
                     parents=torch.zeros(1025, device=DEV, dtype=torch.int32))):
        with pytest.raises(ValueError):
            nat.kv_fork(**{**good, **bad})
    with pytest.raises(TypeError):
        nat.kv_fork(**{**good, "parents": parents.float()})
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_fork(**{**good, "refs": refs.cpu()})
    assert nat.kv_fork(table[:0], refs, lengths[:0], parents[:0], P)[0].shape == (0, 2)


@pytest.mark.parametrize("P,H,D,layers", [(16, 1, 64, 1), (32, 10, 64, 2), (64, 16, 128, 3), (32, 3, 128, 70)])
def test_copy_pages(nat, P, H, D, layers):
    n, g = 12, gen(P + H)
    make = lambda: (torch.randint(0, 256, (n, H, P, D), device=DEV, generator=g, dtype=torch.uint8).view(E4M3),  # noqa: E731
                    torch.rand(n, H, device=DEV, generator=g))
    pools = [make() + make() for _ in range(layers)]
    want = [[t.clone() for t in layer] for layer in pools]
    pages = [[0, 11], [-1, -1], [3, 4], [0, 5], [7, 6]]
    for layer in want:
        for t in layer:
            raw = t.view(torch.uint8) if t.dtype == E4M3 else t
            for src, dst in pages:
                if dst >= 0:
                    raw[dst] = raw[src]
    at = torch.tensor(pages, device=DEV, dtype=torch.int32)
    version = pools[0][0]._version
    nat.kv_copy_pages(pools, at)
    assert all(same_codes(a, b) if a.dtype == E4M3 else torch.equal(a, b) for x, y in zip(pools, want) for a, b in zip(x, y))
    assert pools[0][0]._version > version and nat.device_error_flags(0) == 0
    nat.kv_copy_pages(pools, torch.tensor([[12, 1], [1, 12], [-1, 2], [2, -2]], device=DEV, dtype=torch.int32))
    assert nat.device_error_flags(0) == 8
    assert all(same_codes(a, b) if a.dtype == E4M3 else torch.equal(a, b) for x, y in zip(pools, want) for a, b in zip(x, y))
    graph = torch.cuda.CUDAGraph()
    at.fill_(-1)
    with torch.cuda.graph(graph):
        nat.kv_copy_pages(pools, at)
    at[2] = torch.tensor([11, 8], device=DEV)
    graph.replay()
    assert same_codes(pools[-1][2][8], want[-1][2][0]) and torch.equal(pools[0][1][8], want[0][1][0])


def test_copy_pages_past_32_bits(nat):
    H, P, D = 16, 64, 128
    n = 2 ** 32 // (H * P * D) + 3
    codes = torch.empty(n, H, P, D, device=DEV, dtype=torch.uint8)
    other = torch.zeros(1, H, P, D, device=DEV, dtype=torch.uint8).expand(n, H, P, D)
    scale = torch.ones(n, H, device=DEV)
    codes[n - 2] = torch.randint(0, 256, (H, P, D), device=DEV, generator=gen(3), dtype=torch.uint8)
    codes[n - 1].zero_()
    codes[1].zero_()
    with pytest.raises(ValueError):
        nat.kv_copy_pages([(codes, scale, other, scale.clone())], torch.tensor([[n - 2, n - 1]], device=DEV, dtype=torch.int32))
    scale[n - 2] = 8.0
    nat.kv_copy_pages([(codes, scale, codes.clone(), scale.clone())], torch.tensor([[n - 2, n - 1], [-1, -1]], device=DEV, dtype=torch.int32))
    assert torch.equal(codes[n - 1], codes[n - 2]) and (scale[n - 1] == 8).all() and codes[1].max() == 0


def test_copy_pages_refusals(nat):
    n, H, P, D = 4, 2, 16, 64
    c, s = torch.zeros(n, H, P, D, device=DEV, dtype=torch.uint8), torch.zeros(n, H, device=DEV)
    at = torch.zeros(1, 2, device=DEV, dtype=torch.int32)
    for layer, pages in (((c, s, c.float(), s), at), ((c, s, c[:3], s), at), ((c, s, c, s.double()), at), ((c, s[:3], c, s), at),
                         ((c[:, :, ::2], s, c, s), at), ((c, s, c, s), at.long()), ((c, s, c, s), at[0]),
                         ((c.view(n, H, 8, 128), s, c, s), at)):
        with pytest.raises(ValueError):
            nat.kv_copy_pages([layer], pages)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_copy_pages([(c, s, c, s)], at.cpu())
    nat.kv_copy_pages([], at)
    nat.kv_copy_pages([(c, s, c.clone(), s.clone())], at[:0])
