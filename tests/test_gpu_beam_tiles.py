"""beam_select over many rows (B200): slices of a dozen tiles and more, in the orders that are hardest on a running bound.

Six hundred rows and more leave a slice a row, so that a slice's list of candidates is carried, cut and overrun from tile
to tile.  Compared with the definition in float64; what ties decide is compared exactly."""
import math

import pytest
import torch

from test_gpu_beam_ops import LSE, candidates
from test_gpu_step_ops import BF16, DEV, F32, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0


def order(how, V):
    at = torch.arange(V, device=DEV)
    noise = 2.5 * torch.randn(V, device=DEV, generator=gen(V))
    return {"constant": lambda: torch.full((V,), 1.5, device=DEV), "ascending": lambda: at / 8.0, "descending": lambda: -at / 8.0,
            "two": lambda: (at % 2).float(), "masked": lambda: torch.where(at % 97 == 96, 2.0, -math.inf),
            "zeros": lambda: torch.where(at % 2 == 0, -0.0, 0.0),
            # a part of the vocabulary that is not used comes first: far below the rest, or a little, or not at all
            "low start": lambda: torch.where(at < 9000, -1e9, noise), "lower start": lambda: torch.where(at < 9000, -20.0, noise),
            "late": lambda: torch.where(at < V - 7000, -math.inf, noise),
            # more equal values than a list holds, from the middle on; and steps, of which each has many
            "plateau": lambda: torch.where(at < V // 2, noise - 30.0, torch.where(at % 3 == 0, 3.0, noise - 30.0)),
            "steps": lambda: (4 * noise).round() / 4, "stairs": lambda: (at // 5000).float()}[how]()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [49152, 50001])            # whole tiles of aligned rows; rows at every alignment
@pytest.mark.parametrize("n", [1, 8, 32, 64])
@pytest.mark.parametrize("how", ["constant", "ascending", "descending", "two", "masked", "zeros", "low start", "lower start", "late", "plateau",
                                 "steps", "stairs"])
def test_adverse_orders_over_many_tiles(nat, dtype, V, n, how):
    B, K = 200, 3
    x = order(how, V).to(dtype).expand(B * K, V).contiguous()
    scores = torch.tensor([-1.0, -1.0, -4.3], device=DEV).expand(B, K).contiguous()
    got = nat.beam_select(x, scores, n=n, pad=5)
    want = candidates(x[:K].float().cpu(), scores, None, None, 0.0, 5, 0, K, n)[:n]
    assert [(int(r), int(t)) for r, t in zip(got[1][0], got[2][0])] == [(c[1], c[3]) for c in want]
    for s, c in zip(got[0][0].tolist(), want):
        assert abs(s - c[4]) <= LSE + 2.0 ** -24 * abs(c[4])
    base = K * torch.arange(B, device=DEV, dtype=torch.int32)[:, None]
    for o, first in zip((got[0], got[1] - base, got[2]), (got[0][:1], got[1][:1], got[2][:1])):
        assert torch.equal(o, first.expand(B, n))        # every item is the same
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, nat.beam_select(x, scores, n=n, pad=5)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,K,V,n,alpha,stay", [(160, 4, 131072, 8, 0.0, False), (40, 16, 50001, 32, 0.6, False), (150, 4, 50001, 4, 0.7, True),
                                                (10, 64, 32003, 64, 1.0, True), (640, 1, 30000, 5, 0.0, False)])
def test_random_rows_over_many_tiles(nat, dtype, B, K, V, n, alpha, stay):
    g = gen(B + K)
    x = 2.5 * torch.randn(B * K, V, device=DEV, generator=g)
    x[::3, :5000] = -math.inf                             # of some rows the first tiles are empty
    x = x.to(dtype)
    scores = -50 * torch.rand(B, 1, device=DEV, generator=g) - 3 * torch.rand(B, K, device=DEV, generator=g)
    finished = torch.rand(B, K, device=DEV, generator=g) < 0.05
    lengths = torch.randint(1, 50, (B, K), device=DEV, generator=g)
    call = lambda: nat.beam_select(x, scores, finished=finished, lengths=lengths, length_penalty=alpha, n=n, pad=7, stay=stay)  # noqa: E731
    got = call()
    for b in range(0, B, max(1, B * K // 24)):            # some items, all of their beams
        rows = x[b * K:b * K + K].float().cpu()
        want = candidates(rows, scores[b:b + 1], finished[b:b + 1], lengths[b:b + 1], alpha, 7, 0, K, n)
        by = {(c[1], c[3]): c for c in want}
        live = got[0][b] > -math.inf                      # a finished beam offers one candidate
        assert int(live.sum()) == min(n, len(want)) and (got[2][b][~live] == 7).all()
        chosen = [by[(int(r) - b * K, int(t))] for r, t in zip(got[1][b][live], got[2][b][live])]
        assert len({c[1:4] for c in chosen}) == len(chosen)
        for s, c in zip(got[0][b][live].tolist(), chosen):
            assert abs(s - c[4]) <= LSE + 2.0 ** -24 * abs(c[4])
        ranks = [c[0] for c in chosen]
        for r, w in zip(sorted(ranks, reverse=True), want):          # the best there are, up to what the sums can be off by
            assert abs(r - w[0]) <= 2 * LSE
        if not stay:
            assert all(a >= z - 2 * LSE for a, z in zip(ranks, ranks[1:]))
    for _ in range(3):
        assert all(torch.equal(a, z) for a, z in zip(got, call()))
