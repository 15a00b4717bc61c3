"""Calls at the edges of what the operators of a beam search document (B200)."""
import math

import pytest
import torch

from test_gpu_step_ops import BF16, DEV, F32, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import native
    native.load()
    native.device_error_flags(0)
    yield native
    assert native.device_error_flags(0) == 0      # every test clears what it provokes


def ints(v, dtype=torch.int32):
    return torch.tensor(v, device=DEV, dtype=dtype)


def test_fork_over_a_table_of_no_blocks_flags_what_is_bad(nat):
    table, refs = torch.empty(3, 0, device=DEV, dtype=torch.int32), ints([0, 0])
    for parents, lengths, bad in (([0, 1, 2], [0, 0, 0], 0), ([0, -1, 0], [0, 0, 0], 0), ([0, 3, 2], [0, 0, 0], 8), ([0, -2, 2], [0, 0, 0], 8),
                                  ([0, 1, 2], [0, 1, 0], 8), ([0, 1, 2], [0, 0, -1], 8)):
        n = ints(lengths)
        copies, shared = nat.kv_fork(table, refs, n, ints(parents), 16, tokens=0, group=3)
        assert nat.device_error_flags(0) == bad
        assert n.tolist() == [0, 0, 0] and copies.tolist() == [[-1, -1]] * 3 and shared.tolist() == [0] and refs.tolist() == [0, 0]
    nat.kv_fork(table, refs, ints([0, 0, 0]), ints([0, 1, 2]), 16, tokens=1)         # room for a token where there is none
    assert nat.device_error_flags(0) == 8
    # and over a pool of no pages
    n, table = ints([0, 0]), torch.full((2, 3), -1, device=DEV, dtype=torch.int32)
    nat.kv_fork(table, refs[:0], n, ints([0, 1]), 16, tokens=0)
    assert nat.device_error_flags(0) == 0
    nat.kv_fork(table, refs[:0], n, ints([0, 1]), 16, tokens=1)
    assert nat.device_error_flags(0) == 8 and (table == -1).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K,V,n", [(1, 20011, 8), (3, 20011, 8), (8, 50001, 64), (2, 700, 64)])
@pytest.mark.parametrize("score", [-3e38, -1e25, 1e30])
def test_a_beams_own_are_in_the_order_of_their_logits_where_sums_are_alike(nat, dtype, K, V, n, score):
    """A score so large that the logits vanish beside it in float64 too, as one that marks a beam as the last resort."""
    x = (2.5 * torch.randn(K, V, device=DEV, generator=gen(V + K))).to(dtype)
    got, rows, tokens = nat.beam_select(x, torch.full((1, K), score, device=DEV), n=n)
    _, ids = torch.sort(x[0].double(), descending=True, stable=True)
    assert (rows == 0).all() and torch.equal(tokens[0], ids[:n])                     # all tie: the lowest beam's
    assert torch.allclose(got, torch.full_like(got, score), rtol=1e-6)
    # behind a live beam's candidates, with a finished one that ties with them
    scores, finished = torch.full((1, K + 2), score, device=DEV), torch.zeros(1, K + 2, device=DEV, dtype=torch.bool)
    scores[0, 0], finished[0, 1] = abs(score) if score < 0 else 3e38, True
    y = torch.cat([torch.full((2, V), -math.inf, device=DEV, dtype=dtype), x])
    y[0, 5], y[0, 3] = 1.0, 2.0
    m = max(n, 4)
    got, rows, tokens = nat.beam_select(y, scores, finished=finished, n=m, pad=9)
    assert rows[0].tolist() == [0, 0, 1] + [2] * (m - 3) and tokens[0, :3].tolist() == [3, 5, 9] and torch.equal(tokens[0, 3:], ids[:m - 3])
