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


@pytest.mark.parametrize("far", [2 ** 32, -(2 ** 32), 2 ** 31, 2 ** 62])
def test_indexes_past_32_bits_are_out_of_range(nat, far):
    """int64 indexes that would be others in int32."""
    t = torch.arange(12.0, device=DEV).view(6, 2)
    nat.reorder_rows([t], ints([0, 1, 2, far + 1, 5, far + 4], torch.int64), group=3)
    assert nat.device_error_flags(0) == 8
    assert t.tolist() == [[0, 1], [2, 3], [4, 5], [6, 7], [10, 11], [10, 11]]        # those rows stay
    table, refs, lengths = torch.full((3, 4), -1, device=DEV, dtype=torch.int32), ints([1, 1, 1, 0, 0, 0, 0]), ints([16, 16, 16])
    table[:, 0] = ints([0, 1, 2])
    nat.kv_fork(table, refs, lengths, ints([0, far, far + 1], torch.int64), 16, tokens=0)
    assert nat.device_error_flags(0) == 8
    assert lengths.tolist() == [16, 0, 0] and refs.tolist() == [1, 0, 0, 0, 0, 0, 0] and (table[1:] == -1).all()


def test_lengths_and_shared_counts_past_32_bits(nat):
    x = torch.randn(2, 50, device=DEV, generator=gen(1))
    x[1] = x[0]
    scores = torch.tensor([[-2.0, -2.0]], device=DEV)
    # the longer beam's sums are divided by more, so that it is ahead
    _, rows, _ = nat.beam_select(x, scores, lengths=ints([[3, 2 ** 32 + 1]], torch.int64), length_penalty=1.0, n=2)
    assert (rows == 1).all()
    H, D, P = 1, 64, 16
    q = torch.randn(2, 1, H, D, device=DEV, generator=gen(2))
    codes = torch.randint(0, 0x70, (300, H, P, D), device=DEV, dtype=torch.uint8, generator=gen(3))
    scale = torch.full((300, H), 2.0 ** -8, device=DEV)
    table = torch.arange(256, device=DEV, dtype=torch.int32).expand(2, 256).contiguous()
    table[1, 2:] = 256 + torch.arange(254, device=DEV, dtype=torch.int32) % 40
    table = torch.cat([table, torch.full((2, 1 << 14), -1, device=DEV, dtype=torch.int32)], 1)
    args = (q, codes, scale, codes.clone(), scale.clone(), table, ints([4096, 4096]))
    want = nat.kv_attention_shared(*args, ints([0]))
    # counted as negative, which is nothing
    assert torch.equal(nat.kv_attention_shared(*args, ints([-(2 ** 32) + 4096], torch.int64)), want)


@pytest.mark.parametrize("groups,group", [(1, 7), (300, 4), (2, 1000)])
def test_a_map_that_moves_with_the_rows(nat, groups, group):
    """The map may be one of the tensors: it is read as it was."""
    g = gen(group)
    R = groups * group
    rows = (torch.randint(0, group, (groups, group), device=DEV, generator=g) + group * torch.arange(groups, device=DEV)[:, None]).view(-1).int()
    x = torch.randn(R, 300, device=DEV, generator=g)
    src = rows.long()
    want = [rows[src], x[src]]
    nat.reorder_rows([rows, x], rows, group=group)
    assert torch.equal(rows, want[0]) and torch.equal(x, want[1])
