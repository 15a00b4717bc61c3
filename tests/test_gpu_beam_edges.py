"""Calls at the edges of what the operators of a beam search document (B200)."""
import pytest
import torch

from test_gpu_step_ops import DEV

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
