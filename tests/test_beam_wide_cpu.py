"""Rows kept or replaced as wide elements are the rows bit for bit, whatever their length and type."""
import pytest
import torch

from neuratensor_b200.inference.beams import _wide


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(256,), (256, 16), (1153, 17), (6,), (1,), (2, 3)])
def test_wide_rows(dtype, shape):
    R, bits = 5, torch.int32 if dtype == torch.float32 else torch.int16
    make = lambda seed: torch.randint(torch.iinfo(bits).min, torch.iinfo(bits).max, (R, *shape), dtype=bits,  # noqa: E731
                                      generator=torch.Generator().manual_seed(seed))
    old, new = make(1), make(2)                           # any bits, NaNs of all kinds among them
    keep = torch.tensor([True, False, False, True, False]).view(-1, 1)
    want = torch.where(keep.view(-1, *[1] * len(shape)), old, new)
    a, b = _wide(old.view(dtype)), _wide(new.view(dtype))
    row = torch.tensor(shape).prod().item() * old.element_size()
    assert a.element_size() == next(s for s in (16, 8, 4, 2) if row % s == 0)
    torch.where(keep, a, b, out=a)
    assert torch.equal(old, want)
