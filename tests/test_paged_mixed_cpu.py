"""Rotation, paged append and paged decode without a GPU: arguments of other types and kinds than the usual ones."""
import pytest
import torch

from varlenabsorbflashattn_b200 import paged


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_integers_beyond_32_bits_stay_out_of_range(dtype):
    top = 2**31 - 1
    values = [0, 7, top, top + 1, 2**32 - 1] + ([2**32 + 3, 2**62] if dtype != torch.uint32 else []) + ([-1, -2**31 - 1, -2**32 - 5] if dtype == torch.int64 else [])
    got = paged._ints(torch.tensor(values, dtype=dtype), torch.device("cpu"), "page_table")
    assert got.dtype == torch.int32 and got.tolist() == [max(-2**31, min(top, v)) for v in values]


def test_integers_of_32_bits_and_less_stay_as_they_are():
    x = torch.tensor([5, -3], dtype=torch.int32)
    assert paged._ints(x, x.device, "x") is x
    for dtype in (torch.int8, torch.int16):
        assert paged._ints(x.to(dtype), x.device, "x").tolist() == [5, -3]
