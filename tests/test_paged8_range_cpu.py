"""Rows of 8 bits at both ends of their powers of two, in PyTorch's operations."""
import pytest
import torch

from ghost_flow_b200 import ops
from ghost_flow_b200.ops import paged

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.mark.parametrize("exponent", [-1074, -300, -140, -127, -126, -118, 0, 100, 127, 128, 134, 135, 136, 140, 300, 1023])
def test_rows_of_64_bits_of_any_size(exponent):
    """The unit is a power of two from 2^-126 to 2^127. What is above 448 of the largest one has no number in the pages and becomes NaN; the rest of its row stays."""
    y = torch.tensor([[1.0, -0.5, 0.25, 0.0]], dtype=torch.float64).ldexp(torch.tensor(exponent))
    codes, byte = paged._in_8_bits(y)
    assert byte.item() == min(max(exponent + 119, 1), 254)       # 1.0 = 0.5 2^1: 448 units hold 2^8 of them
    unit = 2.0 ** (byte.item() - 127)
    got = codes.view(E4M3).double() * unit
    for g, want in zip(got[0].tolist(), y[0].tolist()):
        if abs(want) >= 464 * unit:                              # half a step above 448
            assert g != g
        else:
            assert abs(g - want) <= max(abs(want) * 2.0 ** -4, unit * 2.0 ** -10)
