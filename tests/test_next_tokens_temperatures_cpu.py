"""next_tokens and the forms that a temperature may have: a number, a tensor of one element, one of each row; alone and with other choices."""
import math

import pytest
import torch

from ghost_flow_b200 import ops

ONE = [0.7, torch.tensor(0.7), torch.tensor([0.7]), torch.tensor([[0.7]]), torch.tensor(0.7, dtype=torch.float64), torch.tensor(2)]
NOT_ABOVE_0 = [0, -1.0, math.nan, -math.inf, None, torch.tensor(0.0), torch.tensor(-2.0), torch.tensor(math.nan)]


@pytest.mark.parametrize("temperature", ONE, ids=str)
@pytest.mark.parametrize("B", [1, 3])
def test_one_temperature_of_all_rows(temperature, B):
    x, u = 3 * torch.randn(B, 40), torch.rand(B)
    got = ops.next_tokens(x, temperature)
    assert got.shape == (B, 1) and ((got >= 0) & (got < 40)).all()
    want = ops.sample_tokens(x, u, float(temperature), 7, 0.9)
    assert torch.equal(ops.next_tokens(x, temperature, top_k=7, top_p=0.9, u=u), want)


def test_one_temperature_alone_draws_as_a_number_does():
    x = 3 * torch.randn(64, 40)
    for t in (torch.tensor(0.5), torch.tensor([0.5]), torch.tensor(0.5, dtype=torch.float64)):
        torch.manual_seed(5)
        a = ops.next_tokens(x, t)
        torch.manual_seed(5)
        assert torch.equal(a, ops.next_tokens(x, 0.5))


@pytest.mark.parametrize("temperature", NOT_ABOVE_0, ids=str)
@pytest.mark.parametrize("choice", [{}, dict(top_k=5), dict(top_p=0.5), dict(min_p=0.1), dict(u=torch.full((4,), 0.75))], ids=lambda c: "-".join(c) or "none")
def test_what_is_not_above_0_takes_the_likeliest(temperature, choice):
    x = torch.randn(4, 30)
    assert torch.equal(ops.next_tokens(x, temperature, **choice), x.argmax(-1, keepdim=True))


def test_a_temperature_of_each_row():
    x, u = 3 * torch.randn(3, 40), torch.rand(3)
    t = torch.tensor([0.0, 0.5, math.nan])
    assert torch.equal(ops.next_tokens(x, t, u=u), ops.sample_tokens(x, u, t))
    torch.manual_seed(2)
    a = ops.next_tokens(x, t)
    torch.manual_seed(2)
    assert torch.equal(a, ops.sample_tokens(x, torch.rand(3), t))
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.float64), torch.ones(3, 1)):
        with pytest.raises(ValueError, match="temperature"):
            ops.next_tokens(x, bad)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_random_numbers_do_not_go_by_the_default_type(dtype):
    x = torch.randn(4, 30, dtype=torch.float32)
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        got = ops.next_tokens(x, 0.8, top_k=5)
    finally:
        torch.set_default_dtype(before)
    assert got.shape == (4, 1)
