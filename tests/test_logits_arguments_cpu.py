"""Arguments of what stands between logits and a token: ranges, and what goes with what."""
import pytest
import torch

import _paged_oracle as oracle
from ghost_flow_b200 import ops


@pytest.mark.parametrize("r", [1e-39, 2.0 ** -127, 2.0 ** 127, float("inf"), float("nan"), 0.0, -2.0])
def test_a_repetition_whose_reciprocal_has_fewer_bits_is_refused(r):
    with pytest.raises(ValueError, match="repetition"):
        ops.process_logits(torch.zeros(2, 8), torch.zeros(2, 4, dtype=torch.int32), repetition=r)


@pytest.mark.parametrize("r", [2.0 ** -126, 3e-38, 2.0 ** 126, 5e37])
def test_the_ends_of_the_range(r):
    x = torch.tensor([[1e-3, -1e-3, 0.0, 5.0]])
    t = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want, off = oracle.logits(x, t, r=r)
    oracle.close(ops.process_logits(x, t, repetition=r), want, off)


@pytest.mark.parametrize("kw", [dict(repetition=1.5), dict(presence=0.1), dict(frequency=-0.1), dict(repetition=torch.ones(2)),
                                dict(presence=torch.zeros(2), bias=torch.zeros(8))], ids=lambda k: "-".join(k))
def test_a_choice_with_penalties_and_nothing_to_count_is_refused(kw):
    with pytest.raises(ValueError, match="next_tokens"):
        ops.next_tokens(torch.zeros(2, 8), **kw)
    ops.next_tokens(torch.zeros(2, 8), repetition=1.0, presence=0, frequency=0.0)


@pytest.mark.parametrize("default", [torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_numbers_keep_their_bits_whatever_the_default_type(default, dtype):
    x = torch.randn(3, 40, dtype=torch.float64).to(dtype)
    t = torch.randint(0, 40, (3, 30), dtype=torch.int32)
    kw = dict(r=1.2345678, p=0.3333333, f=0.1234567)
    want, off = oracle.logits(x, t, **kw)
    if dtype is torch.float64:             # 64 bits throughout: six operations, each off by half a step of what it works on
        off = 6 * 2.0 ** -53 * (x.abs() + 30)
    torch.set_default_dtype(default)
    try:
        got = ops.process_logits(x, t, repetition=kw["r"], presence=kw["p"], frequency=kw["f"])
    finally:
        torch.set_default_dtype(torch.float32)
    assert got.dtype is dtype
    oracle.close(got, want, off)


@pytest.mark.parametrize("dtype", [torch.int32, torch.uint8, torch.float32])
def test_masks_of_numbers(dtype):
    mask = torch.tensor([[0, 2, 1, 0, 3] * 9, [5, 0, 0, 0, 0] * 9], dtype=dtype)
    if dtype.is_floating_point:
        mask[0, 1] = 0.5
    assert torch.equal(ops.pack_allowed(mask), ops.pack_allowed(mask != 0))
