"""Rotation tables that a gradient is wanted of, and the paths that take them."""
import pytest
import torch

import _paged_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("learned", ["cos", "sin", "both"])
def test_a_gradient_of_the_tables_alone_is_recorded(learned, kernel_status):
    from ghost_flow_b200 import ops

    H, Hk, D = 4, 2, 64
    s = oracle.batch([9, 5], [3, 1], H, Hk, D, 16, device="cuda")
    tables = [t.clone() for t in ops.rope_tables(16, D, 1e4, "cuda")]
    args = s["table"], s["lens"], s["cu"]
    plain = ops.rope_qkv_to_pages(s["qkv"], H, Hk, *tables, s["kp"], s["vp"], *args)
    for name, t in zip(("cos", "sin"), tables):
        t.requires_grad_(learned in (name, "both"))
    q = ops.rope_qkv_to_pages(s["qkv"], H, Hk, *tables, s["kp"].clone(), s["vp"].clone(), *args)
    assert q.requires_grad and not plain.requires_grad
    q.float().sum().backward()
    x, y = s["qkv"][:, :H].float().chunk(2, -1)
    at = torch.tensor([6, 7, 8, 4], device="cuda")
    # q holds lo cos - hi sin and hi cos + lo sin of every head: their sum's slopes are lo + hi and lo - hi
    for t, slope in zip(tables, (x + y, x - y)):
        if not t.requires_grad:
            continue
        want = torch.zeros_like(t, requires_grad=False).index_add_(0, at, slope.sum(1))
        # H + 1 sums in 32 bits, each off by half a step of at most the sum of sizes
        off = 2 * H * 2 ** -24 * torch.zeros_like(want).index_add_(0, at, (x.abs() + y.abs()).sum(1))
        assert ((t.grad - want).abs() <= off).all()
    with torch.no_grad():
        assert torch.equal(ops.rope_qkv_to_pages(s["qkv"], H, Hk, *tables, s["kp"], s["vp"], *args), plain)


@pytest.mark.parametrize("lens,new", [([40, 9], [1, 1]), ([300, 70, 9], [33, 70, 1])])
@pytest.mark.parametrize("scale", [1e-50, -1e-50, 2e-46, 0.0])
def test_a_scale_below_all_numbers_of_32_bits(scale, lens, new, kernel_status):
    from ghost_flow_b200 import ops

    s = oracle.batch(lens, new, 8, 2, 64, 16, device="cuda")
    args = s["q"], s["kp"], s["vp"], s["table"], s["lens"], None if set(new) == {1} else s["cu"]
    oracle.close(ops.paged_attention(*args, scale=scale), *oracle.attention(s, scale))
    with pytest.raises(ValueError, match="scale"):
        ops.paged_attention(*args, scale=2.0 ** 127)
