"""Pools and logits whose offsets pass 32 bits, sequences longer than 2^17 keys."""
import pytest
import torch

import _paged_oracle as oracle

pytestmark = pytest.mark.gpu


def _far(s, P, H, Hk, D, page):
    """The batch over pools of P pages, of which it has the last ones."""
    used = s["kp"].shape[0]
    for n in ("kp", "vp"):
        pool = torch.empty(P, page, Hk, D, dtype=torch.bfloat16, device="cuda")
        pool[P - used:] = s[n]
        s[n] = pool
    s["table"] = torch.where(s["table"] >= 0, s["table"] + (P - used), s["table"])


@pytest.mark.parametrize("lens,new", [([70, 33], [1, 1]), ([300, 41], [170, 41])])
def test_pages_behind_two_to_the_32_bytes(lens, new, kernel_status):
    from ghost_flow_b200 import ops

    H, Hk, D, page = 32, 32, 128, 16
    P = 2 ** 31 // (page * Hk * D) + 64            # more than 2^31 elements
    s = oracle.batch(lens, new, H, Hk, D, page, device="cuda")
    small = dict(s, kp=s["kp"].clone(), vp=s["vp"].clone())
    _far(s, P, H, Hk, D, page)
    cos, sin = ops.rope_tables(512, D, 1e4, "cuda")
    got, want = [], []
    for x, out in ((s, got), (small, want)):
        q = ops.rope_qkv_to_pages(x["qkv"], H, Hk, cos, sin, x["kp"], x["vp"], x["table"], x["lens"], x["cu"])
        out += [q, ops.paged_attention(q, x["kp"], x["vp"], x["table"], x["lens"], x["cu"] if new[0] > 1 else None)]
    used = small["kp"].shape[0]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(s["kp"][P - used:].nan_to_num(9), small["kp"].nan_to_num(9))
    assert torch.equal(s["vp"][P - used:].nan_to_num(9), small["vp"].nan_to_num(9))
    small["q"] = want[0]
    oracle.close(got[1], *oracle.attention(small))


@pytest.mark.parametrize("new", [1, 5, 130])
def test_a_long_sequence(new, kernel_status):
    from ghost_flow_b200 import ops

    lens = [140001, 3]
    s = oracle.batch(lens, [new, 1], 8, 1, 64, 64, device="cuda")
    got = ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], None if new == 1 else s["cu"])
    oracle.close(got, *oracle.attention(s))


def test_logits_behind_two_to_the_31(kernel_status):
    from ghost_flow_b200 import ops

    B, V = 2 ** 31 // 50257 + 5, 50257
    x = torch.zeros(B, V, dtype=torch.bfloat16, device="cuda")
    x[-6:] = torch.randn(6, V, device="cuda")
    t = torch.randint(0, V, (B, 20), device="cuda", dtype=torch.int32)
    bias = torch.randn(V, device="cuda")
    want = ops.process_logits(x[-6:].clone(), t[-6:], repetition=1.5, presence=0.5, bias=bias)
    ops.process_logits(x, t, repetition=1.5, presence=0.5, bias=bias, out=x)
    assert torch.equal(x[-6:], want)
