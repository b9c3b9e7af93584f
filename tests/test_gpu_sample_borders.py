"""sample_tokens where numbers end: temperatures at which neighbouring numbers of 32 bits are far apart, weights below the last
bit, random numbers of 0."""
import pytest
import torch

import _sample_oracle as oracle

pytestmark = pytest.mark.gpu
INF = float("inf")


def _neighbours(top, n):
    """The float below ``top``, the one below that, and so on."""
    x = torch.tensor([top])
    out = []
    for _ in range(n):
        x = torch.nextafter(x, torch.tensor([-INF]))
        out.append(x.item())
    return out


# Weights of the neighbours of the largest logit are 2^-2 .. 2^-137 of it (the exponents are their distance over the temperature): what a draw takes goes by far less
# than the 2^-24 between two random numbers that are tried.
@pytest.mark.parametrize("top,temperature", [(12.0, 1e-8), (12.0, 2e-8), (20.0, 1e-8), (20.0, 2e-8), (20.0, 1e-6), (100.0, 1e-7), (1e5, 1e-4), (1e5, 1e-2), (-20.0, 2e-8), (-3e-3, 4e-12)])
@pytest.mark.parametrize("choice", [{}, dict(top_k=3), dict(top_k=29990), dict(top_p=0.9), dict(top_k=8, top_p=0.7), dict(min_p=1e-3)], ids=lambda c: "-".join(c) or "none")
@pytest.mark.parametrize("V", [40, 30000])
def test_neighbouring_numbers_at_small_temperatures(top, temperature, choice, V):
    from ghost_flow_b200 import ops

    near = _neighbours(top, 11)
    x = torch.full((4, V), top - abs(top) / 2 - 1)
    for b in range(4):
        at = torch.randperm(V)[:12]
        x[b, at] = torch.tensor([top, *near])
    x, u = x.cuda(), torch.tensor([0.125, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    want = oracle.tokens(x, u, temperature, **choice)
    assert ops.sample_tokens(x, u, temperature, **choice).flatten().tolist() == want
    rows = torch.full((4,), temperature, device="cuda")                  # (of 32 bits: not quite the same temperature)
    assert ops.sample_tokens(x, u, rows, **choice).flatten().tolist() == oracle.tokens(x, u, rows, **choice)


# The entries in front of the likeliest one hold V w / 2 of the sum: next to nothing of it, less than the 2^-24 between two random numbers (-60 and less), or tokens of their
# own (-20, of which 2^-24 and 5 2^-24 take one, 29 and more of them further on). A random number of 0 takes the first entry that has a weight at all, down to 2^-1074.
@pytest.mark.parametrize("V,dtype,choice", [(V, t, c) for V, t in ((40, torch.float32), (50257, torch.bfloat16), (128256, torch.float32))
                                            for c in ({}, dict(top_p=0.9999), dict(top_k=30000), dict(top_k=12), dict(min_p=1e-300))] +
                         [(1 << 20, torch.bfloat16, {}), (1 << 20, torch.float32, dict(min_p=1e-300))], ids=str)
def test_a_long_tail_of_little_weight(V, dtype, choice):
    from ghost_flow_b200 import ops

    tails, us = [-20.0, -60.0, -740.0, -800.0][:4 if V < 1 << 20 else 2], [0.0, 2.0 ** -24, 5 * 2.0 ** -24]
    x = torch.tensor(tails).repeat_interleave(3)[:, None].repeat(1, V)
    x[:, 0] = -INF
    x[:, V // 2], x[:, V // 2 + 1] = 0.0, -1.0
    x = x.to(dtype).cuda()
    u = torch.tensor(us * len(tails), device="cuda")
    got = ops.sample_tokens(x, u, **choice).flatten().tolist()
    assert got == oracle.tokens(x, u, **choice)


# As above, with the tail behind the token too and several rows to a call, which clusters take: borders of the tail's own tokens.
@pytest.mark.parametrize("V", [8000, 50257])
def test_borders_within_a_tail(V):
    from ghost_flow_b200 import ops

    x = torch.full((4, V), -16.0, device="cuda")              # 1.1e-7 each: a token of the tail is two steps of a random number wide
    x[:, V // 3] = 0.0
    # in the middle of the 5th, 700th, 2000th and last but one token's share
    w, total = torch.exp(torch.tensor(-16.0, dtype=torch.float64)).item(), 1 + (V - 1) * torch.exp(torch.tensor(-16.0, dtype=torch.float64)).item()
    want = [4, 699, 1999, V - 2]
    at = [(v + 0.5) * w / total for v in want[:3]] + [1 - 1.5 * w / total]
    assert ops.sample_tokens(x, torch.tensor(at, device="cuda")).flatten().tolist() == want
