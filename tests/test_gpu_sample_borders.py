"""sample_tokens where numbers end: temperatures at which neighbouring numbers of 32 bits are far apart."""
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
