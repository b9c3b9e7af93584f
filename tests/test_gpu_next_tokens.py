"""The choice of a token on the device: rows without a token, or without probabilities, stop neither the batch nor a captured step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_without_a_token_or_without_probabilities(dtype, temperature):
    from ghost_flow_b200 import ops

    x = torch.randn(5, 500, device="cuda").to(dtype)
    x[3, 9], x[4, 11] = float("nan"), float("inf")
    ok = torch.ones(5, 500, dtype=torch.bool, device="cuda")
    ok[1], ok[2] = False, False
    ok[2, 77] = True
    allowed = ops.pack_allowed(ok)
    got = ops.next_tokens(x, temperature, allowed=allowed).flatten().tolist()
    assert 0 <= got[0] < 500 and got[1:] == [-1, 77, 9, 11]
    plain = ops.next_tokens(x, temperature).flatten().tolist()
    assert min(plain) >= 0 and max(plain) < 500 and plain[3:] == [9, 11]
    torch.manual_seed(3)
    a = ops.next_tokens(x[:3], temperature, allowed=allowed[:3])
    torch.manual_seed(3)
    b = ops.next_tokens(x[:3], temperature, allowed=ops.pack_allowed(ok[[0, 0, 2]]))
    assert torch.equal(a[[0, 2]], b[[0, 2]])


def test_captured(kernel_status):
    from ghost_flow_b200 import ops

    x = torch.randn(3, 200, device="cuda")
    allowed = ops.pack_allowed(torch.ones(3, 200, dtype=torch.bool, device="cuda"))
    ops.next_tokens(x, 0.7, allowed=allowed)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampled, likeliest = ops.next_tokens(x, 0.7, allowed=allowed), ops.next_tokens(x, allowed=allowed)
    allowed[1] = 0
    x[2] = float("nan")
    g.replay()
    assert sampled[1] == likeliest[1] == -1 and sampled[2] == likeliest[2] and 0 <= int(sampled[0]) < 200 and likeliest[0] == x[0].argmax()
