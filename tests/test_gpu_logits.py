"""The kernel between logits and the choice of a token against its definition in 64 bits."""
import pytest
import torch

import _paged_oracle as oracle
from test_paged_cpu import _penalties

pytestmark = pytest.mark.gpu


def _check(x, want_of=None, **kw):
    from ghost_flow_b200 import ops

    names = dict(tokens="tokens", token_lens="lens", generated_from="first", repetition="r", presence="p", frequency="f", bias="bias",
                 allowed="allowed")
    o = {names[k]: (v.cpu() if torch.is_tensor(v) else v) for k, v in kw.items()}
    if "allowed" in kw:
        kw["allowed"] = ops.pack_allowed(kw["allowed"])
    want, off = oracle.logits(x, **o)
    before = x.clone()
    got = ops.process_logits(x, **kw)
    oracle.close(got, want, off)
    assert torch.equal(x.nan_to_num(3), before.nan_to_num(3))
    y = torch.full((x.shape[0], x.shape[1] + 9), 7.0, dtype=x.dtype, device=x.device)       # rows elsewhere, on any boundary
    ops.process_logits(x, **kw, out=y[:, 3:-6])
    assert torch.equal(y[:, 3:-6].nan_to_num(3), got.nan_to_num(3)) and (y[:, :3] == 7).all() and (y[:, -6:] == 7).all()
    ops.process_logits(x, **kw, out=x)
    assert torch.equal(x.nan_to_num(3), got.nan_to_num(3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 7, 31, 100, 1000, 8192, 8200, 16385, 50257])
@pytest.mark.parametrize("pitch", ["dense", "padded", "odd"])
def test_everything_at_once(dtype, V, pitch):
    B = 3
    ld = {"dense": V, "padded": (V + 63) // 64 * 64, "odd": V + 5}[pitch]
    x = torch.empty(B, ld, dtype=dtype, device="cuda")[:, :V]
    x.copy_(4 * torch.randn(B, V, device="cuda"))
    tokens, lens, first, r, p, f = _penalties(B, V, 300, device="cuda")
    ok, bias = torch.rand(B, V, device="cuda") < 0.6, torch.randn(B, V, device="cuda")
    ok[1] = False
    _check(x.clone(memory_format=torch.preserve_format) if pitch == "dense" else x, tokens=tokens, token_lens=lens, generated_from=first,
           repetition=r, presence=p, frequency=f, bias=bias, allowed=ok)


@pytest.mark.parametrize("kind", ["nothing", "numbers", "prompt only", "no tokens", "int32", "one bias", "one mask", "expanded", "long"])
def test_one_at_a_time(kind):
    B, V = 5, 9001
    x = 3 * torch.randn(B, V, device="cuda").bfloat16()
    tokens, lens, first, r, p, f = _penalties(B, V, 64 if kind != "long" else 20000, device="cuda")
    kw = {"nothing": {}, "numbers": dict(tokens=tokens, repetition=1.2, presence=0.5, frequency=0.25),
          "prompt only": dict(tokens=tokens, generated_from=torch.full_like(lens, 64), repetition=r, presence=p, frequency=f),
          "no tokens": dict(tokens=tokens, token_lens=torch.zeros_like(lens), repetition=r, presence=p),
          "int32": dict(tokens=tokens.int(), token_lens=lens, repetition=r, frequency=f), "one bias": dict(bias=torch.randn(V, device="cuda")),
          "one mask": dict(allowed=torch.rand(V, device="cuda") < 0.5),
          "expanded": dict(bias=torch.randn(1, V, device="cuda").expand(B, V)),
          "long": dict(tokens=tokens, repetition=r, presence=p, frequency=f)}[kind]
    _check(x, **kw)


def test_special_values():
    """Infinities and NaN go through as the formula has them; lengths and starts outside the rows are bounded."""
    from ghost_flow_b200 import ops

    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1.0, -1.0, 2.0]], device="cuda").repeat(2, 1)
    tokens = torch.tensor([[0, 1, 2, 3, 4, 5, 6, 5], [5, 5, 5, 5, 5, 5, 5, 5]], device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.process_logits(x, tokens, ints(100, -3), ints(-9, 0), repetition=2.0, presence=0.5, frequency=0.25)
    assert got[0].isnan().tolist() == [False, False, True] + [False] * 5
    assert got[0, [0, 1, 3, 4, 5, 6, 7]].tolist() == [inf, -inf, -0.75, -0.75, 0.5 - 1.0, -2.75, 2.0]
    assert torch.equal(got[1].nan_to_num(3), x[1].nan_to_num(3))
    bias = torch.zeros(8, device="cuda")
    bias[[0, 5]] = -inf
    got = ops.process_logits(x, bias=bias)
    assert got[0, 0].isnan() and got[0, 5] == -inf


def test_replayed_and_on_another_stream():
    from ghost_flow_b200 import ops

    x = torch.randn(4, 5000, device="cuda")
    tokens, lens, first, r, p, f = _penalties(4, 5000, 50, device="cuda")
    kw = dict(tokens=tokens, token_lens=lens, generated_from=first, repetition=r, presence=p, frequency=f)
    ops.process_logits(x, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.process_logits(x, **kw)
    lens.fill_(50)
    x.mul_(2)
    g.replay()
    assert torch.equal(y, ops.process_logits(x, **kw))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        z = ops.process_logits(x, **kw)
    torch.cuda.synchronize()
    assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [32767, 32768, 70001])
@pytest.mark.parametrize("pitch", [0, 3])
def test_long_histories_of_few_tokens(dtype, L, pitch):
    """Counts up to the whole history: one token all along, and one only in the prompt."""
    B, V = 3, 20011
    x = (3 * torch.randn(B, V + pitch, device="cuda")).to(dtype)[:, :V]
    tokens = 500 * torch.randint(0, 41, (B, L), device="cuda")
    tokens[0] = 7                                        # c = L
    tokens[1, :L // 2], tokens[1, L // 2:] = 20010, 6
    first = torch.tensor([0, L // 2, L - 3], dtype=torch.int32, device="cuda")
    kw = dict(tokens=tokens, generated_from=first, repetition=1.3, presence=0.5, frequency=2 ** -14)
    _check(x, **kw)
    _check(x, **kw, bias=torch.randn(V, device="cuda"), allowed=torch.rand(B, V, device="cuda") < 0.5)
