"""sample_tokens and the choices of next_tokens and of generation on the CPU, and arguments that are refused."""
import pytest
import torch

import _sample_oracle as oracle
from ghost_flow_b200 import ops
from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM
from ghost_flow_b200.ops import _lib

INF, NAN = float("inf"), float("nan")


def _rows(kind, B, V):
    r = torch.randn(B, V)
    return {"random": 3 * r, "flat": 0.01 * r, "equal": torch.zeros(B, V), "two": (r > 0).float(), "far": 1e4 * r,
            "masked": torch.where(torch.rand(B, V) < 0.7, -INF, 2 * r)}[kind]


@pytest.mark.parametrize("kind", ["random", "flat", "equal", "two", "far", "masked"])
@pytest.mark.parametrize("choice", [{}, dict(top_k=3), dict(top_p=0.75), dict(min_p=0.25), dict(top_k=1), dict(top_k=90), dict(top_p=2.0 ** -20),
                                    dict(top_k=7, top_p=0.5, min_p=0.125, temperature=0.5), dict(temperature=0.0), dict(temperature=16.0)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_against_the_definition(kind, choice, dtype):
    x, u = _rows(kind, 5, 37).to(dtype), torch.rand(5)
    x[:, 0] = 0.0                                         # (a masked row of one number at least)
    got = ops.sample_tokens(x, u, **choice)
    assert got.shape == (5, 1) and got.dtype is torch.int64
    assert got.flatten().tolist() == oracle.tokens(x, u, **choice)


def test_a_choice_of_each_row():
    x, u = 2 * torch.randn(6, 50), torch.rand(6)
    c = dict(temperature=torch.tensor([0.0, 1.0, 0.5, 2.0, 1.0, 0.25]), top_k=torch.tensor([0, 1, 5, 50, 60, 2], dtype=torch.int32),
             top_p=torch.tensor([0.5, 1.0, 0.5, 0.25, 0.75, 1.0]), min_p=torch.tensor([0.0, 0.0, 0.5, 0.0, 0.125, 1.0]))
    assert ops.sample_tokens(x, u, **c).flatten().tolist() == oracle.tokens(x, u, **c)


def test_rows_without_probabilities_and_the_ends_of_the_random_numbers():
    x = torch.randn(5, 20)
    x[0, [4, 9]], x[1, [3, 8]], x[2], x[3] = NAN, INF, -INF, -INF
    x[3, 11] = 0.0
    u = torch.tensor([0.5, 0.5, 0.5, 0.9, 0.0])
    assert ops.sample_tokens(x, u, top_p=0.5).flatten().tolist()[:4] == [4, 3, -1, 11]
    y = torch.tensor([[-30.0, 0.0, 1.0, -50.0]])
    assert ops.sample_tokens(y, torch.tensor([0.0])) == 0                           # however unlikely
    assert ops.sample_tokens(y, torch.tensor([1 - 2.0 ** -24])) == 2


def test_shares_follow_the_weights():
    """u walks over a grid: every token comes as often as its share of what stays says, to a step of the grid."""
    x = torch.tensor([[0.0, 2.0, 1.0, -1.0, 1.0]])
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = ops.sample_tokens(x.expand(n, 5).contiguous(), u, temperature=0.5, top_k=4).flatten().bincount(minlength=5)
    p = torch.softmax(torch.tensor([0.0, 2.0, 1.0, -INF, 1.0], dtype=torch.float64) / 0.5, 0) * n
    assert ((got - p).abs() <= 1).all() and got[3] == 0


@pytest.mark.parametrize("kw", [dict(temperature=-0.5), dict(temperature=NAN), dict(top_k=-1), dict(top_k=2.5), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=NAN),
                                dict(min_p=-0.1), dict(min_p=1.1), dict(u=0.5), dict(u=torch.rand(2)), dict(u=torch.rand(3).double()),
                                dict(u=torch.rand(3, device="meta")), dict(temperature=torch.ones(2)), dict(temperature=torch.ones(3, 1)),
                                dict(top_k=torch.ones(3)), dict(top_k=torch.ones(3, dtype=torch.int64)), dict(top_p=torch.ones(3).bfloat16()),
                                dict(min_p=torch.ones(())), dict(logits=torch.randn(9)), dict(logits=torch.ones(3, 9, dtype=torch.int64)),
                                dict(logits=torch.randn(3, 0))], ids=lambda k: "-".join(k))
def test_refusals(kw):
    with pytest.raises(ValueError, match="sample_tokens"):
        ops.sample_tokens(**{"logits": torch.randn(3, 9), "u": torch.rand(3), **kw})


def test_no_rows():
    assert ops.sample_tokens(torch.randn(0, 9), torch.rand(0)).shape == (0, 1)


def test_the_entry_point_refuses_before_it_launches():
    import struct

    lib, P = _lib.cuda_lib(), 1 << 20
    good = dict(x=P, ldx=64, dtype=0, B=3, V=50, u=P, t=0, p=0, m=0, k=0, t0=1.0, p0=1.0, m0=0.0, k0=0, out=P)
    for kw in (dict(x=0), dict(u=0), dict(out=0), dict(B=0), dict(B=1 << 31), dict(V=0), dict(V=(1 << 20) + 1), dict(dtype=3), dict(dtype=-1)):
        v = {**good, **kw}
        assert lib.gf_sample_tokens(struct.pack("10q3d2q", *(v[n] for n in "x ldx dtype B V u t p m k t0 p0 m0 k0 out".split())), None) == -1
    assert lib.gf_sample_tokens(None, None) == -1


def test_the_module_leaves_what_is_not_its():
    calls = _lib.calls()
    assert calls.sample(torch.randn(2, 9), torch.rand(2), 1.0, 0, 1.0, 0.0) is None
    for f in (calls.sample, calls.run_sample, calls.bind_more):
        with pytest.raises(TypeError, match="arguments"):
            f()
    with pytest.raises(TypeError, match="not a call"):
        calls.run_sample(b"x", torch.zeros(2), 0)


def test_next_tokens_with_choices():
    x, u = 2 * torch.randn(4, 30), torch.rand(4)
    choice = dict(top_k=5, top_p=0.75, min_p=0.125)
    assert torch.equal(ops.next_tokens(x, 0.5, u=u, **choice), ops.sample_tokens(x, u, 0.5, **choice))
    torch.manual_seed(3)
    a = ops.next_tokens(x, 0.5, top_k=5)
    torch.manual_seed(3)
    assert torch.equal(a, ops.sample_tokens(x, torch.rand(4), 0.5, 5))
    assert torch.equal(ops.next_tokens(x, top_k=5), x.argmax(-1, keepdim=True))                    # temperature 0
    allowed = torch.zeros(4, 30, dtype=torch.bool)
    allowed[0, 7] = allowed[2, [3, 4]] = allowed[3] = True
    got = ops.next_tokens(x, 0.5, allowed=ops.pack_allowed(allowed), u=u, **choice).flatten().tolist()
    assert got[:2] == [7, -1] and got[2] in (3, 4)
    assert got == oracle.tokens(x.masked_fill(~allowed, -INF), u, 0.5, **choice)


@pytest.mark.parametrize("pages", [False, True])
def test_generation_among_the_likeliest_alone_is_greedy(pages):
    m = LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=4,
                                     num_key_value_heads=2, max_position_embeddings=32, initializer_range=0.3), dtype=torch.float32).eval()
    ids = torch.randint(0, 97, (2, 5))
    run = (lambda **c: torch.stack(m.generate_batch(list(ids), 4, page_size=16, **c))) if pages else (lambda **c: m.generate(ids, 4, **c))
    assert torch.equal(run(temperature=0.8, top_k=1), run())
    assert torch.equal(run(temperature=0.8, min_p=1.0), run())
    torch.manual_seed(1)
    a = run(temperature=5.0, top_k=40, top_p=0.9)
    torch.manual_seed(1)
    assert torch.equal(a, run(temperature=5.0, top_k=40, top_p=0.9))


@pytest.mark.parametrize("kw", [{}, dict(top_k=5), dict(top_p=0.5), dict(min_p=0.9), dict(top_p=0.7, min_p=0.3)], ids=lambda k: "-".join(k) or "none")
def test_temperatures_without_end(kw):
    """At an infinite temperature what has a probability has the same; what has none still has none."""
    x = torch.tensor([[-INF, 2.0, -INF, 1.0, -3.0, -INF, 0.5, 7.0]]).repeat(64, 1)
    u = (torch.arange(64) + 0.5) / 64
    order = [7, 1, 3, 6, 4]
    kept = order[:3] if kw.get("top_p") == 0.5 else order[:4] if kw.get("top_p") == 0.7 else order
    want = [sorted(kept)[int(v * len(kept))] for v in u.tolist()]
    for t in (INF, torch.full((64,), INF), 3e38):
        assert ops.sample_tokens(x, u, t, **kw).flatten().tolist() == want, t
