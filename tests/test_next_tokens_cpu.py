"""The choice of a token on the CPU: rows that a mask or what is not a number leaves without a likeliest token, beside others."""
import pytest
import torch

from ghost_flow_b200 import ops
from ghost_flow_b200.models import GPTConfig, GPTForCausalLM, LLaMAConfig, LLaMAForCausalLM

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_row_that_nothing_is_left_of_has_no_token_and_the_others_have_theirs(temperature, dtype):
    x = torch.randn(4, 40).to(dtype)
    ok = torch.zeros(4, 40, dtype=torch.bool)
    ok[0, 3] = ok[3, [5, 39]] = True                     # rows 1 and 2: nothing
    got = ops.next_tokens(x, temperature, allowed=ops.pack_allowed(ok))
    assert got.shape == (4, 1) and got.dtype == torch.long
    assert got[0] == 3 and got[1] == got[2] == -1 and int(got[3]) in (5, 39)
    assert (ops.next_tokens(x, temperature, bias=torch.full((40,), -INF)) == -1).all()
    one = ops.next_tokens(x[:, :1], temperature, allowed=torch.tensor([[1], [0], [1], [0]], dtype=torch.int32))
    assert one.flatten().tolist() == [0, -1, 0, -1]


def test_a_row_without_a_token_changes_nothing_for_the_others():
    x = torch.randn(3, 50)
    ok = torch.rand(3, 50) < 0.5
    torch.manual_seed(5)
    want = ops.next_tokens(x, 0.9, allowed=ops.pack_allowed(ok))
    dead = ok.clone()
    dead[1] = False
    torch.manual_seed(5)
    got = ops.next_tokens(x, 0.9, allowed=ops.pack_allowed(dead))
    assert got[1] == -1 and torch.equal(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("bad,where", [(NAN, 7), (INF, 7), (-INF, 0)])
def test_rows_without_probabilities_take_the_likeliest_token(bad, where):
    x = torch.randn(2, 30)
    x[0, 7] = bad
    if bad == -INF:
        x[0] = bad
    assert ops.next_tokens(x)[0] == where
    got = ops.next_tokens(x, 0.8)
    assert got[0] == where and 0 <= int(got[1]) < 30
    assert torch.equal(ops.next_tokens(torch.tensor([[1.0, 3.0, 2.0]]), 1e-42), torch.tensor([[1]]))      # a quotient beyond 32 bits


@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("kind", ["llama", "gpt", "llama pages"])
def test_generation_goes_on_beside_a_row_that_nothing_is_left_of(kind, temperature):
    torch.manual_seed(0)
    if kind == "gpt":
        m = GPTForCausalLM(GPTConfig(vocab_size=97, n_positions=64, n_embd=32, n_layer=1, n_head=2, n_inner=64, dropout=0.0)).eval()
    else:
        m = LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                         num_key_value_heads=2, max_position_embeddings=32, initializer_range=0.3), dtype=torch.float32).eval()
    ids = torch.randint(0, 97, (3, 5))
    ok = torch.ones(3, 97, dtype=torch.bool)
    ok[1] = False
    make = lambda rows, mask: torch.stack(m.generate_batch(list(rows), 6, temperature, allowed=mask)) if kind == "llama pages" else \
        m.generate(rows, 6, temperature, allowed=mask)  # noqa: E731
    got = make(ids, ops.pack_allowed(ok))
    assert torch.equal(got[:, :5], ids) and (got[1, 5:] == -1).all()
    live = got[[0, 2], 5:]
    assert live.min() >= 0 and live.max() < 97
    if not temperature:
        assert torch.equal(got[[0, 2]], make(ids[[0, 2]], ops.pack_allowed(ok[[0, 2]])))


@pytest.mark.parametrize("kind", ["llama", "gpt", "llama pages"])
def test_tokens_are_counted_for_penalties_only(kind, monkeypatch):
    torch.manual_seed(0)
    if kind == "gpt":
        m = GPTForCausalLM(GPTConfig(vocab_size=97, n_positions=64, n_embd=32, n_layer=1, n_head=2, n_inner=64, dropout=0.0)).eval()
    else:
        m = LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=4,
                                         num_key_value_heads=2, max_position_embeddings=32), dtype=torch.float32).eval()
    seen, plain = [], ops.sampling.process_logits

    def process(logits, tokens=None, *a, **kw):
        seen.append(tokens is not None)
        return plain(logits, tokens, *a, **kw)

    monkeypatch.setattr(ops.sampling, "process_logits", process)
    ids = torch.randint(0, 97, (2, 5))
    for choice, counted in ((dict(bias=torch.zeros(97)), False), (dict(allowed=ops.pack_allowed(torch.ones(97))), False),
                            (dict(bias=torch.zeros(97), presence=0.1), True), (dict(repetition=1.5), True), (dict(frequency=0.5), True)):
        seen.clear()
        m.generate_batch(list(ids), 3, **choice) if kind == "llama pages" else m.generate(ids, 3, **choice)
        assert seen == [counted] * 3


def test_logits_of_one_row_alone():
    x = torch.tensor([0.0, 4.0, NAN])
    for temperature in (0.0, 0.5):
        assert ops.next_tokens(x[:2] * 100, temperature).tolist() == [1] and ops.next_tokens(x, temperature).tolist() == [2]
        assert ops.next_tokens(torch.zeros(0, 5), temperature).shape == (0, 1)
