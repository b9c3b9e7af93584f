"""Generation over a paged cache on the CPU: batches of prompts of different lengths, chunks, penalties and masks, the account of pages."""
import pytest
import torch

from ghost_flow_b200 import ops
from ghost_flow_b200.models import GPTConfig, GPTForCausalLM, LLaMAConfig, LLaMAForCausalLM, PagedKVCache


def _model(interleaved=False):
    torch.manual_seed(0)
    cfg = LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=32, rope_interleaved=interleaved, initializer_range=0.3)
    return LLaMAForCausalLM(cfg, dtype=torch.float32).eval()


@pytest.mark.parametrize("chunk", [1, 5, 7, 1000])
@pytest.mark.parametrize("page", [4, 16])
def test_prompts_of_different_lengths_continue_as_each_alone(chunk, page):
    m = _model(page == 4)
    prompts = [torch.randint(0, 97, (n,)) for n in (1, 9, 4, 17)]
    got = m.generate_batch(prompts, 6, page_size=page, chunk_tokens=chunk)
    for t, g in zip(prompts, got):
        assert torch.equal(g, m.generate(t[None], 6)[0])


def test_logits_over_pages_are_those_of_the_model():
    m = _model()
    a, b = torch.randint(0, 97, (12,)), torch.randint(0, 97, (7,))
    cache = m.new_paged_cache(8, 8)
    cache.reserve("a", 12)
    cache.reserve("b", 7)
    x = m.forward_pages(torch.cat((a[:5], b[:7])), cache, cache.batch("ab", [5, 7], [5, 7]))
    y = m.forward_pages(a[5:], cache, cache.batch("a", [12], [7]))
    with torch.no_grad():
        want = m(a[None])[0], m(b[None])[0]
    assert torch.allclose(torch.cat((x[:5], y)), want[0], atol=1e-4) and torch.allclose(x[5:], want[1], atol=1e-4)


def test_nothing_to_do_and_what_is_refused():
    m = _model()
    t = torch.randint(0, 97, (3,))
    assert m.generate_batch([], 4) == [] and torch.equal(m.generate_batch([t], 0)[0], t)
    for prompts, kw in (([t, t[:0]], {}), ([t], dict(chunk_tokens=0))):
        with pytest.raises(ValueError):
            m.generate_batch(prompts, 2, **kw)


def test_account_of_pages():
    c = PagedKVCache(1, 5, 4, 1, 8)
    c.reserve("a", 9)
    assert c.free_pages == 2
    with pytest.raises(RuntimeError, match="are free"):
        c.reserve("b", 9)
    assert c.free_pages == 2
    c.reserve("a", 12)                     # has them already
    c.reserve("b", 8)
    b = c.batch(["b", "a"], [3, 12], [3, 1])
    assert b.lens.tolist() == [3, 12] and b.cu.tolist() == [0, 3, 4] and b.longest == 12
    used = b.table[0, :2].tolist() + b.table[1].tolist()
    assert sorted(used) == [0, 1, 2, 3, 4] and b.table[0, 2] == -1
    for who, n in (("a", 13), ("c", 1)):
        with pytest.raises(ValueError, match="not room"):
            c.batch([who], [n])
    for who, lens, new in ((["a"], [3, 4], None), (["a"], [3], [1, 1]), (["a"], [3], [4]), (["a"], [3], [-1]), (["a"], [-1], None)):
        with pytest.raises(ValueError):
            c.batch(who, lens, new)
    empty = c.batch(["nobody", "b"], [0, 8])                  # an empty slot
    assert empty.lens.tolist() == [0, 8] and empty.table[0].tolist() == [-1, -1]
    c.release("a")
    assert c.free_pages == 3
    one = c.batch(["b"], [4])
    assert one.cu is None
    one.advance()
    assert one.lens.tolist() == [5] and one.longest == 5


@pytest.mark.parametrize("kind", ["llama", "gpt"])
def test_penalties_and_masks_while_generating(kind):
    if kind == "llama":
        m = _model()
    else:
        torch.manual_seed(0)
        m = GPTForCausalLM(GPTConfig(vocab_size=97, n_positions=64, n_embd=32, n_layer=1, n_head=2, n_inner=64, dropout=0.0)).eval()
    ids = torch.randint(0, 97, (2, 5))
    plain = m.generate(ids, 8)
    assert torch.equal(m.generate(ids, 8, repetition=1.0), plain)
    # a penalty that outweighs everything: no token of the row comes again
    for kw in (dict(presence=1e4), dict(frequency=1e4), dict(repetition=1e6, presence=1e4)):
        for row in m.generate(ids, 8, **kw)[:, 5:]:
            assert len(set(row.tolist())) == 8
    ok = torch.zeros(97, dtype=torch.bool)
    ok[[3, 5]] = True
    assert set(m.generate(ids, 8, allowed=ops.pack_allowed(ok))[:, 5:].flatten().tolist()) <= {3, 5}
    bias = torch.zeros(97)
    bias[7] = 1e6
    assert (m.generate(ids, 4, bias=bias)[:, 5:] == 7).all()
    assert m.generate(ids, 4, temperature=0.7, presence=0.5).shape == (2, 9)
    if kind == "llama":
        for a, b in zip(m.generate_batch(list(ids), 8, presence=1e4), m.generate(ids, 8, presence=1e4)):
            assert torch.equal(a, b)
