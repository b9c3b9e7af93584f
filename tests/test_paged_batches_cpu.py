"""Batches of a paged cache: the same sequence more than once."""
import pytest
import torch

from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM, PagedKVCache


def _cache():
    c = PagedKVCache(1, 6, 4, 1, 8)
    c.reserve("a", 12)
    c.reserve("b", 8)
    return c


@pytest.mark.parametrize("who,lens,new", [("aa", [5, 5], None), ("aba", [5, 3, 5], None), ("aa", [5, 8], [5, 4]), ("aa", [8, 5], [4, 5]),
                                          ("aa", [8, 5], [8, 1]), ("aba", [8, 8, 8], [1, 8, 8])])
def test_two_tokens_are_not_written_to_the_same_row(who, lens, new):
    with pytest.raises(ValueError, match="more than once"):
        _cache().batch(who, lens, new)


def test_parts_of_a_sequence_and_empty_slots_stand_beside_each_other():
    c = _cache()
    b = c.batch("aab", [5, 8, 3], [5, 3, 3])
    assert b.lens.tolist() == [5, 8, 3] and b.cu.tolist() == [0, 5, 8, 11] and torch.equal(b.table[0], b.table[1])
    assert c.batch("aa", [5, 6], None).lens.tolist() == [5, 6]
    assert c.batch([None, None, "a"], [0, 0, 4]).lens.tolist() == [0, 0, 4]
    assert c.batch("aab", [5, 5, 3], [0, 1, 1]).cu.tolist() == [0, 0, 1, 2]
    with pytest.raises(ValueError):
        c.batch([None], [-1])


def test_a_prompt_in_two_parts_of_one_batch():
    torch.manual_seed(0)
    m = LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                     num_key_value_heads=2, max_position_embeddings=32, initializer_range=0.3), dtype=torch.float32).eval()
    t = torch.randint(0, 97, (11,))
    cache = m.new_paged_cache(3, 4)
    cache.reserve("a", 11)
    got = m.forward_pages(t, cache, cache.batch("aa", [6, 11], [6, 5]))
    with torch.no_grad():
        assert torch.allclose(got, m(t[None])[0], atol=1e-4)
