"""Rotation tables of a model that meets longer sequences."""
import gc
import weakref

import torch

from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM


def test_tables_that_a_captured_step_may_read_are_not_given_back():
    m = LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=4,
                                     num_key_value_heads=2, max_position_embeddings=32), dtype=torch.float32)
    old = [weakref.ref(t) for t in m.model.rope(10, "cpu")]
    at = [r().data_ptr() for r in old]
    values = [r().clone() for r in old]
    new = m.model.rope(100, "cpu")
    gc.collect()
    assert new[0].shape[0] >= 100 and [r() is not None and r().data_ptr() for r in old] == at
    assert all(torch.equal(r(), v) and torch.equal(n[:32], v) for r, v, n in zip(old, values, new))
