"""A captured step of a server: what a replay reads, that replay or one before it has written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model():
    from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM

    cfg = LLaMAConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=512, initializer_range=0.05)
    return LLaMAForCausalLM(cfg, device="cuda", dtype=torch.bfloat16).eval()


@pytest.mark.parametrize("page", [16, 64])
def test_replays_append_what_they_read(page, kernel_status):
    from ghost_flow_b200 import ops

    m, lens, steps = _model(), [9, 40], 20
    cache = m.new_paged_cache(256 // page * 3, page)
    for k, v in cache.pools:               # rows that nobody has written
        k.fill_(float("nan"))
        v.fill_(float("nan"))
    for b in range(3):
        cache.reserve(b, 100)
    prompts = [torch.randint(0, 500, (n,), device="cuda") for n in lens]
    bias = torch.randn(500, device="cuda")
    with torch.no_grad():
        logits = m.forward_pages(torch.cat(prompts), cache, cache.batch(range(2), lens, lens), torch.tensor([8, 48], device="cuda"))
        first = torch.cat((logits.argmax(-1), torch.zeros(1, dtype=torch.long, device="cuda")))
        keep = [(k.clone(), v.clone()) for k, v in cache.pools]
        grows = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
        runs = []
        for captured in (False, True):
            for (k, v), (a, b) in zip(cache.pools, keep):
                k.copy_(a)
                v.copy_(b)
            ids, batch, seen = first.clone(), cache.batch(range(3), [10, 41, 0]), []

            def body():
                x = m.forward_pages(ids, cache, batch)
                ids.copy_(ops.next_tokens(x, bias=bias).view(-1))
                batch.lens.add_(grows)
                return x

            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    x = body()
            for _ in range(steps):
                if captured:
                    graph.replay()
                else:
                    x = body()
                seen.append((ids[:2].clone(), x[:2].clone()))
            runs.append((seen, [(k.clone(), v.clone()) for k, v in cache.pools]))
        for (ids, x), (ids_g, x_g) in zip(runs[0][0], runs[1][0]):
            assert x.isfinite().all() and torch.equal(ids, ids_g) and torch.equal(x, x_g)
        for (k, v), (k_g, v_g), (k0, v0) in zip(runs[0][1], runs[1][1], keep):
            for a, b, c in ((k, k_g, k0), (v, v_g, v0)):
                assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) and int((c.isnan() & ~a.isnan()).sum()) == 2 * steps * c[0, 0].numel()
