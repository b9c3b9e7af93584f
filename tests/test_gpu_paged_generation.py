"""A LLaMA model over a paged cache on the kernels: chunks, batches of different lengths, single tokens, a captured step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _models(heads, kv_heads, hidden):
    from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM

    cfg = LLaMAConfig(vocab_size=500, hidden_size=hidden, intermediate_size=512, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, max_position_embeddings=512, initializer_range=0.05)
    m = LLaMAForCausalLM(cfg, device="cuda", dtype=torch.bfloat16).eval()
    ref = LLaMAForCausalLM(cfg, device="cuda", dtype=torch.float32).eval()
    ref.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    return m, ref


@pytest.mark.parametrize("heads,kv_heads,hidden", [(4, 2, 256), (8, 8, 512), (4, 1, 512)])
def test_logits_are_as_near_to_32_bits_as_those_of_the_dense_cache(heads, kv_heads, hidden, kernel_status):
    m, ref = _models(heads, kv_heads, hidden)
    seqs = [torch.randint(0, 500, (n,), device="cuda") for n in (1, 130, 37, 300, 16, 5, 64, 200, 33)]
    with torch.no_grad():
        want = [ref(t[None])[0] for t in seqs]
        dense = [m(t[None])[0].float() for t in seqs]
        cache = m.new_paged_cache(200, 16)
        for b, t in enumerate(seqs):
            cache.reserve(b, t.numel())
        got, at = [[] for _ in seqs], [0] * len(seqs)
        for n in (1, 17, 1, 64, 1, 1, 300):             # chunks and single tokens, sequences that have ended left out
            new = {b: min(n if b % 3 else 1, t.numel() - at[b]) for b, t in enumerate(seqs) if at[b] < t.numel()}
            if n == 300:
                new = {b: seqs[b].numel() - at[b] for b in new}
            if not new:
                continue
            batch = cache.batch(new, [at[b] + k for b, k in new.items()], None if set(new.values()) == {1} else new.values())
            x = m.forward_pages(torch.cat([seqs[b][at[b]:at[b] + k] for b, k in new.items()]), cache, batch)
            for b, part in zip(new, x.split(list(new.values()))):
                got[b].append(part.float())
                at[b] += new[b]
    for g, d, w in zip(got, dense, want):
        # roundings to bf16 of the same sizes at the same places, whichever cache is used
        assert (torch.cat(g) - w).norm() <= 2 * (d - w).norm() + 1e-3 * w.norm()


def test_generate_batch_runs_and_keeps_prompts(kernel_status):
    m, _ = _models(4, 2, 256)
    prompts = [torch.randint(0, 500, (n,)) for n in (3, 70, 18, 129)]
    for kw in ({}, dict(chunk_tokens=50), dict(temperature=0.8, presence=0.3, repetition=1.2), dict(page_size=16)):
        out = m.generate_batch(prompts, 12, **kw)
        for t, o in zip(prompts, out):
            assert o.shape == (t.numel() + 12,) and torch.equal(o[:t.numel()].cpu(), t) and 0 <= int(o.min()) and int(o.max()) < 500


def test_captured_step_of_a_server(kernel_status):
    """One step of a batch with an empty slot, captured: append, attend, penalties, choice; replayed as the lengths grow."""
    from ghost_flow_b200 import ops

    m, _ = _models(4, 2, 256)
    cache = m.new_paged_cache(64, 16)
    for b in range(3):
        cache.reserve(b, 100)
    prompts = [torch.randint(0, 500, (n,), device="cuda") for n in (9, 40)]
    logits = m.forward_pages(torch.cat(prompts), cache, cache.batch(range(2), [9, 40], [9, 40]), torch.tensor([8, 48], device="cuda"))
    first = torch.cat((logits.argmax(-1), torch.zeros(1, dtype=torch.long, device="cuda")))
    bias = torch.randn(500, device="cuda")

    def run(step, n):
        ids, batch = first.clone(), cache.batch(range(3), [10, 41, 0])
        grows = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")

        def body():
            x = m.forward_pages(ids, cache, batch)
            ids.copy_(ops.next_tokens(x, 0.0, bias=bias).view(-1))
            batch.lens.add_(grows)

        return step(body, ids, n)

    def eager(body, ids, n):
        out = []
        for _ in range(n):
            body()
            out.append(ids[:2].clone())
        return torch.stack(out)

    def captured(body, ids, n):
        keep = [(k.clone(), v.clone()) for k, v in cache.pools]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            body()
        for (k, v), (a, b) in zip(cache.pools, keep):
            k.copy_(a)
            v.copy_(b)
        out = []
        for _ in range(n):
            g.replay()
            out.append(ids[:2].clone())
        return torch.stack(out)

    with torch.no_grad():
        want = run(eager, 20)
        assert torch.equal(run(captured, 20), want)
