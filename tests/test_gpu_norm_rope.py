"""norm_rope_qkv on the device against the definition in 64 bits: results and gradients, layouts, captured steps."""
import pytest
import torch

import _heads_oracle as oracle

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _run(B, S, H, Hk, D, n, interleaved, pos=0, norms=True, layout="dense", grads="dense", scale=1.0, eps=1e-6):
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    N = H + 2 * Hk
    cos, sin = ops.rope_tables(S + pos + 1, 2 * n, device="cuda") if n else (torch.zeros(S + pos + 1, 0, device="cuda"),) * 2
    x = scale * torch.randn(B, S, N, D, device="cuda")
    if layout == "wide":
        x = torch.cat((x, x), 2).to(BF16)[:, :, :N]
    elif layout == "sequence first":
        x = x.to(BF16).transpose(0, 1).contiguous().transpose(0, 1)
    x = x.to(BF16).requires_grad_()
    w = [(1 + 0.3 * torch.randn(D, device="cuda")).to(BF16).requires_grad_() if norms else None for _ in range(2)]
    before = _lib.launch_count()
    got = ops.norm_rope_qkv(x, H, Hk, *w, cos, sin, eps, interleaved, pos)
    assert _lib.launch_count() == before + 1
    dy = [torch.randn(B, S, m, D, device="cuda").to(BF16) for m in (H, Hk, Hk)]
    if grads == "heads first":
        dy = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in dy]
    elif grads == "one":
        dy = [g[:, :, :1, :1].expand(g.shape) for g in dy]
    leaves = [t for t in (x, *w) if t is not None]
    before = _lib.launch_count()
    d = torch.autograd.grad(got, leaves, dy)
    assert _lib.launch_count() == before + (2 if norms else 1)
    c, s = cos[pos:pos + S, None], sin[pos:pos + S, None]
    dx = []
    for i, (at, m) in enumerate(((0, H), (H, Hk))):
        part = x[:, :, at:at + m]
        want, off = oracle.heads(part, w[i], c, s, eps, interleaved)
        oracle.close(got[i], want, off + oracle.BF16_STEP * (want.abs() + off), f"part {i}")
        g, g_off, dw, dw_off = oracle.gradients(part, w[i], c, s, eps, interleaved, dy[i])
        oracle.close(d[0][:, :, at:at + m], g, g_off, f"gradient of part {i}")
        if norms:
            oracle.close(d[1 + i], dw, dw_off, f"gradient of weight {i}")
    assert torch.equal(got[2], x[:, :, H + Hk:]) and torch.equal(d[0][:, :, H + Hk:], dy[2])


@pytest.mark.parametrize("B,S,H,Hk,D", [(1, 1, 1, 1, 32), (2, 37, 3, 3, 64), (2, 5, 8, 2, 64), (1, 130, 40, 8, 128), (3, 1, 4, 4, 256), (1, 3, 33, 1, 128),
                                        (2, 401, 16, 1, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes(B, S, H, Hk, D, interleaved, kernel_status):
    _run(B, S, H, Hk, D, D // 2, interleaved, pos=3)


@pytest.mark.parametrize("D,n", [(32, 8), (64, 8), (64, 24), (128, 0), (128, 16), (128, 56), (256, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_a_part_of_the_head(D, n, interleaved, norms):
    _run(2, 19, 6, 2, D, n, interleaved, norms=norms)


@pytest.mark.parametrize("layout", ["wide", "sequence first"])
@pytest.mark.parametrize("grads", ["heads first", "one"])
def test_layouts(layout, grads):
    _run(2, 11, 4, 2, 128, 64, False, layout=layout, grads=grads)


@pytest.mark.parametrize("scale,eps", [(0.0, 1e-6), (1e-3, 1e-5), (1e4, 1e-6), (1e-12, 1e-6)])
def test_small_large_and_no_numbers(scale, eps):
    _run(1, 9, 4, 2, 64, 32, False, scale=scale, eps=eps)


def test_many_tokens():
    _run(3, 1111, 12, 4, 64, 32, False)


def test_what_the_kernels_do_not_take_has_the_same_meaning():
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    cos, sin = ops.rope_tables(9, 40, device="cuda")
    for dtype, D in ((torch.float32, 64), (BF16, 48), (BF16, 40), (torch.float16, 64)):
        x, w = torch.randn(2, 9, 6, D, device="cuda", dtype=dtype), torch.ones(D, device="cuda", dtype=dtype)
        n = _lib.launch_count()
        q = ops.norm_rope_qkv(x, 2, 2, w, w, cos, sin)[0]
        assert _lib.launch_count() == n
        want, off = oracle.heads(x[:, :, :2], w, cos[:, None], sin[:, None], 1e-6, False)
        oracle.close(q, want, off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + 1e-6 * want.abs())


def test_captured_forward_and_backward_and_another_stream():
    from ghost_flow_b200 import ops

    cos, sin = ops.rope_tables(8, 64, device="cuda")
    x = torch.randn(2, 8, 8, 64, device="cuda", dtype=BF16).requires_grad_()
    w = [torch.ones(64, device="cuda", dtype=BF16).requires_grad_() for _ in range(2)]
    dy = [torch.randn(2, 8, n, 64, device="cuda", dtype=BF16) for n in (4, 2, 2)]
    # (v is a view of x, which is written below: it is not looked at again)
    run = lambda: (lambda y: (*y[:2], *torch.autograd.grad(y, (x, *w), dy)))(ops.norm_rope_qkv(x, 4, 2, *w, cos, sin))  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = run()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(side, run()):
        assert torch.equal(a, b)
    del side
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    g.replay()
    got = [t.clone() for t in out]
    for a, b in zip(got, run()):
        assert torch.equal(a, b)


def test_no_second_derivatives():
    from ghost_flow_b200 import ops

    cos, sin = ops.rope_tables(4, 64, device="cuda")
    x = torch.randn(1, 4, 3, 64, device="cuda", dtype=BF16).requires_grad_()
    w = torch.ones(64, device="cuda", dtype=BF16)
    q = ops.norm_rope_qkv(x, 1, 1, w, w, cos, sin)[0]
    d, = torch.autograd.grad(q.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice|twice"):
        d.float().sum().backward()


@pytest.mark.parametrize("kw", [dict(qk_norm=True), dict(qk_norm=True, rotary_dim=32), dict(rotary_dim=16, rope_interleaved=True)], ids=str)
def test_a_model_decodes_what_it_computes_at_once(kw, kernel_status):
    from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM

    torch.manual_seed(0)
    cfg = LLaMAConfig(vocab_size=97, hidden_size=256, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=64, initializer_range=0.2, **kw)
    m = LLaMAForCausalLM(cfg, device="cuda", dtype=BF16).eval()
    ids = torch.randint(0, 97, (2, 12), device="cuda")
    with torch.no_grad():
        at_once = m(ids).float()
        caches = m.new_caches(2, 12)
        steps = [m(ids[:, :7], caches=caches)] + [m(ids[:, i:i + 1], caches=caches, start_pos=i) for i in range(7, 12)]
        cache = m.new_paged_cache(4, 16)
        for b in range(2):
            cache.reserve(b, 12)
        paged = [m.forward_pages(ids[:, :7].reshape(-1), cache, cache.batch([0, 1], [7, 7], [7, 7])).view(2, 7, -1)]
        paged += [m.forward_pages(ids[:, i], cache, cache.batch([0, 1], [i + 1] * 2)).view(2, 1, -1) for i in range(7, 12)]
    # two layers of bf16 roundings (2^-8 of a number, some thirty one behind the other) on logits of the order of their norm
    for got in (torch.cat(steps, 1), torch.cat(paged, 1)):
        assert (got.float() - at_once).norm() <= 30 * 2 ** -8 / 2 * at_once.norm()
