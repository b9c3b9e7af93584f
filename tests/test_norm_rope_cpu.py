"""norm_rope_qkv on the CPU: definition, gradients against differences, refusals, and models whose heads are normed or rotated in part."""
import pytest
import torch

import _heads_oracle as oracle
from ghost_flow_b200 import ops
from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM
from ghost_flow_b200.ops import _lib


def _case(B, S, H, Hk, D, n, dtype=torch.float32, pos=2, norms=True):
    cos, sin = ops.rope_tables(S + pos, 2 * n) if n else (torch.zeros(S + pos, 0),) * 2
    w = [(1 + 0.3 * torch.randn(D)).to(dtype) if norms else None for _ in range(2)]
    return torch.randn(B, S, H + 2 * Hk, D).to(dtype), *w, cos, sin


@pytest.mark.parametrize("B,S,H,Hk,D,n", [(2, 5, 4, 2, 64, 32), (1, 1, 3, 1, 24, 6), (3, 2, 2, 2, 10, 0), (1, 7, 5, 1, 128, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_against_the_definition(B, S, H, Hk, D, n, interleaved, norms):
    x, qw, kw, cos, sin = _case(B, S, H, Hk, D, n, norms=norms)
    q, k, v = ops.norm_rope_qkv(x, H, Hk, qw, kw, cos, sin, 1e-5, interleaved, 2)
    for y, part, w in ((q, x[:, :, :H], qw), (k, x[:, :, H:H + Hk], kw)):
        want, off = oracle.heads(part, w, cos[2:, None], sin[2:, None], 1e-5, interleaved)
        oracle.close(y, want, off + 2 * oracle.STEP * want.abs())
    assert torch.equal(v, x[:, :, H + Hk:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_gradients_against_differences(interleaved, norms):
    x, qw, kw, cos, sin = _case(2, 3, 2, 1, 8, 3, torch.float64, norms=norms)
    leaves = [t.requires_grad_() for t in (x, qw, kw) if t is not None]
    f = lambda x, *w: ops.norm_rope_qkv(x, 2, 1, *(w or (None, None)), cos.double(), sin.double(), 1e-3, interleaved, 1)  # noqa: E731
    assert torch.autograd.gradcheck(f, leaves)


def test_the_oracles_gradients_are_those_of_the_definition():
    x, qw, _, cos, sin = _case(2, 3, 4, 1, 16, 4, torch.float64)
    x, w, c, s = x[:, :, :4].clone().requires_grad_(), qw.requires_grad_(), cos[:3, None].double(), sin[:3, None].double()
    y = x * (x.square().mean(-1, keepdim=True) + 1e-5) ** -0.5 * w
    z, _ = oracle.turned(y, c, s, True)
    dy = torch.randn_like(z)
    dx, dw = torch.autograd.grad(z, (x, w), dy)
    got = oracle.gradients(x, w, c, s, 1e-5, True, dy)
    assert torch.allclose(got[0], dx) and torch.allclose(got[2], dw)


@pytest.mark.parametrize("kw", [dict(qkv=torch.randn(2, 3, 7, 16)), dict(qkv=torch.randn(3, 8, 16)), dict(num_heads=0), dict(q_weight=torch.ones(8)),
                                dict(k_weight=None), dict(k_weight=torch.ones(16, device="meta")), dict(cos=torch.ones(9, 9), sin=torch.ones(9, 9)),
                                dict(cos=torch.ones(9, 4)), dict(pos_offset=7), dict(pos_offset=-1), dict(sin=torch.ones(9, 8, device="meta"))], ids=lambda k: "-".join(k))
def test_refusals(kw):
    base = dict(qkv=torch.randn(2, 3, 8, 16), num_heads=4, num_kv_heads=2, q_weight=torch.ones(16), k_weight=torch.ones(16), cos=torch.ones(9, 8),
                sin=torch.ones(9, 8))
    ops.norm_rope_qkv(**base)
    with pytest.raises(ValueError, match="norm_rope_qkv"):
        ops.norm_rope_qkv(**{**base, **kw})


def test_the_entry_points_refuse_before_they_launch():
    import ctypes

    lib, P = _lib.cuda_lib(), 1 << 20
    names = "x ldx qw kw cos sin q k T S H Hk D rotary pos0 il".split()
    good = dict(x=P, ldx=512, qw=P, kw=P, cos=P, sin=P, q=P, k=P, T=6, S=3, H=4, Hk=2, D=64, rotary=64, pos0=0, il=0)
    shared = [*({n: P + 8} for n in "x qw kw cos sin".split()), *({n: None} for n in "x qw kw cos sin".split()), dict(ldx=508), dict(ldx=320), dict(T=0),
              dict(S=0), dict(S=4), dict(H=0), dict(Hk=0), dict(H=70000), dict(D=48), dict(D=512), dict(rotary=72), dict(rotary=80), dict(rotary=8),
              dict(pos0=-1)]
    for kw in (*shared, dict(q=None), dict(k=P + 4)):
        v = {**good, **kw}
        assert lib.gf_norm_rope_qkv(*(v[n] for n in names), 1e-6, None) == -1, kw
    names = "x ldx qw kw cos sin dq dk dv lds dx dqw dkw scratch T S H Hk D rotary pos0 il".split()
    lds = lambda *n: (ctypes.c_longlong * 3)(*n)  # noqa: E731
    good = {**good, **dict(dq=P, dk=P, dv=P, lds=lds(256, 128, 128), dx=P, dqw=P, dkw=P, scratch=P)}
    for kw in (*shared, dict(dq=P + 2), dict(dv=None), dict(dx=None), dict(dqw=None), dict(scratch=None), dict(lds=lds(252, 128, 128)),
               dict(lds=lds(256, 64, 128)), dict(lds=None)):
        v = {**good, **kw}
        assert lib.gf_norm_rope_qkv_bwd(*(v[n] for n in names), 1e-6, None) == -1, kw


def _model(**kw):
    torch.manual_seed(0)
    cfg = LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=32, initializer_range=0.3, **kw)
    m = LLaMAForCausalLM(cfg, dtype=torch.float32).eval()
    if cfg.qk_norm:
        with torch.no_grad():
            for layer in m.model.layers:
                for n in (layer.attn.q_norm, layer.attn.k_norm):
                    n.weight.copy_(1 + 0.3 * torch.randn(16))
    return m


@pytest.mark.parametrize("kw", [dict(qk_norm=True), dict(rotary_dim=8), dict(qk_norm=True, rotary_dim=4, rope_interleaved=True)], ids=str)
def test_models(kw):
    """Token by token over a cache, over pages, and all at once: the same tokens; and gradients reach the norms."""
    m = _model(**kw)
    ids = torch.randint(0, 97, (2, 6))
    out = m.generate(ids, 5)
    again = ids
    for _ in range(5):
        again = torch.cat([again, m(again)[:, -1].argmax(-1, keepdim=True)], 1)
    assert torch.equal(out, again)
    assert torch.equal(torch.stack(m.generate_batch(list(ids), 5, page_size=16)), out)
    plain = _model()
    plain.load_state_dict(m.state_dict(), strict=False)
    assert not torch.allclose(plain(ids), m(ids))
    m(ids, labels=ids)[0].backward()
    assert all(p.grad is not None and p.grad.abs().sum() > 0 for p in m.parameters())
    assert m.cfg.num_parameters() == sum(p.numel() for p in m.parameters())


def test_engines_without_such_heads_say_so():
    from ghost_flow_b200.parallel.tp_inference import TPLlamaInference
    from ghost_flow_b200.parallel.zero3 import Zero3LlamaEngine

    for kw in (dict(qk_norm=True), dict(rotary_dim=8)):
        cfg = _model(**kw).cfg
        with pytest.raises(NotImplementedError, match="heads"):
            Zero3LlamaEngine(cfg, "cpu", dtype=torch.float32)
        with pytest.raises(NotImplementedError, match="heads"):
            TPLlamaInference(cfg, 1, 4, 4, "cpu")


def test_a_served_checkpoint_with_norms_has_them():
    from ghost_flow_b200.serve import _llama_config_from_state

    sd = _model(qk_norm=True).state_dict()
    assert _llama_config_from_state(sd, dict(num_attention_heads=4)).qk_norm
    assert not _llama_config_from_state(_model().state_dict(), dict(num_attention_heads=4)).qk_norm


def test_no_dims_rotated_and_a_part_of_them_with_experts():
    from ghost_flow_b200.models import MixtralConfig
    from ghost_flow_b200.models.encoders import MixtralForCausalLM

    m, ids = _model(rotary_dim=0), torch.randint(0, 97, (2, 6))
    assert not m.cfg.plain_heads and torch.equal(torch.stack(m.generate_batch(list(ids), 5, page_size=16)), m.generate(ids, 5))
    m(ids)
    assert m.model.layers[0].attn.cfg.rope_dims == 0
    seen = []
    m = MixtralForCausalLM(MixtralConfig(vocab_size=97, hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                                         num_local_experts=2, max_position_embeddings=16, rotary_dim=8, qk_norm=True), dtype=torch.float32)
    m.layers[0].attn.register_forward_hook(lambda mod, args, out: seen.append(args[1].shape))
    m(ids)
    assert seen == [(16, 4)]
