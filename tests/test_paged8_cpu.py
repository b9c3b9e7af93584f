"""A cache of 8 bits on CPU tensors: rows written, read back and attended over against the definitions, what is refused, and models over it."""
import pytest
import torch

import _heads_oracle as heads
import _paged8_oracle as oracle
import _paged_oracle as paged
from ghost_flow_b200 import ops
from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM
from ghost_flow_b200.models.paged import PagedKVCache
from ghost_flow_b200.ops import _lib

E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


def _append(s, H, Hk, cos, sin, interleaved=False, **kw):
    return ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"], interleaved, s["ks"], s["vs"], **kw)


@pytest.mark.parametrize("lens,new", [([7, 20], [1, 20]), ([0, 33, 16], [1, 4, 16]), ([3], [5])])
@pytest.mark.parametrize("D,n", [(16, 8), (24, 6), (32, 0)])
@pytest.mark.parametrize("norms,interleaved", [(False, False), (True, True), (True, False)])
def test_append_and_read(lens, new, D, n, norms, interleaved):
    s = oracle.batch(lens, new, 4, 2, D, 16, behind=2)
    cos, sin = ops.rope_tables(64, 2 * n) if n else (torch.zeros(64, 0),) * 2
    w = [(1 + 0.3 * torch.randn(D)).to(BF16) if norms else None for _ in range(2)]
    q, qo, k, ko, v = oracle.append(s, 4, 2, cos, sin, *w, 1e-5, interleaved)
    got = _append(s, 4, 2, cos, sin, interleaved, q_weight=w[0], k_weight=w[1], eps=1e-5)
    T = sum(new)
    paged.close(got[:T], q[:T], qo[:T])
    oracle.kept(s["kp"], s["ks"], k, ko, "keys")
    oracle.kept(s["vp"], s["vs"], v, 0.0, "values")
    for y, x, e in zip(ops.read_pages(T + 2, s["kp"], s["vp"], s["table"], s["lens"], s["cu"], s["ks"], s["vs"]), (s["kp"], s["vp"]), (s["ks"], s["vs"])):
        want = oracle.values(x, e)
        assert y.dtype is BF16 and y.shape == (T + 2, 2, D) and not y[T:].any()
        for b, (length, m) in enumerate(zip(lens, new)):
            for i in range(m):
                pos = length - m + i
                row = want[int(s["table"][b, pos // 16]), pos % 16] if pos >= 0 else torch.zeros(2, D).double()
                assert torch.equal(y[int(s["cu"][b]) + i].double(), row)


def test_powers_of_two_and_what_is_not_finite():
    """Rows whose largest number lies at, below and above a border, in every power of two, and rows of zeros, of tiny and of no numbers."""
    rows = [448.0, 447.0, 450.0, 449.0, 224.0, 225.0, 1.75, 1.7578125, 0.0, 2.0 ** -126, 2.0 ** -133, 3e38, 2.0 ** -110, 1.0]
    y = torch.zeros(len(rows), 4, 16)
    y[:, :, 0] = torch.tensor(rows)[:, None]
    y[:, 1] *= -1
    y[:, 2, 1:] = y[:, 2, :1] * torch.randn(len(rows), 15).clamp(-1, 1)
    y[3, 0, 3], y[4, 0, 3], y[5, 0, 3] = float("nan"), float("inf"), -float("inf")
    y[13, 3] = float("inf")
    s = oracle.batch([len(rows)], [len(rows)], 1, 4, 16, 16)
    s["qkv"] = torch.cat((torch.zeros(len(rows), 1, 16), y, y), 1).to(BF16)
    _append(s, 1, 4, torch.ones(64, 8), torch.zeros(64, 8))
    at = int(s["table"][0, 0])
    turned, _ = heads.turned(s["qkv"][:, 1:5].double(), torch.ones(8).double(), torch.zeros(8).double(), False)      # infinity's partner: 0 times it
    for x, b, y in ((s["kp"], s["ks"], turned), (s["vp"], s["vs"], s["qkv"][:, 5:9])):
        want, e = oracle.quantised(y)
        assert torch.equal(x[at, :len(rows)].double().nan_to_num(-1), want.nan_to_num(-1))
        assert torch.equal(b.view(torch.uint8)[at, :, :len(rows)].t().long(), e + 127)


@pytest.mark.parametrize("lens,new", [([7, 20], [1, 3]), ([0, 33, 16], [1, 4, 16]), ([3], [5])])
def test_attention(lens, new):
    s = oracle.batch(lens, new, 4, 2, 16, 16, behind=1)
    want, off = oracle.attention(s)
    got = ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], kscales=s["ks"], vscales=s["vs"])
    T = sum(new)
    paged.close(got[:T], want[:T], off[:T])


REFUSED = [dict(ks=None), dict(vs=None), dict(ks=torch.zeros(3, 16, 2, dtype=torch.uint8).view(E8M0)), dict(vs=torch.zeros(4, 2, 16)),
           dict(vs=torch.zeros(4, 2, 16, dtype=torch.uint8)), dict(kp=torch.zeros(4, 16, 2, 16, dtype=BF16)), dict(vp=torch.zeros(4, 16, 2, 8).to(E4M3)),
           dict(ks="vs")]


@pytest.mark.parametrize("kw", REFUSED, ids=lambda k: "-".join(k))
def test_pools_that_are_refused(kw):
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, spare=1)
    assert s["kp"].shape[0] == 4
    cos, sin = ops.rope_tables(64, 16)
    s.update({n: s[t] if isinstance(t, str) else t for n, t in kw.items()})
    b = s["kp"], s["vp"], s["table"], s["lens"], s["cu"]
    with pytest.raises(ValueError, match="paged_attention"):
        ops.paged_attention(s["q"], *b, kscales=s["ks"], vscales=s["vs"])
    with pytest.raises(ValueError, match="read_pages"):
        ops.read_pages(3, *b, s["ks"], s["vs"])
    with pytest.raises(ValueError, match="rope_qkv_to_pages"):
        _append(s, 4, 2, cos, sin)


@pytest.mark.parametrize("kw", [dict(q_weight=torch.ones(16)), dict(q_weight=torch.ones(8), k_weight=torch.ones(8)),
                                dict(q_weight=torch.ones(16), k_weight=torch.ones(16, device="meta")), dict(cos=torch.zeros(64, 9), sin=torch.zeros(64, 9)),
                                dict(cos=torch.zeros(64, 4))], ids=lambda k: "-".join(k))
def test_norms_and_tables_that_are_refused(kw):
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16)
    cos, sin = ops.rope_tables(64, 16)
    kw = {"cos": cos, "sin": sin, **kw}
    with pytest.raises(ValueError, match="rope_qkv_to_pages"):
        _append(s, 4, 2, kw.pop("cos"), kw.pop("sin"), **kw)


def test_read_refuses_and_reports():
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16)
    b = s["kp"], s["vp"], s["table"], s["lens"]
    for rows, cu in ((-1, s["cu"]), (3, None), (3, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="read_pages"):
            ops.read_pages(rows, *b, cu, s["ks"], s["vs"])
    with pytest.raises(ValueError, match="read_pages"):
        ops.read_pages(3, s["kp"].float().to(BF16), s["vp"], s["table"], s["lens"], s["cu"])
    assert ops.read_pages(0, *b, torch.zeros(3, dtype=torch.int32), s["ks"], s["vs"])[0].shape == (0, 2, 16)
    s["table"][1, 1] = 99
    with pytest.raises(ValueError, match="not there"):
        ops.read_pages(3, *b, s["cu"], s["ks"], s["vs"])


def test_read_of_pages_of_other_types_copies():
    for dtype in (torch.float32, BF16):
        s = paged.batch([7, 20], [3, 20], 4, 2, 16, 16, dtype)
        k, v = ops.read_pages(23, s["kp"], s["vp"], s["table"], s["lens"], s["cu"])
        rows = torch.arange(20)
        assert k.dtype is dtype and torch.equal(k[3:], s["kp"][s["table"][1, rows // 16].long(), rows % 16])
        assert torch.equal(v[:3], s["vp"][int(s["table"][0, 0]), 4:7])


def test_the_entry_points_refuse_before_they_launch():
    import struct

    lib, P = _lib.cuda_lib(), 1 << 20
    names = "x ldx y ldy kp vp k0 k1 k2 v0 v1 v2 table ld_table width lens cu B T H Hk D page pages status ks vs".split()
    good = dict(x=P, ldx=512, y=P, ldy=256, kp=2 * P, vp=3 * P, k0=2048, k1=128, k2=64, v0=2048, v1=128, v2=64, table=P, ld_table=4, width=4, lens=P,
                cu=P, B=2, T=5, H=4, Hk=2, D=64, page=16, pages=9, status=0, ks=4 * P, vs=5 * P)
    call = lambda **kw: struct.pack("27q", *({**good, **kw}[n] for n in names))  # noqa: E731
    heads = lambda c, rot=64, qw=P, kw=P, cos=P, sin=P, n=9: lib.gf_paged_append_heads(c, cos, sin, n, rot, 0, qw, kw, 1e-6, None)  # noqa: E731
    pools = [*({n: P + 8} for n in "kp vp ks vs".split()), *({n: 0} for n in "kp vp vs".split()), dict(k0=2056), dict(v1=120), dict(k2=-64), dict(B=0),
             dict(T=0), dict(page=24), dict(pages=-1), dict(lens=0), dict(Hk=0)]
    for kw in (*pools, dict(ks=0), dict(x=P + 8), dict(ldy=512), dict(D=96), dict(D=512), dict(H=0)):
        assert heads(call(**kw)) == -1, kw
    for kw in (dict(rot=72), dict(rot=80), dict(rot=-16), dict(qw=None), dict(kw=P + 2), dict(cos=None), dict(sin=P + 4), dict(n=-1)):
        assert heads(call(), **kw) == -1, kw
    assert heads(None) == -1
    for n in "kp vp ks vs".split():                          # x among what is written
        assert heads(call(**{n: P + 2 * 2560 - 16})) == -5
    for kw in (*pools, dict(D=8), dict(D=40), dict(D=80), dict(D=8192)):
        assert lib.gf_paged_read(call(**kw), P, P, None) == -1, kw
    assert lib.gf_paged_read(None, P, P, None) == lib.gf_paged_read(call(), None, P, None) == lib.gf_paged_read(call(), P, P + 8, None) == -1
    for kw in (*pools, dict(ks=0), dict(ks=0, vs=0), dict(D=96), dict(H=5), dict(pages=0)):
        assert lib.gf_paged_attn8(call(**kw), 0.1, P, 1 << 40, 0, None, None) == -1, kw
        assert lib.gf_paged_attn8_one(call(**{"cu": 0, "T": 2, **kw}), 0.1, 1, P, None) == -1, kw
    assert lib.gf_paged_attn8(None, 0.1, P, 1, 0, None, None) == lib.gf_paged_attn8_one(None, 0.1, 1, P, None) == -1


def test_the_module_leaves_what_is_not_its():
    calls, s, t = _lib.calls(), oracle.batch([7, 20], [1, 2], 4, 2, 64, 16), torch.zeros(64, 32)
    b = s["kp"], s["vp"], s["table"], s["lens"], s["cu"]
    assert calls.attention8(s["q"], *b, s["ks"], s["vs"]) is None and calls.read(3, *b, s["ks"], s["vs"]) is None
    assert calls.append_heads(s["qkv"], 4, 2, *b, t, t, s["ks"], s["vs"], None, None) is None
    for f in (calls.append_heads, calls.run_append_heads, calls.read, calls.run_read, calls.attention8, calls.run_attention8):
        with pytest.raises(TypeError, match="arguments"):
            f(1)
    for f, n in ((calls.run_append_heads, 6), (calls.run_read, 5), (calls.run_attention8, 9)):
        with pytest.raises(TypeError, match="not a call"):
            f(b"x" * 100, t, *[0] * (n - 2))


def _model(**kw):
    torch.manual_seed(0)
    return LLaMAForCausalLM(LLaMAConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                        num_key_value_heads=2, max_position_embeddings=32, initializer_range=0.3, **kw), dtype=torch.float32).eval()


@pytest.mark.parametrize("kw", [{}, dict(qk_norm=True), dict(rotary_dim=8)], ids=str)
def test_a_model_over_pages_of_8_bits(kw):
    """In chunks of any size it computes the same; and what it computes is near the model over its own type."""
    m = _model(**kw)
    prompts = [torch.randint(0, 97, (n,)) for n in (11, 3, 17)]
    run = lambda **c: m.generate_batch(prompts, 6, page_size=16, cache_dtype=E4M3, **c)  # noqa: E731
    for a, b in zip(run(), run(chunk_tokens=4)):
        assert torch.equal(a, b)
    cache, exact = m.new_paged_cache(4, 16, dtype=E4M3), m.new_paged_cache(4, 16)
    assert cache.pools[0][0].dtype is E4M3 and cache.pools[0][2].shape == (4, 2, 16) and len(cache.pools[1]) == 4
    for c in (cache, exact):
        c.reserve("a", 17)
    out = [m.forward_pages(prompts[2], c, c.batch(["a"], [17], [17])) for c in (cache, exact)]
    # keys and values are off by 2^-5 of a number on average at most: far less than a logit's size
    assert 0 < (out[0] - out[1]).norm() < 0.2 * out[1].norm()
    (k, v), (kx, vx) = cache.read("a", 17, 0), exact.read("a", 17, 0)
    assert k.dtype is BF16 and kx.dtype is torch.float32 and k.shape == kx.shape == (17, 2, 16)
    for y, x in ((k, kx), (v, vx)):
        assert ((y.double() - x.double()).abs() <= x.double().abs() * 2.0 ** -4 * 1.001 + x.double().abs().amax(-1, keepdim=True) / 224 * 2.0 ** -10).all()


def test_caches():
    c = PagedKVCache(2, 5, 16, 2, 32, dtype=E4M3)
    assert [t.dtype for t in c.pools[0]] == [E4M3, E4M3, E8M0, E8M0] and not c.pools[0][2].view(torch.uint8).any()
    c.reserve(0, 20)
    k, v = c.read(0, 20)
    assert k.shape == (20, 2, 32) and not k.any() and not v.any()
    with pytest.raises(ValueError, match="room"):
        c.read(0, 33)


def test_rows_of_a_page_are_within_32_bits():
    """The kernels add up rows of a page in 32 bits: pools whose rows are further apart are refused."""
    import struct

    lib, P = _lib.cuda_lib(), 1 << 20
    far = 0x7fffffff // 16 // 16 * 16
    call = lambda k1, v1: struct.pack("27q", P, 512, P, 256, 2 * P, 3 * P, 2048, k1, 64, 2048, v1, 64, P, 4, 4, P, P, 2, 5, 4, 2, 64, 16, 9, 0, 4 * P, 5 * P)  # noqa: E731
    for k1, v1 in ((far + 16, 128), (128, far + 16), (1 << 31, 128)):
        c = call(k1, v1)
        assert lib.gf_paged_append_heads(c, P, P, 9, 64, 0, P, P, 1e-6, None) == lib.gf_paged_read(c, P, P, None) == -1
        assert lib.gf_paged_attn8(c, 0.1, P, 1 << 40, 0, None, None) == lib.gf_paged_attn8_one(c, 0.1, 1, P, None) == -1
