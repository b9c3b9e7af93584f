"""Kernels over pages of 8 bits, and of heads that are normed or rotated in part, against the definitions in 64 bits."""
import pytest
import torch

import _heads_oracle as heads
import _paged8_oracle as oracle
import _paged_oracle as paged
from test_gpu_paged import BATCHES, HEADS

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _pools(s):
    return s["kp"], s["vp"], s["table"], s["lens"], s["cu"]


def _count():
    from ghost_flow_b200.ops import _lib

    return _lib.launch_count()


# ------------------------------------------------------------------------------------------ append, read
def _append(s, H, Hk, cos, sin, interleaved, w, eps=1e-6, scales=True):
    from ghost_flow_b200 import ops

    n = _count()
    with torch.no_grad():
        q = ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, *_pools(s), interleaved, s["ks"] if scales else None, s["vs"] if scales else None,
                                  w[0], w[1], eps)
    assert _count() == n + 1
    return q


def _weights(D, norms):
    return [(1 + 0.3 * torch.randn(D, device="cuda")).to(BF16) if norms else None for _ in range(2)]


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("H,Hk,D,n,layout", [(1, 1, 32, 16, "dense"), (4, 2, 64, 32, "together"), (25, 25, 64, 8, "dense"), (32, 8, 128, 64, "heads first"),
                                             (40, 40, 128, 24, "dense"), (2, 1, 256, 0, "dense"), (5, 1, 128, 64, "dense")])
@pytest.mark.parametrize("interleaved,norms", [(False, False), (True, True)])
def test_append_and_read(name, H, Hk, D, n, layout, interleaved, norms, kernel_status):
    from ghost_flow_b200 import ops

    lens, new = BATCHES[name]
    s = oracle.batch(lens, new, H, Hk, D, 16 if D == 64 else 32, device="cuda", layout=layout, behind=2)
    cos, sin = ops.rope_tables(1024, 2 * n, 1e4, "cuda") if n else (torch.zeros(1024, 0, device="cuda"),) * 2
    w = _weights(D, norms)
    before = [t.clone() for t in (s["kp"].view(torch.uint8), s["vp"].view(torch.uint8), s["ks"].view(torch.uint8), s["vs"].view(torch.uint8))]
    q, qo, k, ko, v = oracle.append(s, H, Hk, cos, sin, *w, 1e-5, interleaved)
    got = _append(s, H, Hk, cos, sin, interleaved, w, 1e-5)
    T = sum(new)
    paged.close(got[:T], q[:T], qo[:T], "q")
    oracle.kept(s["kp"], s["ks"], k, ko, "keys")
    oracle.kept(s["vp"], s["vs"], v, 0.0, "values")
    rest = k.isnan().all(-1).cuda()                           # what is not written is as it was
    for x, was in zip((s["kp"], s["vp"]), before):
        assert torch.equal(x.view(torch.uint8)[rest], was[rest])
    for x, was in zip((s["ks"], s["vs"]), before[2:]):
        assert torch.equal(x.view(torch.uint8).transpose(1, 2)[rest], was.transpose(1, 2)[rest])
    c = _count()
    back = ops.read_pages(T + 2, *_pools(s), s["ks"], s["vs"])
    assert _count() == c + 1
    for y, x, e in zip(back, (s["kp"], s["vp"]), (s["ks"], s["vs"])):
        want, y = oracle.values(x, e), y.cpu().double()
        assert not y[T:].any()
        for b, (length, m) in enumerate(zip(lens, new)):
            pos = torch.arange(length - m, length)
            rows = y[int(s["cu"][b]):int(s["cu"][b]) + m]
            at = s["table"].cpu()[b, pos.clamp(min=0) // x.shape[1]].long().clamp(min=0), pos.clamp(min=0) % x.shape[1]
            assert torch.equal(rows, want[at].masked_fill((pos < 0)[:, None, None], 0))


@pytest.mark.parametrize("name", ["one", "mixed", "fewer keys than tokens", "server"])
@pytest.mark.parametrize("H,Hk,D,n,norms", [(4, 2, 64, 32, True), (32, 8, 128, 16, False), (3, 1, 256, 128, True), (9, 3, 32, 8, True)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_to_pages_of_bf16(name, H, Hk, D, n, norms, interleaved, kernel_status):
    from ghost_flow_b200 import ops

    lens, new = BATCHES[name]
    s = paged.batch(lens, new, H, Hk, D, 32, device="cuda", behind=2)
    cos, sin = ops.rope_tables(1024, 2 * n, 1e4, "cuda")
    w = _weights(D, norms)
    old = s["kp"].clone(), s["vp"].clone()
    q, qo, k, ko, v = oracle.append(s, H, Hk, cos, sin, *w, 1e-6, interleaved)
    got = _append(s, H, Hk, cos, sin, interleaved, w, scales=False)
    T = sum(new)
    paged.close(got[:T], q[:T], qo[:T], "q")
    here = ~k.isnan().any(-1)
    paged.close(s["kp"][here.cuda()], k[here], (ko + heads.BF16_STEP * (k.abs() + ko))[here], "keys")
    assert torch.equal(s["vp"][here.cuda()].cpu().double(), v[here])
    for x, was in zip((s["kp"], s["vp"]), old):
        assert torch.equal(x[~here.cuda()].view(torch.int16), was[~here.cuda()].view(torch.int16))
    y = ops.read_pages(T, *_pools(s))
    assert all(torch.isfinite(t).all() for t in y)


def test_powers_of_two_and_what_is_not_finite(kernel_status):
    rows = [448.0, 447.0, 450.0, 449.0, 224.0, 225.0, 1.75, 1.7578125, 0.0, 2.0 ** -126, 2.0 ** -133, 3e38, 2.0 ** -110, 1.0]
    for D in (32, 64, 128, 256):
        y = torch.zeros(len(rows), 4, D)
        y[:, :, 0] = torch.tensor(rows)[:, None]
        y[:, 1] *= -1
        y[:, 2, 1:] = y[:, 2, :1] * torch.randn(len(rows), D - 1).clamp(-1, 1)
        y[3, 0, 3], y[4, 0, D - 1], y[5, 0, D // 2] = float("nan"), float("inf"), -float("inf")
        y[13, 3] = float("inf")
        s = oracle.batch([len(rows)], [len(rows)], 1, 4, D, 16, device="cuda")
        s["qkv"] = torch.cat((torch.zeros(len(rows), 1, D), y, y), 1).to(BF16).cuda()
        none = torch.zeros(64, 0, device="cuda")
        _append(s, 1, 4, none, none, False, (None, None))
        want, e = oracle.quantised(s["qkv"][:, 1:5].cpu())
        at = int(s["table"][0, 0])
        for x, b in ((s["kp"], s["ks"]), (s["vp"], s["vs"])):
            assert torch.equal(x[at, :len(rows)].cpu().double().nan_to_num(-1), want.nan_to_num(-1))
            assert torch.equal(b.view(torch.uint8)[at, :, :len(rows)].t().cpu().long(), e + 127)


def test_pages_and_positions_that_are_not_there():
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    for change in (lambda s: s["table"].__setitem__((1, 1), 10 ** 6), lambda s: s["table"].__setitem__((1, 1), -5), lambda s: s["lens"].__setitem__(1, 4000)):
        s = oracle.batch([7, 40], [1, 30], 4, 2, 64, 16, device="cuda")
        change(s)
        cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
        for call in (lambda: _append(s, 4, 2, cos, sin, False, _weights(64, True)), lambda: ops.read_pages(31, *_pools(s), s["ks"], s["vs"]),
                     lambda: _attend(s), lambda: _attend(s, q=s["q"][:2], cu=None)):
            call()
            with pytest.raises(_lib.KernelStatusError):
                _lib.check_status()
    s = oracle.batch([7, 40], [1, 30], 4, 2, 64, 16, device="cuda")
    cos, sin = ops.rope_tables(20, 64, 1e4, "cuda")
    q = _append(s, 4, 2, cos, sin, False, (None, None))
    assert not q[12:].any() and q[1:11].any()
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()


# ------------------------------------------------------------------------------------------ attention
def _attend(s, **kw):
    from ghost_flow_b200 import ops

    a = {**dict(q=s["q"], cu=s["cu"]), **kw}
    return ops.paged_attention(a.pop("q"), s["kp"], s["vp"], s["table"], s["lens"], a.pop("cu"), kscales=s["ks"], vscales=s["vs"], **a)


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("H,Hk,D", HEADS)
def test_attention(name, H, Hk, D, kernel_status):
    lens, new = BATCHES[name]
    s = oracle.batch(lens, new, H, Hk, D, 16 if D == 64 else 32, device="cuda", behind=3)
    want, off = oracle.attention(s)
    out = torch.full_like(s["q"], 7.0)
    c = _count()
    _attend(s, out=out)
    assert _count() > c
    n = sum(new)
    paged.close(out[:n], want[:n], off[:n], name)
    assert (out[n:] == 7).all()                          # behind the last sequence
    assert torch.equal(_attend(s)[:n], out[:n])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["dense", "heads first", "together"])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 2, 128)])
def test_attention_pages_and_layouts(page, layout, H, Hk, D, kernel_status):
    lens, new = [page - 1, page, page + 1, 3 * page + 5, 300], [1, 2, page + 1, 40, 1]
    s = oracle.batch(lens, new, H, Hk, D, page, device="cuda", layout=layout)
    want, off = oracle.attention(s)
    paged.close(_attend(s), want, off)


@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 1, 128), (16, 1, 64), (20, 2, 128), (11, 1, 64), (40, 1, 128)])
@pytest.mark.parametrize("scale", [None, 0.02, -0.3])
def test_attention_of_one_token_each(H, Hk, D, scale, kernel_status):
    lens = [1, 16, 17, 0, 64, 1000, 515]
    s = oracle.batch(lens, [1] * len(lens), H, Hk, D, 16, device="cuda")
    want, off = oracle.attention(s, scale)
    paged.close(_attend(s, cu=None, scale=scale), want, off)


@pytest.mark.parametrize("parts", [1, 3, 16, -1, -5, -300])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 1, 128), (24, 2, 64), (16, 1, 128)])
def test_attention_of_some_with_one_token(parts, H, Hk, D, monkeypatch, kernel_status):
    from ghost_flow_b200.ops import paged as module

    monkeypatch.setattr(module, "_parts_beside", lambda *a: parts)
    lens = [900, 40, 64, 0, 1, 200, 333, 70, 5, 1200]
    for new in ([1, 40, 1, 1, 1, 2, 1, 33, 0, 1], [2, 40, 3, 2, 0, 2, 7, 33, 5, 0], [1] * 10, [0, 0, 0, 0, 0, 0, 0, 0, 1, 0]):
        s = oracle.batch(lens, new, H, Hk, D, 16, device="cuda", behind=1)
        want, off = oracle.attention(s)
        out = torch.full_like(s["q"], 7.0)
        for _ in range(2):
            _attend(s, out=out)
        n = sum(new)
        paged.close(out[:n], want[:n], off[:n])
        assert (out[n:] == 7).all()


@pytest.mark.parametrize("lens,new", [([9000], [1]), ([5000, 3], [1, 1]), ([4000, 700], [40, 300]), ([20000], [3])])
@pytest.mark.parametrize("H,Hk,D", [(4, 1, 128), (4, 4, 64)])
def test_attention_over_long_sequences(lens, new, H, Hk, D, kernel_status):
    s = oracle.batch(lens, new, H, Hk, D, 64, device="cuda")
    want, off = oracle.attention(s)
    paged.close(_attend(s), want, off)


@pytest.mark.parametrize("new", [[1, 1], [130, 1], [70, 3]])
@pytest.mark.parametrize("spread", [6.0, 20.0])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_very_different_sizes(new, spread, D, kernel_status):
    """Powers of two far apart, of values that count much beside those that count little, and scores of the order of hundreds."""
    s = oracle.batch([700, 300], new, 4, 2, D, 32, device="cuda", spread=spread)
    k = s["ks"].view(torch.uint8)
    k.copy_(torch.where(k < 255, k.int().clamp(100, 124), 255).to(torch.uint8))          # scores that do not all go to one key
    want, off = oracle.attention(s)
    paged.close(_attend(s), want, off)


def test_what_is_not_a_number_stays_so(kernel_status):
    from ghost_flow_b200 import ops

    for new in ([1, 1, 1], [5, 40, 1]):
        s = oracle.batch([40, 90, 70], new, 4, 2, 64, 16, device="cuda")
        want = _attend(s)
        s["vp"].view(torch.uint8)[int(s["table"][0, 0]), 3, 1, 5] = 0x7f
        s["kp"].view(torch.uint8)[int(s["table"][2, 1]), 2, 0, 9] = 0xff
        got = _attend(s)
        a, b = new[0], new[0] + new[1]
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[:a, 2:, 5] = True
        bad[b:, :2] = True
        assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])
        assert ops.read_pages(1, s["kp"], s["vp"], s["table"][:1], torch.full_like(s["lens"][:1], 4), None, s["ks"], s["vs"])[1][0, 1].isnan().sum() == 1


def test_attention_of_views_and_without_kernels_for_it(kernel_status):
    s = oracle.batch([40, 300], [7, 33], 6, 2, 64, 16, device="cuda")
    want, off = oracle.attention(s)
    packed = torch.randn(40, 10, 64, device="cuda").bfloat16()
    packed[:, :6] = s["q"]
    wide = torch.full((40, 8, 64), 7.0, device="cuda", dtype=BF16)
    paged.close(_attend(s, q=packed[:, :6], out=wide[:, 1:7]), want, off)
    assert (wide[:, 0] == 7).all() and (wide[:, 7] == 7).all()
    paged.close(_attend(s, q=s["q"].transpose(1, 2).contiguous().transpose(1, 2)), want, off)
    for D, page in ((32, 16), (64, 24)):
        s = oracle.batch([40, 300, 0], [7, 33, 1], 6, 2, D, page, device="cuda")
        want, off = oracle.attention(s)
        paged.close(_attend(s), want, off + 2 ** -20)


def test_a_step_captured_and_replayed_on_other_streams(kernel_status):
    """Append, attention and read as a server's step runs them, replayed after lengths, pages and numbers have changed; two graphs at once."""
    from ghost_flow_b200 import ops

    H, Hk, D = 8, 2, 128
    cos, sin = ops.rope_tables(512, D, 1e4, "cuda")
    w = _weights(D, True)

    def step(s, cu):
        q = ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], cu, False, s["ks"], s["vs"], *w)
        return q, _attend(s, q=q, cu=cu), *ops.read_pages(q.shape[0], s["kp"], s["vp"], s["table"], s["lens"], cu, s["ks"], s["vs"])

    with torch.no_grad():
        made = []
        for new in ([1, 1, 1], [40, 3, 1]):
            s = oracle.batch([300, 77, 130], new, H, Hk, D, 16, device="cuda")
            cu = None if max(new) == 1 else s["cu"]
            step(s, cu)
            torch.cuda.synchronize()
            g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(g, stream=stream):
                out = step(s, cu)
            made.append((s, cu, g, out, torch.cuda.Stream()))
        for s, cu, *_ in made:
            s["qkv"].copy_(torch.randn_like(s["qkv"]))
            s["lens"].copy_(torch.tensor([250, 60, 131], dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        for _, _, g, _, st in made:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, cu, _, out, _ in made:
            got = [t.clone() for t in out]
            for a, b in zip(got, step(s, cu)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("kw", [{}, dict(qk_norm=True), dict(qk_norm=True, rotary_dim=32)], ids=str)
def test_a_model_over_pages_of_8_bits(kw, kernel_status):
    """Chunks of any size compute what whole prompts do, near the model over its own type."""
    from ghost_flow_b200.models import LLaMAConfig, LLaMAForCausalLM

    torch.manual_seed(0)
    cfg = LLaMAConfig(vocab_size=97, hidden_size=256, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=64, initializer_range=0.2, **kw)
    m = LLaMAForCausalLM(cfg, device="cuda", dtype=BF16).eval()
    ids = torch.randint(0, 97, (30,), device="cuda")
    out = []
    for dtype, cuts in ((torch.float8_e4m3fn, (30,)), (torch.float8_e4m3fn, (11, 12, 13, 30)), (None, (30,))):
        cache = m.new_paged_cache(2, 16, dtype=dtype)
        cache.reserve(0, 30)
        at, parts = 0, []
        for end in cuts:
            parts.append(m.forward_pages(ids[at:end], cache, cache.batch([0], [end], [end - at])))
            at = end
        out.append(torch.cat(parts).float())
        k, v = cache.read(0, 30, 1)
        assert k.shape == (30, 2, 64) and k.isfinite().all() and v.isfinite().all()
    # other tiles, other sums: roundings to bf16 as elsewhere, and what they flip in the cache (2^-4 of a number, of few)
    assert (out[0] - out[1]).norm() <= 0.1 * out[0].norm()
    assert 0 < (out[0] - out[2]).norm() < 0.2 * out[2].norm()
    tokens = m.generate_batch([ids[:9], ids[:20]], 5, page_size=16, cache_dtype=torch.float8_e4m3fn, temperature=0.9, top_k=20, top_p=0.9)
    assert [t.numel() for t in tokens] == [14, 25] and all(((t >= 0) & (t < 97)).all() for t in tokens)


@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (8, 8, 64), (16, 1, 64)])
@pytest.mark.parametrize("spread", [10, 14, 18])
def test_scores_far_beyond_the_powers_of_two(H, Hk, D, spread, kernel_status):
    """One token each over rows of such sizes that a score's last bit is worth more than all powers of two: results stay finite."""
    lens = [1, 2, 9, 33, 700, 1213]
    s = oracle.batch(lens, [1] * len(lens), H, Hk, D, 16, device="cuda", spread=spread)
    paged.close(_attend(s, cu=None), *oracle.attention(s))
