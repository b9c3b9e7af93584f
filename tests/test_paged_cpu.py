"""Paged cache and logits on CPU tensors: PyTorch's operations against the definitions, what is refused, and what goes on to them."""
import pytest
import torch

import _paged_oracle as oracle
from ghost_flow_b200 import ops

SEQUENCES = [([5], [5]), ([1], [1]), ([33, 16, 40], [1, 16, 7]), ([0, 17, 3], [1, 2, 0]), ([2, 9], [5, 1])]


@pytest.mark.parametrize("lens,new", SEQUENCES)
@pytest.mark.parametrize("H,Hk,D,page,layout,dtype", [(4, 2, 16, 16, "dense", torch.float32), (3, 1, 24, 5, "heads first", torch.bfloat16),
                                                       (6, 3, 64, 32, "together", torch.float64)])
def test_attention(lens, new, H, Hk, D, page, layout, dtype):
    s = oracle.batch(lens, new, H, Hk, D, page, dtype, layout=layout, behind=2)
    want, off = oracle.attention(s)
    got = ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"])
    n = sum(new)
    oracle.close(got[:n], want[:n], off[:n])
    out = torch.full_like(s["q"], 7.0)
    assert ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], out=out) is out
    assert torch.equal(out[:n], got[:n]) and (out[n:] == 7).all()


@pytest.mark.parametrize("lens,new", SEQUENCES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hk,D,page,layout,dtype", [(4, 2, 16, 16, "dense", torch.float32), (3, 1, 24, 5, "heads first", torch.bfloat16),
                                                       (6, 3, 64, 32, "together", torch.float64)])
def test_append(lens, new, interleaved, H, Hk, D, page, layout, dtype):
    s = oracle.batch(lens, new, H, Hk, D, page, dtype, layout=layout, behind=2)
    cos, sin = ops.rope_tables(64, D, 1e4)
    q, qo, k, ko, v = oracle.append(s, H, Hk, cos, sin, interleaved)
    got = ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"], interleaved)
    n = sum(new)
    oracle.close(got[:n], q[:n], qo[:n])
    oracle.close(s["kp"], k, ko)
    oracle.close(s["vp"], v, 0.0)


def test_one_token_of_each_sequence_needs_no_cu():
    lens = [7, 0, 33]
    s = oracle.batch(lens, [1, 1, 1], 4, 2, 16, 16, torch.float32)
    a = ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"])
    assert torch.equal(a, ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"])) and not a[1].any()
    cos, sin = ops.rope_tables(64, 16, 1e4)
    pools = [(s["kp"].clone(), s["vp"].clone()) for _ in range(2)]
    q = [ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, *p, s["table"], s["lens"], cu) for p, cu in zip(pools, (None, s["cu"]))]
    assert torch.equal(*q) and all(torch.equal(x.nan_to_num(3), y.nan_to_num(3)) for x, y in zip(*pools)) and not q[0][1].any()


def test_batches_of_nothing():
    s = oracle.batch([], [], 4, 2, 16, 16, torch.float32, behind=3)
    cos, sin = ops.rope_tables(8, 16, 1e4)
    assert ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"]).shape == (3, 4, 16)
    assert ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]).shape == (3, 4, 16)
    s = oracle.batch([7], [0], 4, 2, 16, 16, torch.float32)
    out = torch.zeros(0, 4, 16)
    assert ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], out=out) is out
    assert ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]).shape == (0, 4, 16)
    x = torch.zeros(0, 7)
    assert ops.process_logits(x).shape == (0, 7) and ops.process_logits(x, out=x) is x


def test_gradient_of_attention_is_that_of_its_formula():
    s = oracle.batch([4, 9], [2, 5], 4, 2, 8, 16, torch.float64)
    for n in ("kp", "vp"):
        s[n] = s[n].nan_to_num(0, 0, 0).requires_grad_()
    q = s["q"].requires_grad_()
    assert torch.autograd.gradcheck(lambda a, k, v: ops.paged_attention(a, k, v, s["table"], s["lens"], s["cu"]), (q, s["kp"], s["vp"]))


def test_gradient_of_append_goes_through_the_rotation():
    s = oracle.batch([4, 9], [2, 5], 4, 2, 8, 16, torch.float64)
    cos, sin = ops.rope_tables(16, 8, 1e4)
    z = torch.zeros_like(s["kp"])

    def f(x):
        k, v = z.clone(), z.clone()
        return ops.rope_qkv_to_pages(x, 4, 2, cos, sin, k, v, s["table"], s["lens"], s["cu"]), k, v

    assert torch.autograd.gradcheck(f, (s["qkv"].requires_grad_(),))


def _call(s, **kw):
    s = {**s, **kw}
    return ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], out=s.get("out"))


REFUSED = [dict(q=torch.zeros(3, 4)), dict(q=torch.zeros(3, 5, 16)), dict(q=torch.zeros(3, 4, 8)), dict(q=torch.zeros(3, 4, 16).half()),
           dict(kp=torch.zeros(2, 16, 2, 8)), dict(vp=torch.zeros(3, 16, 2, 16)), dict(kp=torch.zeros(3, 16, 2)),
           dict(table=torch.zeros(2, 2, dtype=torch.int64)), dict(table=torch.zeros(3, 2, dtype=torch.int32)),
           dict(lens=torch.zeros(2, dtype=torch.int64)), dict(lens=torch.zeros(2, 1, dtype=torch.int32)),
           dict(cu=torch.zeros(2, dtype=torch.int32)), dict(cu=torch.zeros(3)), dict(cu=None),
           dict(out=torch.zeros(2, 4, 16)), dict(out=torch.zeros(3, 4, 16).double())]


@pytest.mark.parametrize("kw", REFUSED, ids=lambda k: "-".join(k))
def test_batches_that_are_refused(kw):
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    with pytest.raises(ValueError, match="paged_attention"):
        _call(s, **kw)


def test_out_that_shares_memory_is_refused():
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    for out in (s["q"], s["kp"].view(-1)[:3 * 64].view(3, 4, 16), s["vp"].view(-1)[64:4 * 64].view(3, 4, 16)):
        with pytest.raises(ValueError, match="shares memory"):
            _call(s, out=out)


@pytest.mark.parametrize("kw", [dict(H=3), dict(Hk=1), dict(cos=torch.zeros(64, 16)), dict(sin=torch.zeros(32, 8)), dict(H=0, Hk=4)])
def test_projections_and_tables_that_are_refused(kw):
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    cos, sin = ops.rope_tables(64, 16, 1e4)
    a = {**dict(H=4, Hk=2, cos=cos, sin=sin), **kw}
    with pytest.raises(ValueError, match="rope_qkv_to_pages"):
        ops.rope_qkv_to_pages(s["qkv"], a["H"], a["Hk"], a["cos"], a["sin"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"])


def test_projections_in_the_pages_are_refused():
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    cos, sin = ops.rope_tables(64, 16, 1e4)
    for pool in (s["kp"], s["vp"]):
        with pytest.raises(ValueError, match="shares memory"):
            ops.rope_qkv_to_pages(pool.reshape(-1)[:3 * 8 * 16].view(3, 8, 16), 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"])


@pytest.mark.parametrize("change", [lambda s: s["table"].__setitem__((1, 1), 99), lambda s: s["table"].__setitem__((1, 1), -1),
                                    lambda s: s["lens"].__setitem__(1, 60)], ids=["page behind", "page below", "length behind the table"])
def test_pages_and_positions_that_are_not_there(change):
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    change(s)
    cos, sin = ops.rope_tables(64, 16, 1e4)
    with pytest.raises(ValueError, match="not there"):
        _call(s)
    with pytest.raises(ValueError, match="not there"):
        ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"])


def test_positions_behind_the_rope_tables():
    s = oracle.batch([7, 20], [1, 2], 4, 2, 16, 16, torch.float32)
    with pytest.raises(ValueError, match="not there"):
        ops.rope_qkv_to_pages(s["qkv"], 4, 2, *ops.rope_tables(19, 16, 1e4), s["kp"], s["vp"], s["table"], s["lens"], s["cu"])


# ------------------------------------------------------------------------------------------ logits
def _penalties(B, V, L, seed=0, device="cpu", dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    tokens = (V * torch.rand(B, L, generator=g).pow(3)).to(dtype)
    if L > 3:
        tokens[:, 1], tokens[:, 2] = -1, V + 5                    # padding, and what no vocabulary has
    lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
    first = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
    r, p, f = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g)
    return [t.to(device) for t in (tokens, lens, first, r, p, f)]


@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (3, 33, 7), (2, 100, 0), (4, 257, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_process_logits(B, V, L, dtype):
    x = 4 * torch.randn(B, V).to(dtype)
    x[0, V // 2] = float("-inf")
    tokens, lens, first, r, p, f = _penalties(B, V, L)
    bias, ok = torch.randn(B, V), torch.rand(B, V) < 0.6
    ok[0] = False
    for kw, o in [({}, {}), (dict(tokens=tokens, repetition=1.3), dict(tokens=tokens, r=1.3)),
                  (dict(tokens=tokens, token_lens=lens, generated_from=first, repetition=r, presence=p, frequency=f),
                   dict(tokens=tokens, lens=lens, first=first, r=r, p=p, f=f)),
                  (dict(bias=bias[0].contiguous()), dict(bias=bias[0])), (dict(bias=bias), dict(bias=bias)),
                  (dict(allowed=ops.pack_allowed(ok)), dict(allowed=ok)), (dict(allowed=ops.pack_allowed(ok[-1])), dict(allowed=ok[-1])),
                  (dict(tokens=tokens, frequency=f, bias=bias, allowed=ops.pack_allowed(ok)), dict(tokens=tokens, f=f, bias=bias, allowed=ok))]:
        want, off = oracle.logits(x, **o)
        got = ops.process_logits(x, **kw)
        oracle.close(got, want, off, str(list(kw)))
        y = x.clone()
        assert ops.process_logits(y, **kw, out=y) is y and torch.equal(y, got)


def test_packed_masks():
    for V in (1, 31, 32, 33, 100):
        m = torch.rand(3, V) < 0.5
        w = ops.pack_allowed(m)
        assert w.dtype is torch.int32 and w.shape == (3, (V + 31) // 32)
        for b in range(3):
            for v in range(V):
                assert bool((int(w[b, v // 32]) >> (v % 32)) & 1) == bool(m[b, v])


def test_gradient_of_processed_logits():
    x = torch.randn(3, 20, dtype=torch.float64, requires_grad=True)
    tokens, lens, first, r, p, f = _penalties(3, 20, 12)
    kw = dict(tokens=tokens, token_lens=lens, generated_from=first, repetition=r, presence=p, frequency=f, bias=torch.randn(20))
    assert torch.autograd.gradcheck(lambda a: ops.process_logits(a, **kw), (x,))


I32 = torch.int32


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(8)), dict(logits=torch.zeros(2, 8, dtype=I32)), dict(tokens=torch.zeros(3, 4, dtype=I32)),
    dict(tokens=torch.zeros(2, 4)), dict(token_lens=torch.zeros(2, dtype=I32)), dict(generated_from=torch.zeros(2, dtype=I32)),
    dict(tokens=torch.zeros(2, 4, dtype=I32), token_lens=torch.zeros(2, dtype=torch.int64)),
    dict(tokens=torch.zeros(2, 4, dtype=I32), generated_from=torch.zeros(3, dtype=I32)), dict(repetition=0.0), dict(repetition=-1.0),
    dict(repetition=torch.ones(3)), dict(presence=torch.ones(2, dtype=torch.float64)), dict(frequency=torch.ones(2, 1)),
    dict(bias=torch.zeros(7)), dict(bias=torch.zeros(2, 8).half()), dict(allowed=torch.zeros(2, 8, dtype=torch.bool)),
    dict(allowed=torch.zeros(2, 2, dtype=I32)), dict(out=torch.zeros(2, 9)), dict(out=torch.zeros(2, 8).half())],
    ids=lambda k: "-".join(k))
def test_logits_that_are_refused(kw):
    kw = {"logits": torch.zeros(2, 8), **kw}
    with pytest.raises(ValueError, match="process_logits"):
        ops.process_logits(**kw)


def test_out_that_overlaps_the_logits_is_refused():
    t = torch.zeros(40)
    with pytest.raises(ValueError, match="shares memory"):
        ops.process_logits(t[:16].view(2, 8), out=t[8:24].view(2, 8))


def test_out_that_overlaps_what_else_is_read_is_refused():
    t = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="shares memory with bias"):
        ops.process_logits(torch.zeros(2, 8), bias=t, out=t)


def test_parts_beside_another_kernel():
    from ghost_flow_b200.ops.paged import _parts_beside

    assert [_parts_beside(n, 148) for n in (8, 32, 64, 128, 256, 259, 4000)] == [16, 7, 4, 2, 1, 1, 1]
