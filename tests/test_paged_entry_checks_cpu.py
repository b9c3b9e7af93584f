"""Arguments that the kernel library refuses before it launches anything. The pointers are numbers that nothing reads."""
import struct

import pytest

from ghost_flow_b200.ops import _lib

BAD_ARG, P = -1, 1 << 20
NAMES = "x ldx y ldy kp vp k0 k1 k2 v0 v1 v2 table ld_table width lens cu B T H Hk D page pages status".split()
VALUES = dict(x=P, ldx=512, y=P, ldy=256, kp=P, vp=P, k0=2048, k1=128, k2=64, v0=2048, v1=128, v2=64, table=P, ld_table=4, width=4, lens=P,
              cu=P, B=2, T=5, H=4, Hk=2, D=64, page=16, pages=9, status=0)


def _call(**kw):
    return struct.pack("25q", *(({**VALUES, **kw})[n] for n in NAMES))


SHARED = [*({n: P + 8} for n in "x y kp vp".split()), *({n: 0} for n in "x y kp vp lens table".split()), dict(ldx=508), dict(ldx=-8),
          dict(ldy=260), dict(k0=2047), dict(v1=4), dict(k2=-64), dict(B=0), dict(T=0), dict(T=-1), dict(T=1 << 31), dict(cu=0), dict(page=24),
          dict(page=8), dict(page=0), dict(pages=-1), dict(pages=1 << 27), dict(width=-1), dict(width=1 << 27), dict(ld_table=-1), dict(H=0),
          dict(Hk=0)]


@pytest.mark.parametrize("kw", [*SHARED, dict(ldy=512), dict(D=72), dict(D=0), dict(D=8192), dict(H=1 << 20)], ids=str)
def test_append(kw):
    assert _lib.cuda_lib().gf_paged_append(_call(**kw), P, P, 100, 0, None) == BAD_ARG


# x: 5 rows 512 apart, the last of 8 x 64; the pools: 9 pages of 16 rows of 128
@pytest.mark.parametrize("kw", [dict(), dict(kp=P + 2 * 2560 - 16, vp=1 << 30), dict(vp=P - 2 * 18432 + 16, kp=1 << 30)], ids=str)
def test_append_of_tokens_that_lie_in_the_pools(kw):
    assert _lib.cuda_lib().gf_paged_append(_call(**kw), P, P, 100, 0, None) == -5


@pytest.mark.parametrize("cos,sin,n", [(None, P, 9), (P, None, 9), (P + 4, P, 9), (P, P + 8, 9), (P, P, -1)])
def test_append_tables(cos, sin, n):
    assert _lib.cuda_lib().gf_paged_append(_call(), cos, sin, n, 0, None) == BAD_ARG
    assert _lib.cuda_lib().gf_paged_append(None, P, P, 9, 0, None) == BAD_ARG


@pytest.mark.parametrize("kw", [*SHARED, dict(D=96), dict(D=256), dict(H=5), dict(H=516, Hk=4), dict(pages=0), dict(Hk=1 << 20, H=1 << 20)], ids=str)
def test_attention(kw):
    lib = _lib.cuda_lib()
    assert lib.gf_paged_attn(_call(**kw), 0.1, P, 1 << 40, 0, None, None) == BAD_ARG
    if kw != dict(cu=0):
        assert lib.gf_paged_attn_one(_call(**{"cu": 0, "T": 2, **kw}), 0.1, 1, P, None) == BAD_ARG


def test_attention_scales_workspaces_and_splits():
    lib = _lib.cuda_lib()
    need = lib.gf_paged_attn_workspace(2, 5, 0, 0, 64 * 16, 4, 2, 64)
    assert need > 0 and lib.gf_paged_attn_workspace(2, 5, 0, 0, 1024, 5, 2, 64) == lib.gf_paged_attn_workspace(2, 5, 0, 0, 1024, 4, 2, 96) == -1
    for scale in (0.0, -0.1, float("nan")):
        assert lib.gf_paged_attn(_call(), scale, P, need, 0, None, None) == BAD_ARG
    for ws, n in ((P, need - 1), (None, need), (P + 8, need)):
        assert lib.gf_paged_attn(_call(width=64), 0.1, ws, n, 0, None, None) == BAD_ARG
    assert lib.gf_paged_attn(_call(width=64), 0.1, P, need, 2, None, None) == BAD_ARG             # no scratch for the splits
    assert lib.gf_paged_attn(_call(H=26, Hk=2), 0.1, P, 1 << 40, 2, P, None) == BAD_ARG   # thirteen query heads to a KV head
    one = dict(cu=0, T=2)
    assert lib.gf_paged_attn_one(_call(**one), 0.1, 0, P, None) == lib.gf_paged_attn_one(_call(**one), 0.1, 2, None, None) == BAD_ARG
    assert lib.gf_paged_attn_one(_call(T=2), 0.1, 1, P, None) == lib.gf_paged_attn_one(None, 0.1, 1, P, None) == BAD_ARG
    assert lib.gf_paged_attn(None, 0.1, P, need, 0, None, None) == BAD_ARG


LOGITS = dict(x=P, ldx=100, y=P, ldy=100, dtype=0, B=2, V=100, tokens=0, ldt=0, tokens64=0, L=0, token_lens=0, generated_from=0, repetition=0,
              presence=0, frequency=0, r=1.0, p=0.0, f=0.0, bias=0, ldb=0, allowed=0, lda=0)


@pytest.mark.parametrize("kw", [dict(x=0), dict(y=0), dict(B=0), dict(V=0), dict(V=1 << 31), dict(B=1 << 31), dict(L=-1), dict(dtype=3), dict(dtype=-1)],
                         ids=str)
def test_logits(kw):
    assert _lib.cuda_lib().gf_process_logits(struct.pack("16q3d4q", *{**LOGITS, **kw}.values()), None) == BAD_ARG
    assert _lib.cuda_lib().gf_process_logits(None, None) == BAD_ARG
