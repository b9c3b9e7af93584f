"""Pools of 8 bits whose offsets pass 32 bits."""
import pytest
import torch

import _paged8_oracle as oracle
import _paged_oracle as paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,new", [([70, 33], [1, 1]), ([300, 41], [170, 41]), ([90, 300, 41], [1, 170, 1])])
@pytest.mark.parametrize("layout", ["dense", "heads first"])
def test_pages_behind_two_to_the_32_bytes(lens, new, layout, kernel_status):
    """The same batch over the last pages of large pools and over small ones: the same bits, written, read and attended over."""
    from ghost_flow_b200 import ops

    H, Hk, D, page = 32, 32, 128, 16
    P = 2 ** 32 // (page * Hk * D) + 64
    small = oracle.batch(lens, new, H, Hk, D, page, device="cuda", layout=layout)
    used, large = small["kp"].shape[0], dict(small)
    for n in ("kp", "vp"):
        pool = torch.empty((P, Hk, page, D) if layout == "heads first" else (P, page, Hk, D), dtype=torch.uint8, device="cuda")
        pool = pool.transpose(1, 2) if layout == "heads first" else pool
        pool[P - used:] = small[n].view(torch.uint8)
        large[n] = pool.view(torch.float8_e4m3fn)
    for n in ("ks", "vs"):
        large[n] = torch.cat([torch.full((P - used, Hk, page), 255, dtype=torch.uint8, device="cuda"), small[n].view(torch.uint8)]).view(torch.float8_e8m0fnu)
    large["table"] = torch.where(small["table"] >= 0, small["table"] + (P - used), small["table"])
    small = {n: t.clone() if n in ("kp", "vp", "ks", "vs") else t for n, t in small.items()}
    cos, sin = ops.rope_tables(512, D, 1e4, "cuda")
    w = torch.randn(D, device="cuda").bfloat16()
    got, want = [], []
    for x, out in ((large, got), (small, want)):
        q = ops.rope_qkv_to_pages(x["qkv"], H, Hk, cos, sin, x["kp"], x["vp"], x["table"], x["lens"], x["cu"], False, x["ks"], x["vs"], w, w)
        out += [q, ops.paged_attention(q, x["kp"], x["vp"], x["table"], x["lens"], x["cu"] if max(new) > 1 else None, kscales=x["ks"], vscales=x["vs"])]
        out += ops.read_pages(sum(new), x["kp"], x["vp"], x["table"], x["lens"], x["cu"], x["ks"], x["vs"])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for n in ("kp", "vp", "ks", "vs"):
        assert torch.equal(large[n].view(torch.uint8)[P - used:], small[n].view(torch.uint8))
    small["q"] = want[0]
    paged.close(got[1], *oracle.attention(small))
