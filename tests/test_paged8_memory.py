"""Pages of 8 bits whose scales share memory with something that a call writes."""
import pytest
import torch

from ghost_flow_b200 import ops

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
P, PAGE, HK, H, D, T = 2, 16, 2, 4, 64, 3
POOL, SCALES, OUT = P * PAGE * HK * D, P * HK * PAGE, T * H * D * 2


def _of(arena, at, shape, dtype):
    n = torch.empty(shape, dtype=dtype).nbytes
    return arena[at:at + n].view(dtype).view(shape)


def _tensors(arena, k, v, ks, vs):
    return [_of(arena, at, (P, PAGE, HK, D), E4M3) for at in (k, v)], dict(kscales=_of(arena, ks, (P, HK, PAGE), E8M0), vscales=_of(arena, vs, (P, HK, PAGE), E8M0))


def _batch(device):
    return [torch.tensor(x, dtype=torch.int32, device=device) for x in ([[1, 0]], [T + 4], [0, T])]


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["kscales", "vscales", None])
def test_results_over_the_scales_are_refused(device, which):
    arena = torch.zeros(2 * POOL + 2 * SCALES + OUT, dtype=torch.uint8, device=device)
    at = dict(kscales=2 * POOL, vscales=2 * POOL + SCALES, out=2 * POOL + 2 * SCALES)
    if which:
        at["out"], at[which] = 2 * POOL, 2 * POOL + OUT - SCALES         # the scales are the end of the results
        at["vscales" if which == "kscales" else "kscales"] = 2 * POOL + OUT
    pools, scales = _tensors(arena, 0, POOL, at["kscales"], at["vscales"])
    out = _of(arena, at["out"], (T, H, D), torch.bfloat16)
    q = torch.randn(T, H, D, device=device).bfloat16()
    if which:
        with pytest.raises(ValueError, match="shares memory"):
            ops.paged_attention(q, *pools, *_batch(device), out=out, **scales)
    else:
        assert ops.paged_attention(q, *pools, *_batch(device), out=out, **scales) is out


def _append(device, pools, scales):
    qkv = torch.randn(T, H + 2 * HK, D, device=device).bfloat16()
    cos, sin = ops.rope_tables(64, D, 1e4, device)
    return ops.rope_qkv_to_pages(qkv, H, HK, cos, sin, *pools, *_batch(device), **scales)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [0, 1])
@pytest.mark.parametrize("pool", [0, 1])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_scales_within_the_pages_are_refused(device, scale, pool, where):
    arena = torch.zeros(2 * POOL + 3 * SCALES, dtype=torch.uint8, device=device)
    at = [2 * POOL + SCALES, 2 * POOL + 2 * SCALES]
    at[scale] = pool * POOL + dict(first=0, middle=POOL // 2, last=POOL - 16)[where]
    pools, scales = _tensors(arena, 0, POOL, *at)
    with pytest.raises(ValueError, match="share"):
        _append(device, pools, scales)
    assert not arena.any()


@pytest.mark.parametrize("device", DEVICES)
def test_scales_behind_the_pages_are_written(device):
    arena = torch.zeros(2 * POOL + 2 * SCALES, dtype=torch.uint8, device=device)
    pools, scales = _tensors(arena, 0, POOL, 2 * POOL, 2 * POOL + SCALES)
    _append(device, pools, scales)
    assert all(t.view(torch.uint8).any() for t in (*pools, *scales.values()))
