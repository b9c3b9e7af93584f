"""Pages of 8 bits at their edges: query heads that are not finite, rows of the least powers of two, scores of any size in prompts
(of either type of pages)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _pools(pages, page, Hk, D, eight=True):
    if not eight:
        return [torch.zeros(pages, page, Hk, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    return [torch.zeros(pages, page, Hk, D, device="cuda", dtype=torch.uint8).view(E4M3) for _ in range(2)] + [
        torch.zeros(pages, Hk, page, device="cuda", dtype=torch.uint8).view(E8M0) for _ in range(2)]


def _scales(pools):
    return dict(zip(("kscales", "vscales"), pools[2:]))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("H,Hk", [(4, 4), (8, 2), (3, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_queries_that_are_not_finite_stay_what_they_are(H, Hk, D, kernel_status):
    """Dims that are not rotated pass through: an infinity stays one, beside heads that are turned into 8 bits too."""
    from ghost_flow_b200 import ops

    T = 5
    qkv = torch.randn(T, H + 2 * Hk, D, device="cuda").bfloat16()
    qkv[0, 0, D - 1], qkv[1, H - 1, D - 2], qkv[2, 0, D - 3], qkv[3, H - 1, D - 4] = INF, -INF, NAN, INF
    qkv[3, H, D - 1] = INF                                      # a key's becomes NaN
    cos, sin = ops.rope_tables(16, D // 2, 1e4, "cuda")
    got = {}
    for eight in (False, True):
        pools = _pools(2, 16, Hk, D, eight)
        got[eight] = ops.rope_qkv_to_pages(qkv, H, Hk, cos, sin, *pools[:2], _ints([[1]]), _ints([T]), _ints([0, T]), **_scales(pools))
    assert torch.equal(got[True].nan_to_num(7.0, 8.0, 9.0), got[False].nan_to_num(7.0, 8.0, 9.0))
    assert torch.equal(got[True][:, :, D // 2:].nan_to_num(7.0, 8.0, 9.0), qkv[:, :H, D // 2:].nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("byte", [1, 2, 3, 4, 9, 127, 246])
def test_every_number_of_a_row_read_back(byte, kernel_status):
    """bf16 has all bits of a number of the pages, but for those below 2^-133, of rows of the two least units: these are rounded to the nearest, by the kernel as by PyTorch."""
    from ghost_flow_b200 import ops

    pools = _pools(2, 16, 2, 128)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, 128)
    for pool, scale in zip(pools[:2], pools[2:]):
        pool.view(torch.uint8)[1, 3] = codes
        scale.view(torch.uint8)[1, :, 3] = byte
    got = ops.read_pages(1, *pools[:2], _ints([[1]]), _ints([4]), **_scales(pools))
    exact = codes.cpu().view(E4M3).double() * 2.0 ** (byte - 127)
    for x in got:
        x = x[0].cpu()
        assert torch.equal(x.isnan(), exact.isnan()) and x.isnan().sum() == 2
        assert torch.equal(x.nan_to_num(0.0), exact.bfloat16().nan_to_num(0.0))
        if byte > 2:
            assert torch.equal(x.double().nan_to_num(0.0), exact.nan_to_num(0.0))
    cpu = ops.read_pages(1, *(t.cpu() for t in pools[:2]), _ints([[1]]).cpu(), _ints([4]).cpu(), **{n: t.cpu() for n, t in _scales(pools).items()})
    for a, b in zip(got, cpu):
        assert torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) or torch.equal(a.cpu().nan_to_num(0.0), b.nan_to_num(0.0))


# Keys are multiples of a row of ones by different numbers of at most 8 bits, so scores are exact in 32 bits and, at these sizes, thousands apart: a token's result is the value
# of the largest key that it sees, of bf16 and of e4m3 numbers alike.
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [10, 14, 18, 22, 26, 60, 100])
@pytest.mark.parametrize("lens,new,H,Hk", [([300], [300], 4, 2), ([3000], [40], 8, 2), ([700, 5, 260], [130, 5, 2], 4, 4)])
def test_scores_of_any_size_in_prompts(eight, D, power, lens, new, H, Hk, kernel_status):
    from ghost_flow_b200 import ops

    page, B = 64, len(lens)
    width = -(-max(lens) // page)
    table = torch.randperm(B * width, device="cuda").int().view(B, width)
    pools = _pools(B * width, page, Hk, D, eight)
    rank = torch.rand(B * width, page, Hk, device="cuda")
    k = (rank * 15).floor() + 1                                 # of 4 bits; of equal ones any may stand in front
    v = torch.randint(-8, 9, (B * width, page, Hk, D), device="cuda").float() / 8
    sign = torch.where(torch.rand(D, device="cuda") < 0.5, -1.0, 1.0)
    kk = k[..., None] * sign
    for x, pool, scale in zip((kk, v), pools, pools[2:] if eight else (None, None)):
        pool.view(torch.uint8 if eight else torch.bfloat16).copy_(x.to(E4M3).view(torch.uint8) if eight else x.bfloat16())
        if eight:
            scale.view(torch.uint8).fill_(127)
    T = sum(new)
    q = (sign * 2.0 ** power).expand(T, H, D).bfloat16().contiguous()
    cu = _ints([0, *torch.tensor(new).cumsum(0).tolist()])
    got = ops.paged_attention(q, *pools[:2], table, _ints(lens), cu, **_scales(pools))
    at = 0
    for b in range(B):
        n, length = new[b], lens[b]
        rows = [x[table[b].long()].flatten(0, 1)[:length].double() for x in (kk, v)]
        s = torch.einsum("thgd,nhd->hgtn", q[at:at + n].double().unflatten(1, (Hk, H // Hk)), rows[0]) * D ** -0.5
        hidden = torch.arange(length, device="cuda") > (length - n + torch.arange(n, device="cuda"))[:, None]
        p = torch.softmax(s.masked_fill(hidden, -INF), -1)
        want = torch.einsum("hgtn,nhd->thgd", p, rows[1]).flatten(1, 2)
        # a weight is rounded to bf16, and the result, of values up to 1
        assert (got[at:at + n].double() - want).abs().max().item() <= 2 * 2.0 ** -8
        at += n
