"""Pages of 8 bits from their definition, in 64 bits on the CPU."""
import torch

import _heads_oracle as heads
import _paged_oracle as paged

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def quantised(y):
    """Rows ``[.., D]`` as (numbers of type e4m3 in 64 bits, exponents of their powers of two); what is not finite is NaN."""
    y = y.double()
    finite = y.isfinite()
    most = torch.where(finite, y, 0).abs().amax(-1)
    e = torch.full(most.shape, -126, dtype=torch.int64)
    while True:                                            # the smallest power that leaves nothing above 448
        more = most > 448 * torch.exp2(e.double())
        if not more.any():
            break
        e = e + more
    x = torch.where(finite, y / torch.exp2(e.double()).unsqueeze(-1), 0)
    last = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(finite, torch.round(x / last) * last, float("nan")), e


def values(pages, scales):
    """A pool as numbers of 64 bits."""
    return pages.detach().cpu().double() * torch.exp2(scales.detach().cpu().view(torch.uint8).double() - 127).transpose(1, 2).unsqueeze(-1)


def batch(lens, new, H, Hk, D, page, device="cpu", seed=0, layout="dense", behind=0, spread=1.0, spare=2):
    """As ``_paged_oracle.batch``; rows of numbers of different sizes (2^(``spread`` times a normal number)), any bytes behind a sequence's last key."""
    s = paged.batch(lens, new, H, Hk, D, page, torch.bfloat16, device, seed, "dense", behind, spare)
    g = torch.Generator().manual_seed(seed + 1)
    P = s["kp"].shape[0]
    bytes_ = lambda *shape: torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)  # noqa: E731
    shape = {"dense": (2, P, page, Hk, D), "heads first": (2, P, Hk, page, D), "together": (P, 2, page, Hk, D)}[layout]
    pool = bytes_(*shape).to(device)
    pool = pool.transpose(2, 3) if layout == "heads first" else pool.transpose(0, 1) if layout == "together" else pool
    for i, n in enumerate("kv"):
        scales = bytes_(P, Hk, page)
        codes = bytes_(P, page, Hk, D)
        for b, length in enumerate(lens):
            rows = torch.arange(length)
            at = s["table"].cpu()[b, rows // page].long(), rows % page
            x = s[n + "p"].cpu()[at].double() * torch.exp2(spread * torch.randn(length, Hk, 1, generator=g))
            q, e = quantised(x)
            codes[at] = q.float().to(E4M3).view(torch.uint8)
            scales.transpose(1, 2)[at] = (e + 127).to(torch.uint8)
        pool[i].copy_(codes.to(device))
        s[n + "p"], s[n + "s"] = pool[i].view(E4M3), scales.to(device).view(E8M0)
    return s


def attention(s, scale=None):
    """As ``_paged_oracle.attention``, of the numbers that the pages stand for."""
    kp, vp = values(s["kp"], s["ks"]), values(s["vp"], s["vs"])
    want, off = paged.attention({**s, "kp": kp, "vp": vp}, scale)
    # a query is turned into f16 in a unit of its own: what is below 2^-14 of its largest number is off by 2^-25 of that
    k = kp.abs().nan_to_num(0, 0, 0).sum(-1)
    lens, new, cu = s["host"]
    scale = s["q"].shape[-1] ** -0.5 if scale is None else abs(scale)
    vmax = vp.abs()
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0 or n <= 0:
            continue
        rows = torch.arange(n)
        at = s["table"].cpu()[b, rows // kp.shape[1]].long(), rows % kp.shape[1]
        most = k[at].amax(0)                               # [Hk]
        q = s["q"][cu[b]:cu[b] + m].detach().cpu().double().abs().amax(-1)         # [m, H]
        G = q.shape[1] // most.shape[0]
        off[cu[b]:cu[b] + m] += (2 * 2.0 ** -25 * scale * q * most.repeat_interleave(G) * vmax[at].amax((0, 2)).repeat_interleave(G)).unsqueeze(-1)
    return want, off


def append(s, H, Hk, cos, sin, qw, kw, eps, interleaved, bytes_=True):
    """q and how far it may be off; keys and values before they are rounded, by page and row, and how far those may be off (values 0)."""
    qkv, table = s["qkv"].detach().cpu().double(), s["table"].cpu()
    lens, new, cu = s["host"]
    (T, _, D), (P, page, _, _) = qkv.shape, s["kp"].shape
    q, qo = (torch.full((T, H, D), float("nan"), dtype=torch.float64) for _ in range(2))
    k, ko, v = (torch.full((P, page, Hk, D), float("nan"), dtype=torch.float64) for _ in range(3))
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            t, pos = cu[b] + i, n - m + i
            if pos < 0:
                q[t], qo[t] = 0, 0
                continue
            y, off = heads.heads(qkv[t, :H], qw, cos[pos], sin[pos], eps, interleaved)
            q[t], qo[t] = y, off + heads.BF16_STEP * (y.abs() + off)
            at = int(table[b, pos // page]), pos % page
            k[at], ko[at] = heads.heads(qkv[t, H:H + Hk], kw, cos[pos], sin[pos], eps, interleaved)
            v[at] = qkv[t, H + Hk:]
    return q, qo, k, ko, v


def kept(pages, scales, want, off, where=""):
    """Rows of a pool that ``want`` has numbers for are those, each in the smallest power of two that holds them, to half a step of the type."""
    here = ~want.isnan().any(-1)
    got, byte = values(pages, scales)[here], scales.detach().cpu().view(torch.uint8).transpose(1, 2)[here].double()
    y, off = want[here], off[here] if torch.is_tensor(off) else torch.zeros(int(here.sum()), want.shape[-1], dtype=torch.float64)
    unit, most, slack = torch.exp2(byte - 127), y.abs().amax(-1), off.amax(-1)
    assert (most - slack <= 448 * unit).all() and ((byte == 1) | (most + slack > 448 * unit / 2)).all(), where + " powers of two"
    half = torch.maximum(y.abs() * 2.0 ** -4, unit.unsqueeze(-1) * 2.0 ** -10)
    paged.close(got, y, (half + off) * (1 + 2.0 ** -20), where)
