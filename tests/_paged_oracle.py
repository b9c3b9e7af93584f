"""The operators over a paged cache and on logits from their definitions, in 64 bits on the CPU, with what a result of a type may be
off by; and batches to call them with."""
import math

import torch


def half_step(t):
    return torch.finfo(t).eps / 2


def batch(lens, new, H, Hk, D, page, dtype=torch.bfloat16, device="cpu", seed=0, layout="dense", behind=0, spare=2):
    """Pools, page table and lengths of sequences with ``new[b]`` new tokens among ``lens[b]`` keys, pages in no order. Rows behind a sequence's
    last key, and pages that nobody has, hold NaN and infinities. ``behind``: tokens behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    used = [(n + page - 1) // page for n in lens]
    P, width = sum(used) + spare, max([*used, 1]) + 1
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), width), -7, dtype=torch.int32)            # behind the last page of a sequence: never looked at
    shape = {"dense": (2, P, page, Hk, D), "heads first": (2, P, Hk, page, D), "together": (P, 2, page, Hk, D)}[layout]
    pool = torch.full(shape, float("nan"))
    pool.view(-1)[::3] = float("inf")
    pool = pool.to(device=device, dtype=dtype)
    if layout == "heads first":
        pool = pool.transpose(2, 3)
    elif layout == "together":
        pool = pool.transpose(0, 1)
    kp, vp = pool[0], pool[1]
    for b, n in enumerate(lens):
        for i in range(used[b]):
            table[b, i] = order.pop()
            m = min(page, n - i * page)
            for x in (kp, vp):
                x[int(table[b, i]), :m] = torch.randn(m, Hk, D, generator=g).to(device=device, dtype=dtype)
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    T = cu[-1] + behind
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=torch.randn(T, H, D, generator=g).to(device=device, dtype=dtype),
                qkv=torch.randn(T, H + 2 * Hk, D, generator=g).to(device=device, dtype=dtype),
                kp=kp, vp=vp, table=table.to(device), lens=ints(lens), cu=ints(cu), host=(lens, new, cu))


def attention(s, scale=None):
    """(result, how far one may be off that rounds probabilities and results to its type) [T, H, D]; NaN for tokens behind the last sequence."""
    q, kp, vp, table = (s[n].detach().cpu() for n in ("q", "kp", "vp", "table"))
    lens, new, cu = s["host"]
    (T, H, D), (P, page, Hk, _) = q.shape, kp.shape
    G, scale = H // Hk, 1 / math.sqrt(D) if scale is None else scale
    step = half_step(q.dtype)
    want, off = (torch.full((T, H, D), float("nan"), dtype=torch.float64) for _ in range(2))
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0:
            continue
        rows = torch.arange(max(n, 0))
        k, v = (x[table[b, rows // page].long(), rows % page].double() for x in (kp, vp))
        seen = rows <= (n - m + torch.arange(m))[:, None]                    # [m, n]
        for h in range(H):
            x = q[cu[b]:cu[b] + m, h].double()
            kh, vh = k[:, h // G], v[:, h // G]
            a = (x @ kh.T * scale).masked_fill(~seen, -math.inf)
            top = a.amax(-1, keepdim=True).clamp(min=-1e300) if n else torch.zeros(m, 1, dtype=torch.float64)
            p = torch.exp(a - top)
            l = p.sum(-1, keepdim=True)
            p = torch.where(l > 0, p / l, 0)
            want[cu[b]:cu[b] + m, h] = p @ vh
            # a score: D products added up in 32 bits, scaled, and the largest taken off; a probability is off by that much relative to
            # itself, once in it and once in their sum, and by one rounding to the type; a result is rounded once more
            size = (x.abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0)
            score = ((D + 8) * 2 ** -23 * size.amax(-1, keepdim=True)) if n else torch.zeros(m, 1, dtype=torch.float64)
            of = p @ vh.abs()
            off[cu[b]:cu[b] + m, h] = step * (p @ vh).abs() + (step + 2 * score + 2 ** -20) * of * (1 + 2 * step)
    return want, off


def append(s, H, Hk, cos, sin, interleaved=False):
    """q, the pools afterwards, and how far q and k may be off; rows of q that nothing is written to are NaN."""
    qkv, kp, vp, table, cos, sin = (t.detach().cpu() for t in (s["qkv"], s["kp"], s["vp"], s["table"], cos, sin))
    lens, new, cu = s["host"]
    (T, _, D), page = qkv.shape, kp.shape[1]
    step = half_step(qkv.dtype)
    q, qo = (torch.full((T, H, D), float("nan"), dtype=torch.float64) for _ in range(2))
    ko, kd, vd = torch.zeros(kp.shape, dtype=torch.float64), kp.double(), vp.double()
    first, second = (slice(0, D, 2), slice(1, D, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, D))
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            t, pos = cu[b] + i, n - m + i
            if pos < 0:
                q[t], qo[t] = 0, 0
                continue
            x, c, w = qkv[t, :H + Hk].double(), cos[pos].double(), sin[pos].double()
            y, size = torch.empty_like(x), torch.empty_like(x)
            y[:, first] = x[:, first] * c - x[:, second] * w
            y[:, second] = x[:, second] * c + x[:, first] * w
            size[:, first] = size[:, second] = x[:, first].abs() + x[:, second].abs()
            off = step * y.abs() + 2 ** -22 * size             # two products and their sum in 32 bits, one rounding
            q[t], qo[t] = y[:H], off[:H]
            page_at, r = int(table[b, pos // page]), pos % page
            kd[page_at, r], ko[page_at, r], vd[page_at, r] = y[H:], off[H:], qkv[t, H + Hk:].double()
    return q, qo, kd, ko, vd


def close(got, want, off, where=""):
    """Every element of ``got`` within ``off`` of ``want``; NaN in ``want``: not compared unless ``off`` is a number there."""
    got = got.detach().double().cpu()
    same = torch.isnan(want) & torch.isnan(got)
    ok = (got == want) | ((got - want).abs() <= off) | same
    assert ok.all(), f"{where} {int((~ok).sum())} of {ok.numel()} off, first at {torch.nonzero(~ok)[0].tolist()}: " \
                     f"{got[~ok][0]} for {want[~ok][0]} +- {off[~ok][0] if torch.is_tensor(off) else off}"


def logits(x, tokens=None, lens=None, first=None, r=1.0, p=0.0, f=0.0, bias=None, allowed=None):
    """(result, how far it may be off) of ``process_logits``; ``allowed``: truth values."""
    x = x.detach().cpu()
    B, V = x.shape
    want, off = x.double().clone(), torch.zeros(B, V, dtype=torch.float64)
    of = lambda t, b: float(t[b]) if torch.is_tensor(t) else float(t)  # noqa: E731
    for b in range(B):
        size = want[b].abs()
        if tokens is not None:
            n = tokens.shape[1] if lens is None else int(lens[b])
            row = tokens[b, :n].tolist()
            from_ = 0 if first is None else int(first[b])
            for v in set(row):
                if not 0 <= v < V:
                    continue
                c = sum(1 for i, t in enumerate(row) if t == v and i >= from_)
                a = want[b, v]
                a = a / of(r, b) if a > 0 else a * of(r, b)
                change = c * of(f, b) + (of(p, b) if c else 0.0)
                want[b, v] = a - change
                size[v] = a.abs() + c * abs(of(f, b)) + abs(of(p, b)) + abs(change)
        if bias is not None:
            add = (bias if bias.dim() == 1 else bias[b]).detach().cpu().double()
            want[b] += add
            size = size + add.abs()
        # at most five operations in 32 bits, each off by half a step of something no larger than `size`, and one rounding
        off[b] = 5 * 2 ** -24 * size * (1 + 2 ** -10) + half_step(x.dtype) * want[b].abs() * (1 + 2 ** -10) + torch.finfo(x.dtype).tiny
        if allowed is not None:
            want[b][~(allowed if allowed.dim() == 1 else allowed[b]).cpu()] = -math.inf
    return want, off
