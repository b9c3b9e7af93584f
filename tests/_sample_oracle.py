"""The choice of a token from its definition, a row at a time, with Python's numbers."""
import math


def token(x, u, temperature, top_k, top_p, min_p):
    """``x``: a row's numbers. Weights are added up exactly (fsum), so a choice is another one only where a border and the random number agree to 15 digits."""
    bad = [v for v, a in enumerate(x) if math.isnan(a)]
    top = max((a for a in x if not math.isnan(a)), default=math.nan)
    if bad:
        return bad[0]
    if top == -math.inf:
        return -1
    if top == math.inf or not temperature > 0 or top_k == 1 or top_p <= 0:
        return x.index(top)
    order = sorted(range(len(x)), key=lambda v: (-x[v], v))
    w = {v: math.exp((x[v] - top) / temperature) if x[v] > -math.inf else 0.0 for v in order}
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        total, front, kept = math.fsum(w[v] for v in order), 0.0, []
        for v in order:
            if not front < top_p * total:
                break
            kept.append(v)
            front += w[v]
        order = kept
    order = sorted(v for v in order if w[v] >= min(min_p, 1.0))
    total, upto = math.fsum(w[v] for v in order), 0.0
    for v in order:
        upto += w[v]
        if upto > u * total:
            return v
    return [v for v in order if w[v] > 0][-1]


def tokens(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = x.detach().double().cpu().tolist()
    of = lambda t, b: t[b].item() if hasattr(t, "shape") else t  # noqa: E731
    return [token(r, u[b].item(), of(temperature, b), of(top_k, b), of(top_p, b), of(min_p, b)) for b, r in enumerate(rows)]
