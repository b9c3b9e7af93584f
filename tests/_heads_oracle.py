"""Heads that are normed and rotated, and their gradients, from the definitions in 64 bits on the CPU, with what a kernel may be off by that computes in 32 bits
and rounds its results to bf16 once."""
import torch

BF16_STEP = torch.finfo(torch.bfloat16).eps / 2
STEP = 2.0 ** -24               # half of fp32's last bit, relative


def turned(x, c, s, interleaved, back=False):
    """The first 2 n dims of ``x [.., D]`` rotated by tables ``[.., n]``, and the sizes of what is added up."""
    n, s = c.shape[-1], -s if back else s
    y, size = x.clone(), x.abs()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def heads(x, w, c, s, eps, interleaved):
    """(y, how far an unrounded one may be off in 32 bits); ``w``: None without a norm."""
    x, D = x.detach().double().cpu(), x.shape[-1]
    c, s = c.detach().double().cpu(), s.detach().double().cpu()
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps) ** -0.5 * w.detach().double().cpu()
    y, size = turned(x, c, s, interleaved)
    # a sum of D squares, of which the root is taken: D / 2 steps; the reciprocal root 4; its three products 3; the rotation 3; a few more
    return y, (D / 2 + 16) * STEP * size


def gradients(x, w, c, s, eps, interleaved, dy):
    """dx and dw of sum(y dy), and how far they may be off, dx rounded to bf16 and dw too. ``x [.., heads, D]``."""
    x, dy, c, s = (t.detach().double().cpu() for t in (x, dy, c, s))
    D = x.shape[-1]
    g, size = turned(dy, c, s, interleaved, back=True)
    if w is None:
        return g, BF16_STEP * g.abs() + 4 * STEP * size, None, None
    w = w.detach().double().cpu()
    r = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    h = x * r
    mean = (g * w * h).mean(-1, keepdim=True)
    dx = r * (g * w - h * mean)
    # r: D / 2 + 4 steps, in h too; the mean: a sum of D products whose factors have been off by that much already
    part = r * ((size * w).abs() + h.abs() * (size * w * h).abs().mean(-1, keepdim=True))
    dx_off = BF16_STEP * dx.abs() * 1.01 + (3 * D + 64) * STEP * part
    terms = (size * h).abs().flatten(0, -2)
    dw, n = (g * h).flatten(0, -2).sum(0), terms.shape[0]
    return dx, dx_off, dw, BF16_STEP * dw.abs() * 1.01 + (n + D / 2 + 32) * STEP * terms.sum(0)


def close(got, want, off, where=""):
    got = got.detach().double().cpu()
    ok = (got - want).abs() <= off
    assert ok.all(), f"{where} {int((~ok).sum())} of {ok.numel()} off, first at {torch.nonzero(~ok)[0].tolist()}: {got[~ok][0]} for {want[~ok][0]} +- {off[~ok][0]}"
