"""More operators of language models, as work to be timed: norms of query and key heads with the rotation in the same pass (and their
gradients), a paged KV cache in 8 bits that is written, read back and attended over, and the choice of tokens by temperature, top-k, top-p and min-p.

A case is a dict of plain values; ``kind`` names the operator, the rest are its sizes. ``listed()`` gives the cases that stand
for the ranges, ``draw(rng)`` another one of the same ranges. With ``own`` the calls are the framework's, else elementary
torch operations in 32 bits (64 where weights of tokens are added up and compared); ``exact`` is the definition in 64 bits.

A row of a head in the cache is numbers of type e4m3 times 2^e, e the smallest whole number that leaves none above 448 (and at least -126), kept as the byte e + 127.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
THETA = 10000.0
EPS = 1e-6


# ------------------------------------------------------------------------------------------ the cases
# norm_rope: [batch, seq] tokens; `rotary` dims of a head are rotated; `train`: with the gradients.
# append, attention: `batch` sequences with `shortest` .. `longest` keys (new tokens among them). The first `chunks` of them have up to `chunk`
# new tokens (0: the whole sequence is new), the others one.
def listed():
    return [
        # one training step's attention input, Mixtral's heads, two sequences
        dict(name="norm_rope_train", kind="norm_rope", batch=2, seq=4096, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, train=True),
        # a prompt of odd length, LLaMA-7B's heads, half of each rotated, pairs next to each other
        dict(name="norm_rope_prompt", kind="norm_rope", batch=1, seq=2987, heads=32, kv_heads=32, dim=128, rotary=64, interleaved=True,
             train=False),
        # a small model's training step
        dict(name="norm_rope_small", kind="norm_rope", batch=3, seq=57, heads=4, kv_heads=2, dim=64, rotary=64, interleaved=False, train=True),
        # one token of each of 64 sequences in a server's batch, Mixtral's heads, no norms
        dict(name="append8_decode", kind="append", batch=64, shortest=17, longest=2000, chunks=0, chunk=1, heads=32, kv_heads=8, dim=128,
             page=16, rotary=128, norms=False, interleaved=False),
        # five prompts of different lengths at once, LLaMA-7B's heads, with norms
        dict(name="append8_prompts", kind="append", batch=5, shortest=301, longest=1507, chunks=5, chunk=0, heads=32, kv_heads=32, dim=128,
             page=64, rotary=128, norms=True, interleaved=False),
        # one token of each of 32 sequences of mixed lengths, Mixtral's heads
        dict(name="attn8_decode", kind="attention", batch=32, shortest=100, longest=4096, chunks=0, chunk=1, heads=32, kv_heads=8, dim=128,
             page=16),
        # few long sequences, eight query heads to a KV head
        dict(name="attn8_long", kind="attention", batch=4, shortest=20011, longest=30001, chunks=0, chunk=1, heads=64, kv_heads=8,
             dim=128, page=64),
        # the next chunk of a long prompt
        dict(name="attn8_chunk", kind="attention", batch=1, shortest=7681, longest=7681, chunks=1, chunk=512, heads=32, kv_heads=8, dim=128,
             page=16),
        # a server's step: one sequence's chunk of the prompt among 31 that generate
        dict(name="attn8_mixed", kind="attention", batch=32, shortest=130, longest=2048, chunks=1, chunk=481, heads=32, kv_heads=8, dim=128,
             page=32),
        # a small batch, one choice for all rows
        dict(name="sample_small", kind="sample", rows=3, vocab=32000, dtype="bf16", top_k=50, top_p=0.9, min_p=0.0, each=False),
        # a server's batch over the GPT-2 vocabulary (rows padded as the output head leaves them), each row with its own choice
        dict(name="sample_server", kind="sample", rows=64, vocab=50257, dtype="bf16", top_k=0, top_p=0.95, min_p=0.02, each=True),
        # the largest: 32-bit logits of a large batch
        dict(name="sample_large", kind="sample", rows=512, vocab=50257, dtype="fp32", top_k=0, top_p=0.9, min_p=0.0, each=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12, 64), (16, 2, 64), (25, 25, 64), (4, 2, 64), (32, 32, 128), (32, 8, 128), (40, 40, 128), (64, 8, 128), (16, 1, 128),
         (10, 2, 128)]


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "attention", "attention", "sample"])
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 512), vocab=rng.choice([1000, 30522, 32000, 50257]), dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                    top_k=rng.choice([0, 0, 1, _log(rng, 2, 900)]), top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), each=rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice(HEADS)
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim)
    if kind != "attention":
        c.update(rotary=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.3)
    if kind == "norm_rope":
        batch = _log(rng, 1, 8)
        c.update(batch=batch, seq=_log(rng, 1, max(2, 3 * 10 ** 7 // (batch * (heads + 2 * kv_heads) * dim))), train=rng.random() < 0.5)
        return c
    c["page"] = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "append":
        c["norms"] = rng.random() < 0.5
    form = rng.choice(["one", "chunk", "mixed", "prompts"])
    if form == "one":
        batch = _log(rng, 1, 64)
        c.update(batch=batch, longest=min(_log(rng, 1, 4096), 10 ** 8 // (batch * kv_heads * dim)), chunks=0, chunk=1)
    elif form == "chunk":
        longest = _log(rng, 64, 7000)
        c.update(batch=1, longest=longest, chunks=1, chunk=min(longest, _log(rng, 2, 512)))
    elif form == "mixed":
        batch = _log(rng, 2, 32)
        longest = min(_log(rng, 64, 2048), 10 ** 8 // (batch * kv_heads * dim))
        c.update(batch=batch, longest=longest, chunks=rng.randint(1, 1 + batch // 8), chunk=min(longest, _log(rng, 2, 400)))
    else:
        batch = rng.randint(1, 6)
        c.update(batch=batch, longest=_log(rng, 16, 2600 // batch), chunks=batch, chunk=0)
    c["shortest"] = max(1, int(c["longest"] * rng.choice([1.0, 0.5, 0.1])))
    return c


# ------------------------------------------------------------------------------------------ sizes of a case
def _sequences(c):
    """Keys and new tokens of each sequence: a fixed choice between the shortest and the longest, which occurs."""
    rng = random.Random(1000003 * c["batch"] + c["longest"])
    lens = [c["longest"]] + [rng.randint(c["shortest"], c["longest"]) for _ in range(c["batch"] - 1)]
    new = [min(n, c["chunk"] or n) if b < c["chunks"] else 1 for b, n in enumerate(lens)]
    return lens, new


def work(case):
    if case["kind"] == "sample":
        b, v, size = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": b * v * size + 28 * b, "flops": 4 * b * v}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "norm_rope":
        T, tables = case["batch"] * case["seq"], 4 * case["seq"] * case["rotary"]
        n, f = 4 * T * (H + Hk) * D + tables + 4 * D, 7 * T * (H + Hk) * D
        if case["train"]:          # the gradients of q, k and v, q and k again, and the packed gradient
            n, f = n + 2 * T * D * (2 * (H + Hk) + 2 * Hk + (H + Hk)) + tables + 8 * D, 3 * f
        return {"bytes": n, "flops": f}
    lens, new = _sequences(case)
    T = sum(new)
    if case["kind"] == "append":
        n = T * (2 * (2 * H + 2 * Hk) * D + 4 * case["rotary"])                              # q in and out, k and v, rows of the tables
        n += 2 * T * Hk * (D + 1) + 2 * T * Hk * (D + 1) + 2 * T * Hk * 2 * D                # written, and read back as bf16
        return {"bytes": n, "flops": (9 if case["norms"] else 5) * T * (H + 2 * Hk) * D}
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))
    return {"bytes": 4 * T * H * D + 2 * sum(lens) * Hk * (D + 1), "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(length, rotary):
    inv = THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.outer(torch.arange(length, dtype=torch.float64, device="cuda"), inv)
    return angle.cos().float(), angle.sin().float()


def _power(y):
    """The byte of the power of two that a row is kept with: of 0.875 2^9 = 448 and the row's largest number f 2^x, f from 0.5 to 1."""
    f, x = torch.frexp(y.abs().amax(-1))
    return torch.where(f > 0, x - 9 + (f > 0.875).int(), -126).clamp(min=-126) + 127


def _unit(byte):
    """Powers of two [.., 1] of bytes [..]."""
    return (byte.int() << 23).view(torch.float32).unsqueeze(-1)


def _in_8_bits(y):
    """Rows of heads [.., D] (32 bits) as e4m3 numbers and their bytes [..]."""
    byte = _power(y)
    return (y / _unit(byte)).to(E4M3), byte.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        dtype = {"bf16": BF16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        logits = torch.empty(B, (V + 63) // 64 * 64, dtype=dtype, device="cuda")[:, :V]       # as the output head leaves them
        logits.copy_(randn(B, V) * (1.5 + 2 * rand(B, 1)))                                     # some rows flat, some with few likely tokens
        s = dict(case=case, logits=logits, u=rand(B))
        if case["each"]:
            s["temperature"] = 0.6 + 0.8 * rand(B)
            s["top_k"] = _ints([case["top_k"]] * B)
            s["top_p"] = (case["top_p"] * (1 - 0.1 * rand(B))).clamp(max=1.0)
            s["min_p"] = case["min_p"] * rand(B)
        else:
            s.update(temperature=0.8, top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        return s
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case, qw=None, kw=None)
    if case["kind"] == "norm_rope" or case.get("norms"):
        s["qw"], s["kw"] = ((1 + 0.2 * randn(D)).to(BF16) for _ in range(2))
    if case["kind"] == "norm_rope":
        B, S = case["batch"], case["seq"]
        s["qkv"] = randn(B, S, H + 2 * Hk, D).to(BF16)
        s["cos"], s["sin"] = _tables(S, case["rotary"])
        if case["train"]:
            s["grads"] = [randn(B, S, n, D).to(BF16) for n in (H, Hk, Hk)]
            for n in ("qkv", "qw", "kw"):
                s[n].requires_grad_()
        return s
    lens, new = _sequences(case)
    page, T = case["page"], sum(new)
    used = [(n + page - 1) // page for n in lens]
    width, pool = max(used) + 1, sum(used) + 1 + sum(used) // 8
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    first = [0]
    for m in new:
        first.append(first[-1] + m)
    s.update(table=table, lens=_ints(lens), cu=None if max(new) == 1 and case["chunks"] == 0 else _ints(first), most=max(new))
    for n in "kv":
        if case["kind"] == "append":
            s[n + "pages"] = torch.zeros(pool, page, Hk, D, dtype=torch.uint8, device="cuda").view(E4M3)
            s[n + "scales"] = torch.zeros(pool, Hk, page, dtype=torch.uint8, device="cuda").view(E8M0)
        else:
            # rows of different sizes, a pool's pages in four parts (its numbers in 32 bits are not wanted all at once)
            parts = [_in_8_bits(randn(len(p), page, Hk, D) * torch.exp(0.5 * randn(len(p), page, Hk, 1))) for p in torch.arange(pool).chunk(4)]
            s[n + "pages"] = torch.cat([p[0].view(torch.uint8) for p in parts]).view(E4M3)
            s[n + "scales"] = torch.cat([p[1] for p in parts]).transpose(1, 2).contiguous().view(E8M0)
    if case["kind"] == "append":
        s["qkv"] = randn(T, H + 2 * Hk, D).to(BF16)
        s["cos"], s["sin"] = _tables(case["longest"], case["rotary"])
    else:
        s["q"] = randn(T, H, D).to(BF16)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _places(s, T):
    """Sequence, place among its new tokens, and position of every token."""
    lens, cu = s["lens"].long(), s["cu"]
    t = torch.arange(T, device=lens.device)
    if cu is None:
        return t, torch.zeros_like(t), lens - 1
    cu = cu.long()
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return b, t - cu[b], lens[b] - cu[b + 1] + t


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, c, s, interleaved):
    r, rest = x[..., :2 * c.shape[-1]], x[..., 2 * c.shape[-1]:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, -1)
    lo, hi = a * c - b * s, b * c + a * s
    return torch.cat((torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1), rest), -1)


def _norm_rope(s):
    c, x = s["case"], s["qkv"]
    H, Hk = c["heads"], c["kv_heads"]
    with torch.set_grad_enabled(c["train"]):
        cos, sin = s["cos"].unsqueeze(1), s["sin"].unsqueeze(1)
        q, k = (_rotated(_normed(x[:, :, at:at + n].float(), w), cos, sin, c["interleaved"]).to(BF16)
                for at, n, w in ((0, H, s["qw"]), (H, Hk, s["kw"])))
        if not c["train"]:
            return q, k
        v = x[:, :, H + Hk:].clone()
        return q.detach(), k.detach(), *torch.autograd.grad((q, k, v), (x, s["qw"], s["kw"]), s["grads"])


def _append(s):
    c, qkv = s["case"], s["qkv"].float()
    H, Hk, page = c["heads"], c["kv_heads"], c["page"]
    b, _, pos = _places(s, qkv.shape[0])
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    q, k = (_rotated(_normed(x, w), cos, sin, c["interleaved"]) for x, w in ((qkv[:, :H], s["qw"]), (qkv[:, H:H + Hk], s["kw"])))
    at = s["table"][b, pos // page].long(), pos % page
    back = []
    for x, n in ((k, "k"), (qkv[:, H + Hk:], "v")):
        pages, scales = s[n + "pages"].view(torch.uint8), s[n + "scales"].view(torch.uint8).transpose(1, 2)
        codes, powers = _in_8_bits(x)
        pages[at], scales[at] = codes.view(torch.uint8), powers
        back.append((pages[at].view(E4M3).float() * _unit(scales[at])).to(BF16))
    return q.to(BF16), *back


def _values(s, n, table):
    """Keys or values of the pages of a table [B, pages], in 32 bits: [B, Hk, keys, D]."""
    x, e = s[n + "pages"].view(torch.uint8)[table].view(E4M3), s[n + "scales"].view(torch.uint8)[table]
    return (x.float().transpose(2, 3) * _unit(e)).transpose(1, 2).flatten(2, 3)


def _attend(s, q, lens, cu, table, n):
    """Attention of sequences with up to ``n`` new tokens each, padded to it. ``cu``: their first tokens in ``q``, and the end."""
    c, T = s["case"], q.shape[0]
    H, Hk, D, B = c["heads"], c["kv_heads"], c["dim"], lens.shape[0]
    G = H // Hk
    i = torch.arange(n, device=q.device)
    at = (cu[:-1, None] + i).clamp(max=T - 1)                                            # [B, n]: tokens
    last = (lens - cu[1:] + cu[:-1])[:, None] + i                                        # and their positions
    qs = q[at].float().view(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    x = (qs @ _values(s, "k", table).transpose(-1, -2)).view(B, Hk, G, n, -1) * D ** -0.5
    x = x.masked_fill(torch.arange(x.shape[-1], device=q.device) > last[:, None, None, :, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = (x.flatten(2, 3) @ _values(s, "v", table)).view(B, Hk, G, n, D) / x.sum(-1, keepdim=True)
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[b, t - cu[b]].to(q.dtype)


def _attention(s):
    # those with many new tokens come first: the others are not padded to the same number
    B, m, q, lens, table = s["lens"].shape[0], s["case"]["chunks"], s["q"], s["lens"].long(), s["table"].long()
    cu = torch.arange(B + 1, device=q.device) if s["cu"] is None else s["cu"].long()
    if m == 0 or m == B:
        return _attend(s, q, lens, cu, table, s["most"])
    t = q.shape[0] - (B - m)
    return torch.cat((_attend(s, q[:t], lens[:m], cu[:m + 1], table[:m], s["most"]),
                      _attend(s, q[t:], lens[m:], cu[m:] - t, table[m:], 1)))


def _sample(s):
    x = s["logits"].double()
    B, V = x.shape

    def column(a):
        return a.double()[:, None] if torch.is_tensor(a) else a

    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / column(s["temperature"]))
    k = column(s["top_k"])
    k = torch.where(k > 0, k, V) if torch.is_tensor(k) else k or V
    w = torch.where(torch.arange(V, device=x.device) < k, w, 0.0)
    upto = w.cumsum(-1)
    p = column(s["top_p"])
    keep = (upto - w < p * upto[:, -1:]) & (w >= column(s["min_p"]))
    upto = torch.zeros_like(w).scatter_(1, order, w * keep).cumsum(-1)
    return (upto <= column(s["u"]) * upto[:, -1:]).sum(-1, keepdim=True)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"norm_rope": _norm_rope, "append": _append, "attention": _attention, "sample": _sample}[kind](state)
    from ghost_flow_b200 import ops

    s, c = state, state["case"]
    if kind == "norm_rope":
        with torch.set_grad_enabled(c["train"]):
            q, k, v = ops.norm_rope_qkv(s["qkv"], c["heads"], c["kv_heads"], s["qw"], s["kw"], s["cos"], s["sin"], EPS,
                                        interleaved=c["interleaved"])
            if not c["train"]:
                return q, k
            return q.detach(), k.detach(), *torch.autograd.grad((q, k, v), (s["qkv"], s["qw"], s["kw"]), s["grads"])
    with torch.no_grad():
        if kind == "sample":
            return ops.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        pools, batch = (s["kpages"], s["vpages"]), (s["table"], s["lens"], s["cu"])
        scales = dict(kscales=s["kscales"], vscales=s["vscales"])
        if kind == "append":
            q = ops.rope_qkv_to_pages(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], *pools, *batch, interleaved=c["interleaved"],
                                      q_weight=s["qw"], k_weight=s["kw"], eps=EPS, **scales)
            return q, *ops.read_pages(q.shape[0], *pools, *batch, **scales)
        return ops.paged_attention(s["q"], *pools, *batch, **scales)


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def _turned(x, c, w, interleaved):
    """x [.., D] with pairs of its first dims as complex numbers, turned."""
    r = 2 * c.shape[-1]
    pair = x[..., :r].unflatten(-1, (r // 2, 2)) if interleaved else x[..., :r].unflatten(-1, (2, r // 2)).mT
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.complex(c, w))
    return torch.cat((y.flatten(-2) if interleaved else y.mT.flatten(-2), x[..., r:]), -1)


def _kept(y):
    """Rows [.., D] as the cache has them: multiples of an e4m3 number's last bit, in the row's unit."""
    unit = torch.exp2(torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -200) / 448)).clamp(min=-126))
    y = y / unit
    last = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / last) * last * unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        out = []
        number = lambda n, b: float(s[n][b]) if torch.is_tensor(s[n]) else s[n]  # noqa: E731
        for b in range(case["rows"]):
            p = s["logits"][b].double() / number("temperature", b)
            p = torch.softmax(p, 0)
            likely, at = torch.sort(p, descending=True, stable=True)
            k = int(number("top_k", b)) or case["vocab"]
            likely, at = likely[:k] / likely[:k].sum(), at[:k]
            n = int((likely.cumsum(0) - likely < number("top_p", b)).sum())
            likely, at = likely[:n], at[:n]
            m = int((likely >= number("min_p", b) * likely[0]).sum())
            at, by = torch.sort(at[:m])
            share = likely[:m][by].cumsum(0)
            out.append(at[int((share <= float(s["u"][b]) * share[-1]).sum())])
        return torch.stack(out)[:, None]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "norm_rope":
        x, c, w = s["qkv"].detach().double(), s["cos"].double()[:, None], s["sin"].double()[:, None]
        results, into, weights = [], [], []
        for i, (at, n, name) in enumerate(((0, H, "qw"), (H, Hk, "kw"))):
            a, weight = x[:, :, at:at + n], s[name].detach().double()
            r = 1 / torch.sqrt((a * a).sum(-1, keepdim=True) / D + EPS)
            results.append(_turned(a * r * weight, c, w, case["interleaved"]))
            if case["train"]:
                g = _turned(s["grads"][i].double(), c, -w, case["interleaved"])        # turned back
                weights.append((g * a * r).sum((0, 1, 2)))
                into.append(r * (g * weight - a * r * ((g * weight * a * r).sum(-1, keepdim=True) / D)))
        return results if not case["train"] else (*results, torch.cat([*into, s["grads"][2].double()], 2), *weights)
    lens, new = _sequences(case)
    page = case["page"]
    at = 0
    if case["kind"] == "append":
        q, k, v = [], [], []
        for n, m in zip(lens, new):
            c, w = s["cos"][n - m:n].double()[:, None], s["sin"][n - m:n].double()[:, None]
            x = s["qkv"][at:at + m].double()
            parts = [x[:, :H], x[:, H:H + Hk]]
            if case["norms"]:
                parts = [a / torch.sqrt((a * a).sum(-1, keepdim=True) / D + EPS) * s[name].double() for a, name in zip(parts, ("qw", "kw"))]
            turned = [_turned(a, c, w, case["interleaved"]) for a in parts]
            q.append(turned[0])
            k.append(_kept(turned[1]))
            v.append(_kept(x[:, H + Hk:]))
            at += m
        return torch.cat(q), torch.cat(k), torch.cat(v)
    out = torch.empty(sum(new), H, D, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(lens, new)):
        rows = s["table"][b].long()
        k, v = ((s[x + "pages"].view(torch.uint8)[rows].view(E4M3).double() *
                 torch.exp2(s[x + "scales"].view(torch.uint8)[rows].double() - 127).transpose(1, 2).unsqueeze(-1)).reshape(-1, Hk, D)[:n] for x in "kv")
        later = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
        for h in range(H):
            a = s["q"][at:at + m, h].double() @ k[:, h * Hk // H].T / math.sqrt(D)
            out[at:at + m, h] = torch.softmax(a.masked_fill(later, -math.inf), -1) @ v[:, h * Hk // H]
        at += m
    return out
