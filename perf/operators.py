"""The operators of a serving step over a paged KV cache, as work to be timed: keys and values appended to the cache with
the rotation on the way, attention of new tokens over the cache, and penalties, biases and grammar masks on logits.

A case is a dict of plain values; ``kind`` names the operator, the rest are its sizes. ``listed()`` gives the cases that stand
for the ranges, ``draw(rng)`` another one of the same ranges. With ``own`` the calls are the framework's, else elementary
torch operations in 32 bits; ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
THETA = 10000.0


# ------------------------------------------------------------------------------------------ the cases
# Sequences: `batch` of them with `shortest` .. `longest` keys (new tokens among them). The first `chunks` of them have up to `chunk`
# new tokens (0: the whole sequence is new), the others one.
def listed():
    return [
        # one token of each of 64 sequences in a server's batch, Mixtral's heads, the smallest pages
        dict(name="append_decode", kind="append", batch=64, shortest=17, longest=2000, chunks=0, chunk=1, heads=32, kv_heads=8, dim=128,
             page=16, interleaved=False),
        # five prompts of different lengths at once, LLaMA-7B's heads
        dict(name="append_prompts", kind="append", batch=5, shortest=301, longest=1507, chunks=5, chunk=0, heads=32, kv_heads=32, dim=128,
             page=64, interleaved=False),
        # the smallest call: a small model, three sequences, pairs next to each other
        dict(name="append_small", kind="append", batch=3, shortest=20, longest=57, chunks=0, chunk=1, heads=4, kv_heads=2, dim=64,
             page=16, interleaved=True),
        # one token of each of 32 sequences of mixed lengths, Mixtral's heads
        dict(name="paged_decode", kind="attention", batch=32, shortest=100, longest=4096, chunks=0, chunk=1, heads=32, kv_heads=8, dim=128,
             page=16),
        # few long sequences, eight query heads to a KV head
        dict(name="paged_decode_long", kind="attention", batch=4, shortest=20011, longest=30001, chunks=0, chunk=1, heads=64, kv_heads=8,
             dim=128, page=64),
        # the smallest call: a small model, three short sequences
        dict(name="paged_decode_small", kind="attention", batch=3, shortest=20, longest=57, chunks=0, chunk=1, heads=4, kv_heads=2, dim=64,
             page=16),
        # the next chunk of a long prompt
        dict(name="paged_chunk", kind="attention", batch=1, shortest=7681, longest=7681, chunks=1, chunk=512, heads=32, kv_heads=8, dim=128,
             page=16),
        # a server's step: one sequence's chunk of the prompt among 31 that generate
        dict(name="paged_mixed", kind="attention", batch=32, shortest=130, longest=2048, chunks=1, chunk=481, heads=32, kv_heads=8, dim=128,
             page=32),
        # whole prompts of different lengths, LLaMA-7B's heads
        dict(name="paged_prompts", kind="attention", batch=4, shortest=999, longest=2987, chunks=4, chunk=0, heads=32, kv_heads=32, dim=128,
             page=64),
        # logits of a small batch, all penalties, a short history
        dict(name="logits_small", kind="logits", rows=3, vocab=32000, history=60, dtype="bf16", penalties=True, bias=False, mask=False),
        # logits of a server's batch over the GPT-2 vocabulary (rows padded as the output head leaves them), penalties and grammars
        dict(name="logits_server", kind="logits", rows=64, vocab=50257, history=2048, dtype="bf16", penalties=True, bias=False, mask=True),
        # the largest: 32-bit logits of a large batch, a long history, one bias for all rows
        dict(name="logits_large", kind="logits", rows=512, vocab=50257, history=4096, dtype="fp32", penalties=True, bias=True, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12, 64), (16, 2, 64), (25, 25, 64), (4, 2, 64), (32, 32, 128), (32, 8, 128), (40, 40, 128), (64, 8, 128), (16, 1, 128),
         (10, 2, 128)]


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "logits"])
    if kind == "logits":
        vocab, dtype = rng.choice([1000, 30522, 32000, 50257]), rng.choice(["bf16", "bf16", "fp32", "fp16"])
        penalties = rng.random() < 0.8
        return dict(kind=kind, rows=_log(rng, 1, 512), vocab=vocab, history=_log(rng, 1, 4096), dtype=dtype, penalties=penalties,
                    bias=rng.random() < 0.4, mask=not penalties or rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice(HEADS)
    page = rng.choice([16, 16, 32, 64, 128, 256])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    if kind == "append":
        c["interleaved"] = rng.random() < 0.3
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
    if case["kind"] == "logits":
        b, v, size = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
        n = 2 * b * v * size + (b * v // 8 if case["mask"] else 0) + (4 * v if case["bias"] else 0)
        n += sum(_histories(case)[0]) * 4 + 20 * b if case["penalties"] else 0
        return {"bytes": n, "flops": 6 * b * v}
    lens, new = _sequences(case)
    H, Hk, D, T = case["heads"], case["kv_heads"], case["dim"], sum(new)
    if case["kind"] == "append":
        return {"bytes": T * (4 * (H + 2 * Hk) * D + 4 * D), "flops": 3 * T * (H + Hk) * D}
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))
    return {"bytes": 4 * T * H * D + 4 * sum(lens) * Hk * D, "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _histories(c):
    rng = random.Random(c["rows"] * 7 + c["history"])
    lens = [rng.randint((c["history"] + 1) // 2, c["history"]) for _ in range(c["rows"])]
    return lens, [rng.randint(0, n) for n in lens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["kind"] == "logits":
        B, V = case["rows"], case["vocab"]
        dtype = {"bf16": BF16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        logits = torch.empty(B, (V + 63) // 64 * 64, dtype=dtype, device="cuda")[:, :V]       # as the output head leaves them
        logits.copy_(3 * randn(B, V))
        s = dict(case=case, logits=logits, tokens=None, bias=None, allowed=None)
        if case["penalties"]:
            lens, first = _histories(case)
            # few tokens come often, most hardly ever
            u = torch.rand(B, case["history"], generator=g, device="cuda")
            s["tokens"] = (V * u.pow(4)).to(torch.int32).clamp_(max=V - 1)
            s["token_lens"], s["generated_from"] = _ints(lens), _ints(first)
            s["repetition"] = 1 + 0.5 * torch.rand(B, generator=g, device="cuda")
            s["presence"], s["frequency"] = (0.8 * torch.rand(B, generator=g, device="cuda") for _ in range(2))
        if case["bias"]:
            s["bias"] = torch.where(torch.rand(V, generator=g, device="cuda") < 0.01, 5 * randn(V), 0.0)
        if case["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device="cuda").to(torch.int32)
        return s
    lens, new = _sequences(case)
    H, Hk, D, page, T = case["heads"], case["kv_heads"], case["dim"], case["page"], sum(new)
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
    s = dict(case=case, kpages=randn(pool, page, Hk, D).to(BF16), vpages=randn(pool, page, Hk, D).to(BF16), table=table, lens=_ints(lens),
             cu=None if max(new) == 1 and case["chunks"] == 0 else _ints(first), most=max(new))
    if case["kind"] == "append":
        s["qkv"] = randn(T, H + 2 * Hk, D).to(BF16)
        inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        angle = torch.outer(torch.arange(case["longest"], dtype=torch.float64), inv)
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
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


def _rotated(x, c, s, interleaved):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    lo, hi = a * c - b * s, b * c + a * s
    return torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)


def _append(s):
    c, qkv = s["case"], s["qkv"].float()
    H, Hk, page = c["heads"], c["kv_heads"], c["page"]
    b, _, pos = _places(s, qkv.shape[0])
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    rotated = _rotated(qkv[:, :H + Hk], cos, sin, c["interleaved"]).to(BF16)
    at = s["table"][b, pos // page].long(), pos % page
    s["kpages"][at] = rotated[:, H:]
    s["vpages"][at] = s["qkv"][:, H + Hk:]
    return rotated[:, :H].contiguous(), s["kpages"], s["vpages"]


def _attend(s, q, lens, cu, table, n):
    """Attention of sequences with up to ``n`` new tokens each, padded to it. ``cu``: their first tokens in ``q``, and the end."""
    c, T = s["case"], q.shape[0]
    H, Hk, D, B = c["heads"], c["kv_heads"], c["dim"], lens.shape[0]
    G = H // Hk
    i = torch.arange(n, device=q.device)
    at = (cu[:-1, None] + i).clamp(max=T - 1)                                            # [B, n]: tokens
    last = (lens - cu[1:] + cu[:-1])[:, None] + i                                        # and their positions
    qs = q[at].float().view(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    k, v = (x[table].flatten(1, 2).transpose(1, 2).float() for x in (s["kpages"], s["vpages"]))
    x = (qs @ k.transpose(-1, -2)).view(B, Hk, G, n, -1) * D ** -0.5
    x = x.masked_fill(torch.arange(x.shape[-1], device=q.device) > last[:, None, None, :, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = (x.flatten(2, 3) @ v).view(B, Hk, G, n, D) / x.sum(-1, keepdim=True)
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


def _logits(s):
    x = s["logits"].float()
    B, V = x.shape
    if s["tokens"] is not None:
        t, j = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device=x.device)
        there = j < s["token_lens"][:, None]
        count = torch.zeros(2, B, V, dtype=torch.int32, device=x.device)
        count[0].scatter_add_(1, t, there.int())
        count[1].scatter_add_(1, t, (there & (j >= s["generated_from"][:, None])).int())
        r, p, f = (s[k][:, None] for k in ("repetition", "presence", "frequency"))
        x = torch.where(count[0] > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - (count[1] * f + (count[1] > 0) * p)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(V, device=x.device)
        x = x.masked_fill((s["allowed"][:, v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    return x.to(s["logits"].dtype)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"append": _append, "attention": _attention, "logits": _logits}[kind](state)
    from ghost_flow_b200 import ops

    s, c = state, state["case"]
    with torch.no_grad():
        if kind == "append":
            q = ops.rope_qkv_to_pages(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], s["kpages"], s["vpages"], s["table"],
                                      s["lens"], s["cu"], interleaved=c["interleaved"])
            return q, s["kpages"], s["vpages"]
        if kind == "attention":
            return ops.paged_attention(s["q"], s["kpages"], s["vpages"], s["table"], s["lens"], s["cu"])
        if s["tokens"] is None:
            return ops.process_logits(s["logits"], bias=s["bias"], allowed=s["allowed"])
        return ops.process_logits(s["logits"], s["tokens"], s["token_lens"], s["generated_from"], repetition=s["repetition"],
                                  presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logits":
        out = s["logits"].double()
        B, V = out.shape
        if s["tokens"] is not None:
            lens, first = _histories(case)
            for b in range(B):
                t = s["tokens"][b].long()
                seen = torch.bincount(t[:lens[b]], minlength=V) > 0
                often = torch.bincount(t[first[b]:lens[b]], minlength=V).double()
                r = s["repetition"][b].double()
                row = out[b]
                row = torch.where(seen, row * r ** (1 - 2 * (row > 0).double()), row)
                out[b] = row - often * s["frequency"][b].double() - often.clamp(max=1) * s["presence"][b].double()
        if s["bias"] is not None:
            out += s["bias"].double()
        if s["allowed"] is not None:
            bits = torch.arange(32, device="cuda", dtype=torch.int32)
            open_ = ((s["allowed"].unsqueeze(-1) >> bits) & 1).flatten(1)[:, :V].bool()
            out[~open_] = -math.inf
        return out
    lens, new = _sequences(case)
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    at = 0
    if case["kind"] == "append":
        q, pages = [], [s["kpages"].double(), s["vpages"].double()]
        for b, (n, m) in enumerate(zip(lens, new)):
            pos = torch.arange(n - m, n, device="cuda")
            x, c, w = s["qkv"][at:at + m].double(), s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
            pair = x[:, :H + Hk].reshape(m, H + Hk, D // 2, 2) if case["interleaved"] else x[:, :H + Hk].reshape(m, H + Hk, 2, D // 2).mT
            turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.complex(c, w))
            y = turned.flatten(-2) if case["interleaved"] else turned.mT.flatten(-2)
            row = s["table"][b].long()[pos // page] * page + pos % page
            pages[0].view(-1, Hk, D)[row] = y[:, H:]
            pages[1].view(-1, Hk, D)[row] = x[:, H + Hk:]
            q.append(y[:, :H])
            at += m
        return torch.cat(q), *pages
    out = torch.empty(sum(new), H, D, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = (x[s["table"][b].long()].reshape(-1, Hk, D)[:n].double() for x in (s["kpages"], s["vpages"]))
        later = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
        for h in range(H):
            a = s["q"][at:at + m, h].double() @ k[:, h * Hk // H].T / math.sqrt(D)
            out[at:at + m, h] = torch.softmax(a.masked_fill(later, -math.inf), -1) @ v[:, h * Hk // H]
        at += m
    return out
