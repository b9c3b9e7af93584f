"""What stands between a model's logits and the choice of a token: penalties for tokens that are there already, biases, and masks of the
tokens that a grammar allows. The reference picks the largest logit (ghostflow-nn/src/gpt.rs:402-422).

CUDA logits of fp32, bf16 or fp16 take the kernel of ``csrc/logits.cu``; CPU tensors, other layouts, and calls that something follows (a
gradient, tracing, transforms, modes) plain PyTorch."""
from __future__ import annotations

import torch

from . import _lib
from .fused import _rc
from .paged import _is_compiling, _ranges_overlap


def pack_allowed(mask):
    """Bits of a mask ``[..., V]`` (truth values; numbers that are not 0) for :func:`process_logits`: int32 ``[..., ceil(V / 32)]``, entry ``v``
    is bit ``v % 32`` of word ``v // 32``."""
    V = mask.shape[-1]
    m = torch.nn.functional.pad((mask != 0).long(), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (m << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _logits_ref(x, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed):
    B, V = x.shape
    y = x.to(torch.promote_types(x.dtype, torch.float32))

    def column(a):         # (a number beside whole numbers would be of the default type)
        return a[:, None] if torch.is_tensor(a) else torch.full((), a, dtype=y.dtype, device=y.device)

    if tokens is not None and tokens.shape[1] > 0:
        t, j = tokens.long(), torch.arange(tokens.shape[1], device=x.device)
        there = (t >= 0) & (t < V)
        if token_lens is not None:
            there = there & (j < token_lens[:, None])
        new = there if generated_from is None else there & (j >= generated_from[:, None])
        t = torch.where(there, t, 0)
        seen, count = (torch.zeros(B, V, dtype=torch.int32, device=x.device).scatter_add_(1, t, m.int()) for m in (there, new))
        r = column(repetition)
        y = torch.where(seen > 0, torch.where(y > 0, y / r, y * r), y)
        change = count * column(frequency) + torch.where(count > 0, column(presence), 0.0)
        y = torch.where(seen > 0, y - change, y)
    if bias is not None:
        y = y + bias
    if allowed is not None:
        v = torch.arange(V, device=x.device)
        y = y.masked_fill((allowed[..., v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    return y.to(x.dtype)


def _check(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out) -> None:
    """Raises for arguments that no path takes."""
    what = "process_logits"
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"{what}: logits are [rows, vocabulary], not {logits.dtype} {list(logits.shape)}")
    (B, V), dev = logits.shape, logits.device
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != B or tokens.dtype not in (torch.int32, torch.int64) or tokens.device != dev:
            raise ValueError(f"{what}: tokens are int32 or int64 [{B}, most of a row] on {dev}, not {tokens.dtype} {list(tokens.shape)} on "
                             f"{tokens.device}")
        for name, t in (("token_lens", token_lens), ("generated_from", generated_from)):
            if t is not None and (t.shape != (B,) or t.dtype is not torch.int32 or t.device != dev):
                raise ValueError(f"{what}: {name} is int32 [{B}] on {dev}, not {t.dtype} {list(t.shape)} on {t.device}")
    elif token_lens is not None or generated_from is not None:
        raise ValueError(f"{what}: token_lens and generated_from go with tokens")
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if torch.is_tensor(t):
            if t.shape != (B,) or t.dtype is not torch.float32 or t.device != dev:
                raise ValueError(f"{what}: {name} is a number or fp32 [{B}] on {dev}, not {t.dtype} {list(t.shape)} on {t.device}")
    if not torch.is_tensor(repetition) and not 2.0 ** -126 <= repetition <= 2.0 ** 126:
        raise ValueError(f"{what}: repetition is above 0, from 2^-126 to 2^126, not {repetition}")
    if bias is not None and (bias.shape not in ((V,), (B, V)) or bias.dtype is not torch.float32 or bias.device != dev):
        raise ValueError(f"{what}: bias is fp32 [{V}] or [{B}, {V}] on {dev}, not {bias.dtype} {list(bias.shape)} on {bias.device}")
    words = (V + 31) // 32
    if allowed is not None and (allowed.dtype is not torch.int32 or allowed.shape not in ((words,), (B, words)) or allowed.device != dev):
        raise ValueError(f"{what}: allowed is int32 [{words}] or [{B}, {words}] on {dev}, not {allowed.dtype} {list(allowed.shape)} on "
                         f"{allowed.device}")
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
            raise ValueError(f"{what}: out is {list(logits.shape)} of {logits.dtype} on {dev}, not {list(out.shape)} of {out.dtype} on "
                             f"{out.device}")
        inplace = out is logits or (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride())
        if not inplace and logits.numel() and _ranges_overlap(out, logits):
            raise ValueError(f"{what}: out shares memory with logits and is not logits")
        for name, t in (("bias", bias), ("allowed", allowed), ("tokens", tokens)):
            if t is not None and t.numel() and out.numel() and _ranges_overlap(out, t):
                raise ValueError(f"{what}: out shares memory with {name}")


def _takes(out, x, others) -> bool:
    """Whether the kernel may write there."""
    return (out.shape == x.shape and out.dtype is x.dtype and out.device == x.device and out.stride(1) == 1
            and (x.shape[0] <= 1 or out.stride(0) >= x.shape[1]) and not (out.requires_grad and torch.is_grad_enabled())
            and ((out.data_ptr() == x.data_ptr() and out.stride() == x.stride()) or not _ranges_overlap(out, x))
            and not any(torch.is_tensor(t) and t.numel() and _ranges_overlap(out, t) for t in others))


def process_logits(logits, tokens=None, token_lens=None, generated_from=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                   allowed=None, out=None):
    """Logits ``[B, V]`` ready for the choice of a token. For an entry that stands ``c`` times among the row's generated tokens, in this order:
    if the row's ``tokens`` hold it at all, ``x / repetition`` where ``x > 0`` and ``x * repetition`` elsewhere, and then
    ``x - (c * frequency + presence where c > 0)``; ``x + bias``; ``-inf`` unless ``allowed``. Computed in 32 bits (the kernel multiplies by
    ``1 / repetition``) and rounded once.

    ``tokens [B, L]``, int32 or int64, holds ``token_lens[b]`` tokens (int32 ``[B]``; all ``L``) of which those from ``generated_from[b]``
    (int32 ``[B]``; 0) are generated ones, those before them the prompt; a token outside the vocabulary (padding) is passed over. The
    three penalties are numbers or fp32 ``[B]``, ``repetition`` from 2^-126 to 2^126, where it and its reciprocal have all their bits. Without
    ``tokens`` there is nothing that a penalty is for. ``bias``: fp32 ``[V]`` or ``[B, V]``. ``allowed``: int32 bits ``[words]`` or ``[B, words]``
    (:func:`pack_allowed`). ``out`` may be ``logits`` itself. A row of which nothing is allowed is all ``-inf``."""
    call = None
    if logits.get_device() >= 0 and not _is_compiling():
        call = _lib.calls().logits(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed)
        if call is not None and out is not None and not _takes(out, logits, (repetition, presence, frequency, bias, tokens, allowed)):
            call = None
    if call is None:
        _check(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out)
        if logits.numel() == 0:
            return torch.empty_like(logits) if out is None else out
        y = _logits_ref(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed)
        return y if out is None else out.copy_(y)
    at, device, B, V, ld = call
    stream = _lib.stream_on(device)
    if stream is None:
        with torch.cuda.device(device):
            return process_logits(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out)
    if out is not None:
        y, ldy = out, out.stride(0)
    else:
        # rows as far apart as they are, where they are apart: they then begin on the same boundaries
        ldy = ld if V <= ld < V + 64 else V
        y = logits.new_empty_strided((B, V), (ldy, 1))
    _rc(_lib.calls().run_logits(at, y, ldy, stream), "gf_process_logits")
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return y


def counts_tokens(choice) -> bool:
    """Whether keyword arguments of :func:`next_tokens` have a penalty, which wants to know the tokens so far."""
    return not choice.keys().isdisjoint(("repetition", "presence", "frequency"))


def next_tokens(logits, temperature: float = 0.0, tokens=None, token_lens=None, generated_from=None, prompt: int | None = None,
                repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """The next token ``[B, 1]`` of every row of ``logits [B, V]``: the likeliest (temperature 0) or a sampled one, after
    :func:`process_logits` where ``tokens``, a bias or a mask are given: -1 then for a row that they leave nothing of (all ``-inf``), for which
    an embedding has zeros and :func:`process_logits` no penalty. Sampling takes the likeliest token of a row that has no probabilities (it
    holds what is not a number, or infinity). ``prompt``: the number of tokens of every row that are its prompt, in place of ``generated_from``."""
    if tokens is None and any(torch.is_tensor(t) or t != none for t, none in ((repetition, 1), (presence, 0), (frequency, 0))):
        raise ValueError("next_tokens: penalties go with the tokens that they count")
    processed = tokens is not None or bias is not None or allowed is not None
    if processed:
        if tokens is not None and generated_from is None and prompt is not None:
            generated_from = torch.full((logits.shape[0],), prompt, dtype=torch.int32, device=logits.device)
        logits = process_logits(logits, tokens, token_lens if tokens is not None else None, generated_from if tokens is not None else None,
                                repetition, presence, frequency, bias, allowed)
    likeliest = chosen = logits.argmax(-1, keepdim=True)
    if temperature and temperature > 0:
        # multinomial stops the device at a row that is no distribution; softmax leaves nothing but NaN of one
        p = torch.softmax(logits.float() / temperature, -1)
        none = p[..., :1].isnan()
        chosen = torch.where(none, likeliest, torch.multinomial(p.masked_fill(none, 1.0), 1))
    return torch.where(logits.gather(-1, likeliest) == float("-inf"), -1, chosen) if processed else chosen
