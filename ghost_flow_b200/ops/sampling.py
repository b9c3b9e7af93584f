"""What stands between a model's logits and the choice of a token: penalties for tokens that are there already, biases, and masks of the
tokens that a grammar allows. The reference picks the largest logit (ghostflow-nn/src/gpt.rs:402-422).

CUDA logits of fp32, bf16 or fp16 take the kernel of ``csrc/logits.cu``; CPU tensors, other layouts, and calls that something follows (a
gradient, tracing, transforms, modes) plain PyTorch."""
from __future__ import annotations

import struct

import torch

from . import _lib
from .fused import _observed, _rc
from .paged import _ranges_overlap

_CALL = struct.Struct("16q3d4q").pack      # the LogitsCall of csrc/logits.cu
_WHOLE = (torch.int32, torch.int64)
_KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def pack_allowed(mask):
    """Bits of a truth-valued mask ``[..., V]`` for :func:`process_logits`: int32 ``[..., ceil(V / 32)]``, entry ``v`` is bit ``v % 32`` of word
    ``v // 32``."""
    V = mask.shape[-1]
    m = torch.nn.functional.pad(mask.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (m << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _logits_ref(x, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed):
    B, V = x.shape
    y = x.to(torch.promote_types(x.dtype, torch.float32))

    def column(a):
        return a[:, None] if torch.is_tensor(a) else a

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
    if not torch.is_tensor(repetition) and not repetition > 0:
        raise ValueError(f"{what}: repetition is above 0, not {repetition}")
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


def _row(t, B, device, dtype) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.dim() == 1 and t.shape[0] == B and t.stride(0) == 1


def _for_kernel(x, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out):
    """Device, rows, vocabulary and distance of rows of a call that the kernel takes, in few looks at the tensors. ``None``: see :func:`_check`."""
    device = x.get_device()
    if device < 0 or x.dim() != 2 or x.dtype not in _KINDS or _observed():
        return None
    (B, V), (ld, one) = x.shape, x.stride()
    if B == 0 or V == 0 or one != 1:
        return None
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != B or tokens.dtype not in _WHOLE or tokens.get_device() != device or tokens.stride(1) != 1 \
                or not (token_lens is None or _row(token_lens, B, device, torch.int32)) \
                or not (generated_from is None or _row(generated_from, B, device, torch.int32)):
            return None
    elif token_lens is not None or generated_from is not None:
        return None
    grad = torch.is_grad_enabled()
    if grad and x.requires_grad:
        return None
    for t in (repetition, presence, frequency):
        if type(t) is not float and torch.is_tensor(t) and (not _row(t, B, device, torch.float32) or (grad and t.requires_grad)):
            return None
    if not torch.is_tensor(repetition) and not repetition > 0:
        return None
    if bias is not None and (bias.dtype is not torch.float32 or bias.get_device() != device or bias.shape not in ((V,), (B, V))
                             or bias.stride(-1) != 1 or (grad and bias.requires_grad)):
        return None
    if allowed is not None and (allowed.dtype is not torch.int32 or allowed.get_device() != device or allowed.stride(-1) != 1
                                or allowed.shape not in (((V + 31) // 32,), (B, (V + 31) // 32))):
        return None
    if out is not None:
        if out.shape != x.shape or out.dtype is not x.dtype or out.get_device() != device or out.stride(1) != 1 \
                or (B > 1 and out.stride(0) < V) or (grad and out.requires_grad):
            return None
        if not (out.data_ptr() == x.data_ptr() and out.stride(0) == ld) and _ranges_overlap(out, x):
            return None
        for t in (bias, allowed, tokens):
            if t is not None and t.numel() and _ranges_overlap(out, t):
                return None
    return device, B, V, ld


def process_logits(logits, tokens=None, token_lens=None, generated_from=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                   allowed=None, out=None):
    """Logits ``[B, V]`` ready for the choice of a token. For an entry that stands ``c`` times among the row's generated tokens, in this order:
    if the row's ``tokens`` hold it at all, ``x / repetition`` where ``x > 0`` and ``x * repetition`` elsewhere, and then
    ``x - (c * frequency + presence where c > 0)``; ``x + bias``; ``-inf`` unless ``allowed``. Computed in 32 bits and rounded once.

    ``tokens [B, L]``, int32 or int64, holds ``token_lens[b]`` tokens (int32 ``[B]``; all ``L``) of which those from ``generated_from[b]``
    (int32 ``[B]``; 0) are generated ones, those before them the prompt; a token outside the vocabulary (padding) is passed over. The
    three penalties are numbers or fp32 ``[B]``. ``bias``: fp32 ``[V]`` or ``[B, V]``. ``allowed``: int32 bits ``[words]`` or ``[B, words]``
    (:func:`pack_allowed`). ``out`` may be ``logits`` itself. A row of which nothing is allowed is all ``-inf``."""
    call = _for_kernel(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out)
    if call is None:
        _check(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out)
        if logits.numel() == 0:
            return torch.empty_like(logits) if out is None else out
        y = _logits_ref(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed)
        return y if out is None else out.copy_(y)
    device, B, V, ld = call
    stream = _lib.stream_on(device)
    if stream is None:
        with torch.cuda.device(device):
            return process_logits(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed, out)
    if out is not None:
        y, ldy = out, out.stride(0)
    else:
        # rows as far apart as they are, where they are apart: they then begin on the same boundaries
        ldy = ld if V <= ld < V + 64 else V
        y = torch.empty_strided((B, V), (ldy, 1), dtype=logits.dtype, device=logits.device)
    r, p, f = (t if type(t) is float else None if torch.is_tensor(t) else float(t) for t in (repetition, presence, frequency))
    if tokens is None:
        t, ldt, wide, L = 0, 0, 0, 0
    else:
        t, ldt, wide, L = tokens.data_ptr(), tokens.stride(0), tokens.dtype is torch.int64, tokens.shape[1]
    _rc(_lib.cuda_lib().gf_process_logits(_CALL(
        logits.data_ptr(), ld, y.data_ptr(), ldy, _KINDS[logits.dtype], B, V, t, ldt, wide, L,
        0 if token_lens is None else token_lens.data_ptr(), 0 if generated_from is None else generated_from.data_ptr(),
        repetition.data_ptr() if r is None else 0, presence.data_ptr() if p is None else 0, frequency.data_ptr() if f is None else 0,
        r or 0.0, p or 0.0, f or 0.0, 0 if bias is None else bias.data_ptr(), 0 if bias is None or bias.dim() == 1 else bias.stride(0),
        0 if allowed is None else allowed.data_ptr(), 0 if allowed is None or allowed.dim() == 1 else allowed.stride(0)), stream),
        "gf_process_logits")
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return y


def next_tokens(logits, temperature: float = 0.0, tokens=None, token_lens=None, generated_from=None, prompt: int | None = None,
                repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """The next token ``[B, 1]`` of every row of ``logits [B, V]``: the likeliest (temperature 0) or a sampled one, after
    :func:`process_logits` where ``tokens``, a bias or a mask are given. ``prompt``: the number of tokens of every row that are its prompt,
    in place of ``generated_from``."""
    if tokens is not None or bias is not None or allowed is not None:
        if tokens is not None and generated_from is None and prompt is not None:
            generated_from = torch.full((logits.shape[0],), prompt, dtype=torch.int32, device=logits.device)
        logits = process_logits(logits, tokens, token_lens if tokens is not None else None, generated_from if tokens is not None else None,
                                repetition, presence, frequency, bias, allowed)
    if temperature and temperature > 0:
        return torch.multinomial(torch.softmax(logits.float() / temperature, -1), 1)
    return logits.argmax(-1, keepdim=True)
