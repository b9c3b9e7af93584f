"""A KV cache in pages: appending the keys and values of new tokens with the rotation on the way, and attention of new tokens
(one of each sequence, chunks of prompts, whole prompts, any mix of them) over it.

``kpages`` and ``vpages`` are pools ``[pages, page, Hk, D]``; row ``b`` of ``page_table`` (int32 ``[B, width]``) names the pages of
sequence ``b`` in their order. New tokens of all sequences lie one behind the other: those of sequence ``b`` are rows ``cu[b] .. cu[b + 1] - 1``
(``cu`` int32 ``[B + 1]``; without it every sequence has one), and ``lens[b]`` (int32) counts its keys with the new ones, so that new token
``i`` of ``n`` stands at position ``lens[b] - n + i``. All of these stay on the device and nothing here waits for them: a captured call goes by
what they hold when it is replayed. A sequence of no new tokens, or of no keys (an empty slot of a batch), is allowed.

bf16 CUDA tensors take the kernels of ``csrc/paged_cache.cu`` and ``csrc/attn_paged.cu`` (through ``csrc/calls.cpp``); other types, layouts and CPU tensors, and calls that
something follows (a gradient, tracing, transforms, modes), plain PyTorch. The reference has no cache (ghostflow-nn/src/gpt.rs:402-422).
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .fused import _observed, _rc, _rows_apart
from .gemm import _SMS, _sm_count
from .raw import _SLICES, _decode_parts

_INT32, _BF16 = torch.int32, torch.bfloat16
_OVERLAP = -5      # GFH_OVERLAP of csrc/gf_host.h
_increment_version = torch.autograd.graph.increment_version
_is_compiling = torch.compiler.is_compiling


def _check_batch(what, x, kpages, vpages, page_table, lens, cu) -> None:
    """Raises for arguments that no batch has, whatever path it takes."""
    if kpages.dim() != 4 or kpages.shape != vpages.shape or kpages.dtype != x.dtype or vpages.dtype != x.dtype:
        raise ValueError(f"{what}: kpages and vpages are [pages, page, KV heads, head size] of {x.dtype}, not {list(kpages.shape)} of "
                         f"{kpages.dtype} and {list(vpages.shape)} of {vpages.dtype}")
    if kpages.shape[1] < 1:
        raise ValueError(f"{what}: pages of {kpages.shape[1]} rows")
    B = lens.shape[0] if lens.dim() == 1 else -1
    if B < 0 or page_table.dim() != 2 or page_table.shape[0] != B or lens.dtype is not _INT32 or page_table.dtype is not _INT32:
        raise ValueError(f"{what}: page_table is int32 [sequences, pages of each] and lens int32 [sequences], not {page_table.dtype} "
                         f"{list(page_table.shape)} and {lens.dtype} {list(lens.shape)}")
    if cu is not None and (cu.dtype is not _INT32 or cu.shape != (B + 1,)):
        raise ValueError(f"{what}: cu is int32 [{B + 1}], the first token of each of {B} sequences and the end, not {cu.dtype} {list(cu.shape)}")
    if cu is None and x.shape[0] != B:
        raise ValueError(f"{what}: {x.shape[0]} tokens of {B} sequences need cu, the first token of each")
    dev = x.device
    if not (kpages.device == vpages.device == page_table.device == lens.device == dev and (cu is None or cu.device == dev)):
        raise ValueError(f"{what}: tensors on different devices")


def _pages_apart(P, page, Hk, D, pools) -> bool:
    """Whether no two rows of the pools share memory (addresses of bf16, strides of pages, rows and heads of each)."""
    k, v, a0, a1, a2, b0, b1, b2 = pools
    between = abs(k - v) // 2
    if a2 == b2 == D and a1 == b1 == Hk * D and a0 == b0 == page * a1:         # two dense pools
        return between >= P * a0
    dims = ((a0, P), (a1, page), (a2, Hk)), ((b0, P), (b1, page), (b2, Hk))
    if dims[0] == dims[1]:                 # the pools themselves are one more dimension
        return _rows_apart(D, [*dims[0], (between, 2)])
    ends = sorted((at, at + 2 * (D + sum(st * (n - 1) for st, n in d))) for at, d in zip((k, v), dims))
    return all(_rows_apart(D, d) for d in dims) and ends[0][1] <= ends[1][0]


def _report(device, bad, what: str) -> None:
    """A batch that names pages or positions that are not there: an error on the CPU, else the status word's (see ``_lib.check_status``)."""
    if device.type != "cuda":
        if bool(bad):
            raise ValueError(f"{what}: a page or a position that is not there")
        return
    w = _lib.status_word(device)
    w[0] = torch.where(bad & (w[0] == 0), 7, w[0])


def _places(T, lens, cu):
    """Sequence (that of the last one behind it), position, and whether it belongs to a sequence, of every token."""
    B = lens.shape[0]
    t = torch.arange(T, device=lens.device)
    if cu is None:
        return t, lens.long() - 1, torch.ones_like(t, dtype=torch.bool)
    c = cu.long().clamp(0, T)
    b = torch.searchsorted(c[1:].contiguous(), t, right=True)
    inside = (b < B) & (t >= c[0])
    b = b.clamp(max=max(int(B) - 1, 0))        # (a number under tracing too)
    return b, lens.long()[b] - c[b + 1] + t, inside


# ------------------------------------------------------------------------------------------ append
def _append_ref(qkv, H, Hk, cos, sin, kpages, vpages, page_table, lens, cu, interleaved):
    (P, page, _, D), T, dev = kpages.shape, qkv.shape[0], qkv.device
    up = torch.promote_types(qkv.dtype, torch.float32)
    b, pos, inside = _places(T, lens, cu)
    here = inside & (pos >= 0)
    fits = here & (pos < page_table.shape[1] * page) & (pos < cos.shape[0])
    at = torch.where(fits, pos, 0)
    stored = fits
    if page_table.shape[1]:
        pages = page_table.long()[b, at // page]
        stored = fits & (pages >= 0) & (pages < P)
    _report(dev, (here & ~stored).any(), "rope_qkv_to_pages")
    if cos.shape[0]:
        c, s = (t[at].to(up).unsqueeze(1) for t in (cos, sin))
    else:
        c = s = torch.zeros(T, 1, D // 2, dtype=up, device=dev)
    x = qkv[:, :H + Hk].to(up)
    lo, hi = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    lo, hi = lo * c - hi * s, hi * c + lo * s
    x = torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)
    x = x.masked_fill(~fits[:, None, None], 0).to(qkv.dtype)
    if bool(stored.any()):
        where = pages[stored], at[stored] % page
        kpages[where] = x[stored, H:]
        vpages[where] = qkv[stored, H + Hk:]
    return x[:, :H].contiguous()


def rope_qkv_to_pages(qkv, num_heads: int, num_kv_heads: int, cos, sin, kpages, vpages, page_table, lens, cu=None,
                      interleaved: bool = False):
    """Rotated q ``[T, H, D]`` of a packed projection output ``[T, H + 2 Hk, D]`` of new tokens; rotated k and v go to the rows of their
    positions in the pages (see the module). ``cos`` and ``sin`` as for :func:`rope`, a row for each position. Two sequences may share
    pages, but not rows that are written here. Tokens behind the last sequence are left out, and their rows of q are not written; those of
    a sequence that holds fewer keys than new tokens give zeros where their position is below 0. A page that is not in the pools,
    or a position that is not in the tables or behind the page table, is left out too, and ``_lib.check_status`` raises.
    Inference only: a call with a gradient to record takes PyTorch's operations."""
    H, Hk = num_heads, num_kv_heads
    call = None
    if qkv.get_device() >= 0 and not _is_compiling():
        call = _lib.calls().append(qkv, H, Hk, kpages, vpages, page_table, lens, cu, cos, sin)
        if call is not None and call[5] is not None and not _pages_apart(*kpages.shape, call[5]):
            call = None
    if call is None:
        what = "rope_qkv_to_pages"
        if qkv.dim() != 3 or qkv.shape[1] != H + 2 * Hk or H < 1 or Hk < 1:
            raise ValueError(f"{what}: a packed projection of {H} + 2 x {Hk} heads is [tokens, {H + 2 * Hk}, head size], not {list(qkv.shape)}")
        _check_batch(what, qkv, kpages, vpages, page_table, lens, cu)
        T, _, D = qkv.shape
        if kpages.shape[2] != Hk or kpages.shape[3] != D or D % 2:
            raise ValueError(f"{what}: pages of {kpages.shape[2]} heads of {kpages.shape[3]} for {Hk} heads of {D}")
        if not (cos.dim() == 2 and cos.shape == sin.shape and 2 * cos.shape[1] == D and cos.device == sin.device == qkv.device):
            raise ValueError(f"{what}: rope tables must be [positions, {D // 2}] on {qkv.device}, got {list(cos.shape)} on {cos.device} and "
                             f"{list(sin.shape)} on {sin.device}")
        if T == 0 or lens.shape[0] == 0:
            return qkv.new_zeros(T, H, D)
        if kpages.numel() and not _observed() and (_ranges_overlap(qkv, kpages) or _ranges_overlap(qkv, vpages)):
            raise ValueError(f"{what}: qkv shares memory with the pages")
        return _append_ref(qkv, H, Hk, cos, sin, kpages, vpages, page_table, lens, cu, interleaved)
    at, device, T, D, packed, _ = call
    stream = _lib.stream_on(device)
    if stream is None:
        with torch.cuda.device(device):
            return rope_qkv_to_pages(qkv, H, Hk, cos, sin, kpages, vpages, page_table, lens, cu, interleaved)
    if not packed:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        at = _lib.calls().append(qkv, H, Hk, kpages, vpages, page_table, lens, cu, cos, sin)[0]
    q = qkv.new_empty(T, H, D)
    rc = _lib.calls().run_append(at, q, interleaved, _lib.status_ptr(device), stream)
    if rc == _OVERLAP:
        raise ValueError("rope_qkv_to_pages: qkv shares memory with the pages")
    _rc(rc, "gf_paged_append")
    _increment_version((kpages, vpages))     # a graph that saved the pools has to notice the write
    return q


# ------------------------------------------------------------------------------------------ attention
# A batch of this many sequences may be a server's, most of which have one new token: those then go to the decode kernel, which reads keys
# twice as fast as the tiles for prompts do, for one or two launches more. us, tiles alone / decode kernel beside them, 32 / 8 heads of 128, one chunk and the
# others one token over up to so many keys: 2 sequences, 64 new tokens over 500 18 / 23, 512 over 8000 53 / 68; 7 sequences, 64 over 500 18 / 27, 64 over 2000
# 31 / 35, 512 over 2000 43 / 47, 64 over 8000 68 / 74, but 512 over 8000 129 / 96.
_MANY = 8


def _parts_beside(heads: int, sms: int) -> int:
    """How the decode kernel cuts keys (see ``raw._decode_parts``) beside a kernel that holds SMs for as long as it takes: into so few parts of
    each sequence that they are 1.5 for an SM. Equal shares of all keys, one for every place on the machine, then wait for their places: 64
    sequences of up to 2000 keys, one of them with 16 new tokens, 32 / 8 heads of 128, us with shares / 1 / 2 / 4 parts 90 / 64 / 67 / 72, 32 of up to
    4096, one with 256 90 / 83 / 91 / 87, 16 of up to 8000, one with 64 89 / 132 / 96 / 98."""
    return next((s for s in _SLICES if 2 * heads * s >= 3 * sms), _SLICES[-1])


@functools.lru_cache(maxsize=4096)
def _attention_workspace(device: int, B: int, T: int, one_each: bool, ones: bool, keys: int, H: int, Hk: int, D: int) -> int:
    """Bytes that a call leaves the results of pieces in (the number of SMs decides whether keys, ``keys`` of a sequence at most, are cut)."""
    return _lib.cuda_lib().gf_paged_attn_workspace(B, T, 1 if one_each else 0, 1 if ones else 0, keys, H, Hk, D)


def _attention_ref(q, kpages, vpages, page_table, lens, cu, scale, out):
    (P, page, Hk, D), (T, H, _), dev, B = kpages.shape, q.shape, q.device, lens.shape[0]
    up = torch.promote_types(q.dtype, torch.float32)
    ends = list(range(B + 1)) if cu is None else cu.clamp(0, T).tolist()
    bad, at, pieces = torch.zeros((), dtype=torch.bool, device=dev), 0, []
    for b, length in enumerate(lens.tolist()):
        n = max(0, min(length, page_table.shape[1] * page))
        s, e = ends[b], ends[b + 1]
        if n != length:
            bad = bad | True
        if e <= s:
            continue
        pages = page_table[b, :(n + page - 1) // page].long()
        there = (pages >= 0) & (pages < P)
        bad = bad | ~there.all()
        k, v = (x[pages.clamp(0, max(P - 1, 0))].to(up).masked_fill(~there[:, None, None, None], 0).flatten(0, 1)[:n] if P else
                torch.zeros(n, Hk, D, dtype=up, device=dev) for x in (kpages, vpages))
        x = torch.einsum("thgd,nhd->hgtn", q[s:e].to(up).unflatten(1, (Hk, H // Hk)), k) * scale
        last = length - (e - s) + torch.arange(e - s, device=dev)
        hidden = torch.arange(n, device=dev) > last[:, None]
        x = torch.softmax(x.masked_fill(hidden, float("-inf")), -1).masked_fill(hidden, 0)     # rows without a key: zeros
        o = torch.einsum("hgtn,nhd->thgd", x, v).flatten(1, 2).to(q.dtype)
        if out is not None:
            out[s:e] = o
        else:
            pieces += [q.new_zeros(s - at, H, D), o] if s > at else [o]
            at = e
    _report(dev, bad, "paged_attention")
    if out is not None:
        return out
    return torch.cat([*pieces, q.new_zeros(T - at, H, D)])


def _ranges_overlap(a, b) -> bool:
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def paged_attention(q, kpages, vpages, page_table, lens, cu=None, scale: float | None = None, out=None):
    """Causal attention of new tokens ``q [T, Hq, D]`` over the keys of their sequences in the pages (see the module), which hold the new
    tokens' own already: a token at position ``p`` sees the keys ``0 .. p``. A token that sees none gives zeros; tokens behind
    the last sequence are not written. What the pages hold behind a sequence's last key does not matter; a value of a new token
    that is not finite may reach those in front of it as well. ``out [T, Hq, D]``, where given, is
    written and returned. A page that is not in the pools reads as zeros, keys behind the page table do not exist, and
    ``_lib.check_status`` raises for both. Head sizes 64 and 128 with pages of a power of two from 16 rows take the kernels.
    Inference only: a call with a gradient to record takes PyTorch's operations."""
    call, what = None, "paged_attention"
    if q.get_device() >= 0 and not _is_compiling():
        call = _lib.calls().attention(q, kpages, vpages, page_table, lens, cu)
        if call is not None and out is not None:
            H, D, st = call[4], call[6], out.stride()
            if out.shape != q.shape or out.dtype is not _BF16 or out.device != q.device or st[2] != 1 or st[1] != D or st[0] % 8 \
                    or st[0] < H * D or out.data_ptr() % 16 or (out.requires_grad and torch.is_grad_enabled()):
                call = None
    if call is None:
        if q.dim() != 3:
            raise ValueError(f"{what}: q is [tokens, heads, head size], not {list(q.shape)}")
        _check_batch(what, q, kpages, vpages, page_table, lens, cu)
        T, H, D = q.shape
        Hk = kpages.shape[2]
        if kpages.shape[3] != D or Hk < 1 or H < 1 or H % Hk:
            raise ValueError(f"{what}: {H} heads of {D} over pages of {Hk} heads of {kpages.shape[3]}")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
            raise ValueError(f"{what}: out is {list(q.shape)} of {q.dtype} on {q.device}, not {list(out.shape)} of {out.dtype} on {out.device}")
        if T == 0:
            return torch.empty_like(q) if out is None else out
    else:
        at, device, B, T, H, Hk, D, keys, packed = call
    if out is not None and (_ranges_overlap(out, q) or _ranges_overlap(out, kpages) or _ranges_overlap(out, vpages)):
        raise ValueError(f"{what}: out shares memory with q or the pages")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    elif not 2.0 ** -149 <= abs(scale := float(scale)) <= 2.0 ** 126:
        if not abs(scale) < 1.0:             # in units of log 2 it is no number of 32 bits
            raise ValueError(f"{what}: a scale of {scale}")
        scale = 0.0
    if call is None:
        return _attention_ref(q, kpages, vpages, page_table, lens, cu, scale, out)
    stream = _lib.stream_on(device)
    if stream is None:
        with torch.cuda.device(device):
            return paged_attention(q, kpages, vpages, page_table, lens, cu, scale, out)
    G = H // Hk
    groups = 1 if G <= 8 else 2 if G <= 16 and G % 2 == 0 else 0        # of heads that the decode kernel takes at a time; 0: not its
    one = cu is None and groups > 0
    x = q
    if not scale > 0 and not one:            # this kernel takes the largest score before it scales
        x, scale = (q * (-1 if scale < 0 else 0)).contiguous(), -scale if scale < 0 else 1.0
    elif not packed:
        x = q.clone(memory_format=torch.contiguous_format)
    if x is not q:
        at = _lib.calls().attention(x, kpages, vpages, page_table, lens, cu)[0]
    o = out if out is not None else torch.empty_like(x) if x.is_contiguous() else q.new_empty(T, H, D)
    parts, few, ws = 0, None, None
    if one or (cu is not None and B >= _MANY and groups):
        sms = _SMS.get(device) or _sm_count(q.device)
        parts = _decode_parts(B, Hk * groups, keys, D, sms, True) if one else _parts_beside(B * Hk * groups, sms)
        if parts != 1:
            few = torch.empty((B * parts if parts > 0 else -2 * parts) * H * (D + 2), dtype=torch.float32, device=q.device)
    if not one:
        nbytes = _attention_workspace(device, B, T, cu is None, parts != 0, keys, H, Hk, D)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _rc(_lib.calls().run_attention(at, o, scale, one, ws, parts, few, _lib.status_ptr(device), stream), "gf_paged_attn")
    if out is not None:
        _increment_version(out)
    return o
