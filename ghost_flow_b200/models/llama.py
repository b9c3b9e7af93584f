"""LLaMA-family decoder as ``nn.Module`` (autograd path; the hand-scheduled ZeRO-3 engine in
``parallel/zero3.py`` runs the same math with explicit kernels).

Class and preset names follow ghostflow-nn/src/llama.rs:37-552 (``LLaMAConfig``, ``RMSNorm``, ``RotaryEmbedding``,
``SwiGLU``, ``LLaMAAttention``, ``LLaMADecoderLayer``, ``LLaMAModel``, ``LLaMAForCausalLM.forward/generate``).
Deviations from the reference, on purpose: real causal attention with K and V (its attention is a
placeholder that drops them, llama.rs:319-331), grouped-query attention, no biases, a KV cache in
``generate`` (its doc promises one, the code re-runs the whole prefix), N(0, 0.02) initialisation.
"""
from __future__ import annotations

import torch

from .. import ops
from ..ops import raw
from ..nn.layers import Embedding, Linear, RMSNorm, SwiGLU
from ..nn.module import Module, ModuleList, plain_modules
from .configs import LLaMAConfig
from .paged import PagedKVCache


class LLaMAAttention(Module):
    def __init__(self, cfg: LLaMAConfig, device=None, dtype=None):
        super().__init__()
        self.cfg = cfg
        hd = cfg.head_dim
        self.wqkv = Linear(cfg.hidden_size, (cfg.num_attention_heads + 2 * cfg.num_key_value_heads) * hd, False,
                           device, dtype)
        self.wo = Linear(cfg.num_attention_heads * hd, cfg.hidden_size, False, device, dtype)
        if cfg.qk_norm:
            self.q_norm = RMSNorm(hd, cfg.rms_norm_eps, device, dtype)
            self.k_norm = RMSNorm(hd, cfg.rms_norm_eps, device, dtype)

    def _weights(self):
        """Weights of the heads' norms, if there are any."""
        return (self.q_norm.weight, self.k_norm.weight) if self.cfg.qk_norm else (None, None)

    def _heads(self, qkv, cos, sin, start_pos):
        c = self.cfg
        H, Hk = c.num_attention_heads, c.num_key_value_heads
        if c.plain_heads:
            return ops.rope_qkv(qkv, H, Hk, cos, sin, c.rope_interleaved, start_pos)
        return ops.norm_rope_qkv(qkv, H, Hk, *self._weights(), cos, sin, c.rms_norm_eps, c.rope_interleaved, start_pos)

    def _heads_to_cache(self, qkv, cos, sin, kc, vc, start_pos):
        c = self.cfg
        if c.plain_heads:
            return ops.rope_qkv_to_cache(qkv, c.num_attention_heads, c.num_key_value_heads, cos, sin, kc, vc, c.rope_interleaved, start_pos)
        q, k, v = self._heads(qkv, cos, sin, start_pos)
        kc[:, start_pos:start_pos + q.shape[1]] = k
        vc[:, start_pos:start_pos + q.shape[1]] = v
        return q

    def forward(self, x, cos, sin, residual=None, cache=None, start_pos: int = 0):
        c = self.cfg
        B, S, _ = x.shape
        H, Hk, D = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        qkv = self.wqkv(x).view(B, S, H + 2 * Hk, D)
        if cache is not None:
            # decoding: append to the cache and attend over everything seen so far
            kc, vc = cache
            kernels = x.is_cuda and x.dtype == torch.bfloat16 and D in (64, 128) and not torch.is_grad_enabled()
            if kernels and start_pos == 0 and S > 1:
                # prompt: nothing older than itself to attend to
                q, k, v = self._heads(qkv, cos, sin, start_pos)
                kc[:, :S] = k
                vc[:, :S] = v
                o = ops.flash_attention(q, k, v, causal=True)
            elif kernels and S == 1:
                q = self._heads_to_cache(qkv, cos, sin, kc, vc, start_pos)
                # one new token per sequence: the decode kernel streams the cache once (GQA groups share the reads)
                o = raw.attn_decode(q.reshape(B, H * D), kc.view(B, kc.shape[1], Hk * D), vc.view(B, vc.shape[1], Hk * D),
                                    start_pos + 1, B, H, Hk, D).view(B, 1, H, D)
            else:
                q = self._heads_to_cache(qkv, cos, sin, kc, vc, start_pos)
                kk, vv = kc[:, :start_pos + S], vc[:, :start_pos + S]
                G = H // Hk
                qf = q.transpose(1, 2).float()
                kf = kk.transpose(1, 2).float().repeat_interleave(G, 1)
                vf = vv.transpose(1, 2).float().repeat_interleave(G, 1)
                s = qf @ kf.transpose(-1, -2) / (D ** 0.5)
                T = start_pos + S
                mask = torch.ones(S, T, dtype=torch.bool, device=x.device).tril(T - S)
                s = s.masked_fill(~mask, float("-inf"))
                o = (torch.softmax(s, -1) @ vf).transpose(1, 2).to(x.dtype)
        else:
            q, k, v = self._heads(qkv, cos, sin, start_pos)
            o = ops.flash_attention(q, k, v, causal=True)
        return self.wo(o.reshape(B, S, H * D), residual)

    def forward_pages(self, x, cos, sin, pools, batch, residual=None):
        """New tokens ``[T, hidden]`` of the sequences of a :class:`~.paged.PagedBatch`, whose keys are in this layer's ``pools``."""
        c = self.cfg
        H, Hk, D = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        qkv = self.wqkv(x).view(x.shape[0], H + 2 * Hk, D)
        k, v, *scales = pools
        scales = dict(zip(("kscales", "vscales"), scales))
        norms = dict(q_weight=self.q_norm.weight, k_weight=self.k_norm.weight, eps=c.rms_norm_eps) if c.qk_norm else {}
        q = ops.rope_qkv_to_pages(qkv, H, Hk, cos, sin, k, v, batch.table, batch.lens, batch.cu, c.rope_interleaved, **scales, **norms)
        o = ops.paged_attention(q, k, v, batch.table, batch.lens, batch.cu, **scales)
        return self.wo(o.reshape(x.shape[0], H * D), residual)


def _weight(module):
    """A module's weight: its parameter without the search of an attribute, or what else bears the name."""
    p = module._parameters.get("weight")
    return module.weight if p is None else p


class LLaMADecoderLayer(Module):
    def __init__(self, cfg: LLaMAConfig, device=None, dtype=None):
        super().__init__()
        self.attn_norm = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps, device, dtype)
        self.attn = LLaMAAttention(cfg, device, dtype)
        self.ffn_norm = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps, device, dtype)
        self.mlp = SwiGLU(cfg.hidden_size, cfg.intermediate_size, False, device, dtype)

    def _decodes_in_one_call(self, x, cos, sin, cache, start_pos):
        """The operands of :func:`ops.raw.llama_decode_layer`, or ``None`` where the layer runs module by module: more than one
        token, a gradient, other types or layouts, modules that were replaced or carry hooks, and calls that something
        follows (tracing, transforms, modes), which would miss what happens inside."""
        if x.dim() != 3 or x.shape[1] != 1 or x.dtype is not torch.bfloat16 or not x.is_cuda or torch.is_grad_enabled() \
                or type(x) is not torch.Tensor or not 0 < x.shape[0] <= 64 or not isinstance(start_pos, int) \
                or ops.observed():            # before anything asks a tensor for its memory: transformed ones have none
            return None
        m = self._modules                    # a plain callable that stands for a module is not in here
        an, at, fn, mlp = m.get("attn_norm"), m.get("attn"), m.get("ffn_norm"), m.get("mlp")
        if not (type(an) is RMSNorm and type(at) is LLaMAAttention and type(fn) is RMSNorm and type(mlp) is SwiGLU):
            return None
        lin = at._modules.get("wqkv"), at._modules.get("wo"), mlp._modules.get("gate_up"), mlp._modules.get("down")
        for n in lin:
            if type(n) is not Linear or n.bias is not None:
                return None
        if not plain_modules(an, at, fn, mlp, *lin):
            return None
        c, (kc, vc), (B, _, hidden), dev = at.cfg, cache, x.shape, x.device
        if not c.plain_heads:
            return None
        H, Hk, D = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        w = [_weight(n) for n in (an, lin[0], lin[1], fn, lin[2], lin[3])]
        inner = w[5].shape[1] if w[5].dim() == 2 else 0
        shapes = (hidden,), ((H + 2 * Hk) * D, hidden), (hidden, H * D), (hidden,), (2 * inner, hidden), (hidden, inner)
        if D not in (64, 128) or H % Hk or H // Hk > 8 or hidden % 8 or inner % 8 or inner == 0:
            return None
        for p, s in zip(w, shapes):
            if p.shape != s or p.dtype is not torch.bfloat16 or p.device != dev or not p.is_contiguous() or p.data_ptr() & 15 \
                    or type(p) not in (torch.Tensor, torch.nn.Parameter):
                return None
        if dev.index != torch.cuda.current_device() or not (x.is_contiguous() and x.data_ptr() & 15 == 0) \
                or not ops.decode_cache_ok(kc, vc, cos, sin, (B, Hk, D), dev, start_pos):
            return None
        return (x, w[0], an.eps, w[1], w[2], w[3], fn.eps, w[4], w[5], cos, sin, kc, vc, H, Hk, D,
                c.rope_interleaved, start_pos)

    def forward(self, x, cos, sin, cache=None, start_pos: int = 0):
        if cache is not None:
            args = self._decodes_in_one_call(x, cos, sin, cache, start_pos)
            if args is not None:
                y = raw.llama_decode_layer(*args)
                torch.autograd.graph.increment_version(cache)     # a graph that saved a cache has to notice the write
                return y
        x = self.attn(self.attn_norm(x), cos, sin, residual=x, cache=cache, start_pos=start_pos)
        return self.mlp(self.ffn_norm(x), residual=x)

    def forward_pages(self, x, cos, sin, pools, batch):
        x = self.attn.forward_pages(self.attn_norm(x), cos, sin, pools, batch, residual=x)
        return self.mlp(self.ffn_norm(x), residual=x)


class LLaMAModel(Module):
    def __init__(self, cfg: LLaMAConfig, device=None, dtype=None):
        super().__init__()
        self.cfg = cfg
        self.embed_tokens = Embedding(cfg.vocab_size, cfg.hidden_size, device=device, dtype=dtype)
        self.layers = ModuleList([LLaMADecoderLayer(cfg, device, dtype) for _ in range(cfg.num_hidden_layers)])
        self.norm = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps, device, dtype)
        self._rope = None

    def rope(self, length, device):
        if self._rope is None or self._rope[0].shape[0] < length or self._rope[0].device != torch.device(device):
            n = max(length, self.cfg.max_position_embeddings)
            self._rope = ops.rope_tables(n, self.cfg.rope_dims, self.cfg.rope_theta, device)
        return self._rope

    def _before_norm(self, ids, caches, start_pos):
        S = ids.shape[1]
        cos, sin = self.rope(start_pos + S, ids.device)
        x = self.embed_tokens(ids)
        for i, layer in enumerate(self.layers):
            x = layer(x, cos, sin, None if caches is None else caches[i], start_pos)
        return x

    def forward(self, ids, caches=None, start_pos: int = 0):
        return self.norm(self._before_norm(ids, caches, start_pos))

    def forward_pages(self, ids, cache, batch, rows=None):
        """Hidden states of the new tokens ``ids [T]`` of a batch over a :class:`~.paged.PagedKVCache`, or of those in ``rows`` (indices)."""
        cos, sin = self.rope(batch.longest, ids.device)
        x = self.embed_tokens(ids)
        for layer, pools in zip(self.layers, cache.pools):
            x = layer.forward_pages(x, cos, sin, pools, batch)
        if rows is not None:
            x = x[rows]
        return self.norm(x) if x.shape[0] else x


class LLaMAForCausalLM(Module):
    def __init__(self, cfg: LLaMAConfig, device=None, dtype=None):
        super().__init__()
        self.cfg = cfg
        self.model = LLaMAModel(cfg, device, dtype)
        self.lm_head = Linear(cfg.hidden_size, cfg.vocab_size, False, device, dtype)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self):
        std = self.cfg.initializer_range
        for name, p in self.named_parameters():
            if name.endswith("norm.weight"):
                p.fill_(1.0)
            else:
                p.normal_(0.0, std)
        if self.cfg.tie_word_embeddings:
            self.lm_head.weight = self.model.embed_tokens.weight

    def _norm_in_the_head(self, ids) -> bool:
        """Whether the last norm can run inside the head's product: one token of at most 16 sequences, no gradient, modules that do
        nothing but their own forward, dense bf16 weights on the current GPU, and nothing that follows the calls."""
        model, head = self._modules.get("model"), self._modules.get("lm_head")
        if type(ids) is not torch.Tensor or not ids.is_cuda or ids.dim() != 2 or ids.shape[1] != 1 or not 0 < ids.shape[0] <= 16 \
                or torch.is_grad_enabled() or ops.observed() or type(model) is not LLaMAModel or type(head) is not Linear \
                or head.bias is not None:
            return False
        norm, w = model._modules.get("norm"), head.weight
        if type(norm) is not RMSNorm or not plain_modules(model, norm, head) or ids.device.index != torch.cuda.current_device():
            return False
        for p, s in ((norm.weight, (self.cfg.hidden_size,)), (w, (w.shape[0], self.cfg.hidden_size))):
            if type(p) not in (torch.Tensor, torch.nn.Parameter) or p.shape != s or p.dtype is not torch.bfloat16 \
                    or p.device != ids.device or not p.is_contiguous() or p.data_ptr() & 15:
                return False
        return self.cfg.hidden_size % 8 == 0

    def forward(self, ids, labels=None, caches=None, start_pos: int = 0):
        if labels is None and caches is not None and self._norm_in_the_head(ids):
            x = self.model._before_norm(ids, caches, start_pos)
            if x.dtype is torch.bfloat16 and x.is_contiguous() and not x.data_ptr() & 15:
                norm, w = self.model.norm, self.lm_head.weight
                y = raw.rmsnorm_gemm(x.view(x.shape[0], -1), norm.weight, norm.eps, w)
                return y.unsqueeze(1)
            return self.lm_head(self.model.norm(x))
        h = self.model(ids, caches, start_pos)
        logits = self.lm_head(h)
        if labels is None:
            return logits
        return ops.cross_entropy(logits.view(-1, logits.shape[-1]), labels.reshape(-1)), logits

    @torch.no_grad()
    def forward_pages(self, ids, cache, batch, rows=None):
        """Logits ``[T, vocab]`` of new tokens ``ids [T]`` of the sequences of ``batch``, one behind the other, over a
        :class:`~.paged.PagedKVCache`, or of those in ``rows``. Inference only."""
        h = self.model.forward_pages(ids, cache, batch, rows)
        return self.lm_head(h) if h.shape[0] else h.new_empty(0, self.lm_head.weight.shape[0])

    def new_paged_cache(self, num_pages: int, page_size: int = 64, device=None, dtype=None):
        c, p = self.cfg, next(self.parameters())
        return PagedKVCache(c.num_hidden_layers, num_pages, page_size, c.num_key_value_heads, c.head_dim, device or p.device,
                            dtype or p.dtype)

    def new_caches(self, batch: int, max_len: int, device=None, dtype=None):
        c = self.cfg
        p = next(self.parameters())
        shape = (batch, max_len, c.num_key_value_heads, c.head_dim)
        return [(torch.zeros(shape, device=device or p.device, dtype=dtype or p.dtype),
                 torch.zeros(shape, device=device or p.device, dtype=dtype or p.dtype))
                for _ in range(c.num_hidden_layers)]

    @torch.no_grad()
    def generate(self, ids, max_new_tokens: int, temperature: float = 0.0, **choice):
        """Greedy (temperature 0) or sampled continuation with a KV cache. ``choice``: penalties, bias, mask, top-k, top-p and min-p of
        :func:`~ghost_flow_b200.ops.sampling.next_tokens`."""
        B, S = ids.shape
        caches = self.new_caches(B, S + max_new_tokens)
        logits = self.forward(ids, caches=caches, start_pos=0)[:, -1]
        out, counted = [ids], ops.sampling.counts_tokens(choice)
        pos = S
        for _ in range(max_new_tokens):
            nxt = ops.next_tokens(logits, temperature, torch.cat(out, 1) if counted else None, prompt=S, **choice)
            out.append(nxt)
            logits = self.forward(nxt, caches=caches, start_pos=pos)[:, -1]
            pos += 1
        return torch.cat(out, dim=1)

    @torch.no_grad()
    def generate_batch(self, prompts, max_new_tokens: int, temperature: float = 0.0, page_size: int = 64, chunk_tokens: int = 4096,
                       cache_dtype=None, **choice):
        """Continuations of prompts (1-D token tensors) of any lengths in one batch over a paged cache; a list of prompts with their
        ``max_new_tokens`` new tokens. Prompts go through the model at most ``chunk_tokens`` tokens at a time. ``cache_dtype``: of the cache, the
        model's or ``torch.float8_e4m3fn``. ``choice`` as for :meth:`generate`."""
        p = next(self.parameters())
        prompts = [t.to(p.device).long().reshape(-1) for t in prompts]
        if not prompts or max_new_tokens <= 0:
            return prompts
        if any(t.numel() == 0 for t in prompts) or chunk_tokens < 1:
            raise ValueError("generate_batch continues prompts of one token or more, in chunks of one or more")
        B, lens = len(prompts), [t.numel() for t in prompts]
        cache = self.new_paged_cache(sum(-(-(n + max_new_tokens) // page_size) for n in lens), page_size, dtype=cache_dtype)
        for b, n in enumerate(lens):
            cache.reserve(b, n + max_new_tokens)
        # the prompts, in chunks: logits are wanted of their last tokens only
        done, logits = [0] * B, [None] * B
        while done != lens:
            room, take = chunk_tokens, {}
            for b in range(B):
                n = min(room, lens[b] - done[b])
                if n > 0:
                    take[b] = n
                    room -= n
            batch = cache.batch(take, [done[b] + n for b, n in take.items()], take.values())
            ids = torch.cat([prompts[b][done[b]:done[b] + n] for b, n in take.items()])
            ends, at = {}, 0
            for b, n in take.items():
                at += n
                done[b] += n
                if done[b] == lens[b]:
                    ends[b] = at - 1
            out = self.forward_pages(ids, cache, batch, torch.tensor(list(ends.values()), dtype=torch.long, device=p.device))
            for row, b in zip(out, ends):
                logits[b] = row
        logits = torch.stack(logits)
        # then all sequences, token by token; what is appended is told to the device by the lengths it holds
        tokens = torch.zeros(B, max(lens) + max_new_tokens, dtype=torch.long, device=p.device)
        for b, t in enumerate(prompts):
            tokens[b, :lens[b]] = t
        count = torch.tensor(lens, dtype=torch.int32, device=p.device)
        first = count.clone()
        batch, counted = cache.batch(range(B), [n + 1 for n in lens]), ops.sampling.counts_tokens(choice)
        for i in range(max_new_tokens):
            nxt = ops.next_tokens(logits, temperature, tokens if counted else None, count, first, **choice)
            tokens.scatter_(1, count.long()[:, None], nxt)
            count += 1
            if i + 1 < max_new_tokens:
                logits = self.forward_pages(nxt.view(-1), cache, batch)
                batch.advance()
        return [tokens[b, :n + max_new_tokens] for b, n in enumerate(lens)]

    # names used by the ZeRO engine's state_dict
    def load_engine_state(self, sd: dict):
        """Loads the flat-unit names of ``Zero3LlamaEngine.state_dict()``."""
        own = self.state_dict()
        own["model.embed_tokens.weight"].copy_(sd["embed_tokens.weight"])
        own["model.norm.weight"].copy_(sd["norm.weight"])
        own["lm_head.weight"].copy_(sd["lm_head.weight"])
        for i in range(self.cfg.num_hidden_layers):
            pre = f"model.layers.{i}."
            own[pre + "attn_norm.weight"].copy_(sd[f"layers.{i}.attn_norm"])
            own[pre + "attn.wqkv.weight"].copy_(sd[f"layers.{i}.wqkv"])
            own[pre + "attn.wo.weight"].copy_(sd[f"layers.{i}.wo"])
            own[pre + "ffn_norm.weight"].copy_(sd[f"layers.{i}.ffn_norm"])
            own[pre + "mlp.gate_up.weight"].copy_(sd[f"layers.{i}.w_gate_up"])
            own[pre + "mlp.down.weight"].copy_(sd[f"layers.{i}.w_down"])
