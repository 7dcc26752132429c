"""Serving loop of a patched Llama over the paged cache: prompts of different
lengths are packed into one prefill, decode steps take one token of every
running sequence, and sequences can be forked, freed and compacted in between.

    model = patch_llama_model(model, variant="V3", swiglu=True)
    server = PagedLlama(model, num_pages=4096)
    seqs, logits = server.prefill([[1, 2, 3], [4, 5]])
    logits = server.decode(seqs, logits.argmax(-1).tolist())
    print(server.generate([[1, 2, 3]], max_new_tokens=16))

Per layer: the fused RMSNorm -> QKV launch, rotary embedding, kv_cache_append,
gqa_prompt_attention (prefill) or gqa_paged_decode, the output projection, and
the fused RMSNorm -> gate/up -> SwiGLU launch with the down projection.
"""

from __future__ import annotations

import torch
from transformers.models.llama.modeling_llama import apply_rotary_pos_emb

from src.paged_kv_cache import PagedKVCache, Step


class PagedLlama:
    """A Llama patched with ``patch_llama_model(..., swiglu=True)`` (bf16 or
    fp16, head_dim 64 or 128) and its cache."""

    def __init__(self, model, num_pages: int, page_size: int = 16):
        first = model.model.layers[0]
        if not hasattr(first.self_attn, "fused_qkv") or not hasattr(first.mlp,
                                                                    "fused_gate_up_swiglu"):
            raise ValueError("PagedLlama needs a model patched with patch_llama_model(..., "
                             "swiglu=True)")
        config = model.config
        self.model = model
        self.heads = config.num_attention_heads
        self.kv_heads = config.num_key_value_heads
        self.head_dim = first.self_attn.head_dim
        weight = model.model.embed_tokens.weight
        self.cache = PagedKVCache(len(model.model.layers), num_pages, page_size, self.kv_heads,
                                  self.head_dim, weight.dtype, weight.device)

    @torch.no_grad()
    def _forward(self, step: Step, tokens: list[int], prompt: bool) -> torch.Tensor:
        """Logits of every sequence's last new token."""
        model, cache = self.model.model, self.cache
        ids = torch.tensor(tokens, device=cache.device)
        x = model.embed_tokens(ids)
        cos, sin = model.rotary_emb(x[None], step.positions[None].long())
        for i, layer in enumerate(model.layers):
            attn = layer.self_attn
            q, k, v = attn.fused_qkv(x)
            q = q.view(1, -1, self.heads, self.head_dim)
            k = k.view(1, -1, self.kv_heads, self.head_dim)
            v = v.view(-1, self.kv_heads, self.head_dim)
            q, k = apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim=2)
            q, k = q[0], k[0]
            cache.write(i, step, k, v)
            if prompt:
                out = cache.prompt_attention(step, q, k, v, attn.scaling)
            else:
                out = cache.decode_attention(i, step, q, attn.scaling)
            x = x + attn.o_proj(out.flatten(1))
            x = x + layer.mlp.down_proj(layer.mlp.fused_gate_up_swiglu(x))
        last = step.cu_seqlens[1:].long() - 1
        return self.model.lm_head(model.norm(x[last]))

    def prefill(self, prompts: list[list[int]]) -> tuple[list[int], torch.Tensor]:
        """New sequences with these tokens; their numbers, and logits [batch, vocab]."""
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a prompt must have at least one token")
        seqs = [self.cache.new_sequence() for _ in prompts]
        try:
            step = self.cache.extend(seqs, [len(p) for p in prompts])
            return seqs, self._forward(step, [t for p in prompts for t in p], True)
        except Exception:
            for s in seqs:
                self.cache.free(s)
            raise

    def decode(self, seqs: list[int], tokens: list[int]) -> torch.Tensor:
        """One more token of each sequence; logits [batch, vocab].  Where this fails the
        sequences are as before, and the call can be made again."""
        if len(tokens) != len(seqs):
            raise ValueError("decode: one token a sequence")
        step = self.cache.extend(seqs, [1] * len(seqs))
        try:
            return self._forward(step, tokens, False)
        except Exception:
            self.cache.withdraw(seqs, [1] * len(seqs))
            raise

    def generate(self, prompts: list[list[int]], max_new_tokens: int) -> list[list[int]]:
        """Greedy continuations; the sequences are freed afterwards, also where a step fails."""
        seqs, logits = self.prefill(prompts)
        out: list[list[int]] = [[] for _ in prompts]
        try:
            for n in range(max_new_tokens):
                tokens = logits.argmax(-1).tolist()
                for o, t in zip(out, tokens):
                    o.append(t)
                if n + 1 < max_new_tokens:
                    logits = self.decode(seqs, tokens)
        finally:
            for s in seqs:
                self.cache.free(s)
        return out
