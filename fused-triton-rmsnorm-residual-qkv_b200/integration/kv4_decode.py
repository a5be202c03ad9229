"""Greedy decoding with the paged 4-bit key/value cache, each step replayed from a CUDA graph.

The decoder layer's attention half is four calls of the package: residual add + RMSNorm +
Q/K/V projection with the rotary embedding (one launch at decode sizes), keys and values
quantised into their slots, and attention over the 4-bit codes; the block tables, positions
and slots of the step come from one launch shared by all layers.  Nothing in a step is read
back by the host, so after the prompt one step is captured and replayed, as
``GraphedGreedyDecoder`` does with transformers' 16-bit static cache (the reference's
end-to-end benchmark decodes with transformers' cache too, ``benchmarks/e2e_decode.py:60-148``).
"""
from __future__ import annotations

import torch

from triton_fused_rmsnorm_qkv import fused_add_rmsnorm_qkv_rope, kv4_append, kv4_attention, kv4_cache, kv4_plan

from .llama3_patch import pack_qkv_weight


class PagedKV4Decoder:
    """Greedy decoder for an unpatched ``LlamaForCausalLM`` (head_dim 64 or 128, no attention
    bias) whose cache holds ``max_len`` tokens for each of ``batch`` requests, in blocks of
    ``block_size`` tokens with ``group_size`` dims per scale."""

    def __init__(self, model, batch: int, max_len: int, *, block_size: int = 64, group_size: int | None = None):
        cfg, core = model.config, model.model
        self.model, self.batch, self.max_len = model, batch, max_len
        self.device = next(model.parameters()).device
        self.n_q, self.n_kv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim = core.layers[0].self_attn.head_dim
        self.block_size = block_size
        if any(getattr(layer.self_attn, name).bias is not None for layer in core.layers
               for name in ("q_proj", "k_proj", "v_proj")):
            raise ValueError("the fused projection has no bias: the model's q_proj, k_proj and v_proj must not have one")
        self.qkv_weights = [pack_qkv_weight(layer.self_attn) for layer in core.layers]
        self.width = -(-max_len // block_size)
        dtype = self.qkv_weights[0].dtype
        self.caches = [kv4_cache(batch * self.width, self.n_kv, self.head_dim, block_size=block_size,
                                 group_size=group_size, dtype=dtype, device=self.device) for _ in core.layers]
        self._reset()

    def _reset(self):
        n, dev = self.batch * self.width, self.device
        self.tables = torch.full((self.batch, self.width), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(n, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), n, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.batch, dtype=torch.int32, device=dev)
        self.ones = torch.ones(self.batch, dtype=torch.int32, device=dev)

    @torch.no_grad()
    def _forward(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits of the last of ``ids`` (batch, S) tokens, which join the cache."""
        B, S = ids.shape
        core = self.model.model
        plan = kv4_plan(self.lens, self.ones if S == 1 else torch.full_like(self.lens, S), self.tables, self.free,
                        self.n_free, block_size=self.block_size, n_tokens=B * S)
        plan.context_after(self.lens, out=self.lens)
        self.n_free.copy_(plan.n_free)
        x, residual = core.embed_tokens(ids), None
        cos, sin = core.rotary_emb(x, plan.positions.view(B, S).long())
        for layer, weight, cache in zip(core.layers, self.qkv_weights, self.caches):
            norm = layer.input_layernorm
            q, k, v, hidden = fused_add_rmsnorm_qkv_rope(x, residual, norm.weight, weight, cos, sin, self.n_q, self.n_kv,
                                                         self.head_dim, norm.variance_epsilon)
            kv4_append(cache, k, v, plan.slots)
            out = kv4_attention(q, cache, self.tables, plan.seq_lens, scale=layer.self_attn.scaling)
            residual = hidden + layer.self_attn.o_proj(out.reshape(B, S, -1))
            x = layer.mlp(layer.post_attention_layernorm(residual))
        return self.model.lm_head(core.norm((x + residual)[:, -1:]))[:, 0]

    def _check(self, prompt: torch.Tensor, room: int, wanted: int) -> None:
        """The prompt and ``room`` tokens after it must fit, and something must be asked for."""
        B, P = prompt.shape
        if B != self.batch or P == 0 or wanted <= 0 or P + room > self.max_len:
            raise ValueError(f"prompt {tuple(prompt.shape)} + {room} tokens does not fit batch {self.batch}, "
                             f"max_len {self.max_len}")

    @torch.no_grad()
    def forced_logits(self, prompt: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """Teacher forcing, eagerly: the fp32 logits that predict ``tokens[:, t]`` for every t."""
        self._check(prompt, tokens.shape[1] - 1, tokens.shape[1])
        if tokens.shape[0] != self.batch:
            raise ValueError(f"tokens {tuple(tokens.shape)} do not follow {self.batch} prompts")
        self._reset()
        logits = [self._forward(prompt).float()]
        for t in range(tokens.shape[1] - 1):
            logits.append(self._forward(tokens[:, t:t + 1]).float())
        return torch.stack(logits, dim=1)

    @torch.no_grad()
    def generate(self, prompt: torch.Tensor, n_new: int) -> torch.Tensor:
        """The ``n_new`` greedy tokens after ``prompt`` (batch, P): the prompt and the first step
        run eagerly, every later step is a replay of one captured graph."""
        self._check(prompt, n_new, n_new)
        self._reset()
        tok = self._forward(prompt).argmax(-1, keepdim=True)
        tokens = [tok.clone()]
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))

        def step():
            tok.copy_(self._forward(tok).argmax(-1, keepdim=True))

        with torch.cuda.stream(side):
            if n_new > 1:
                step()
        torch.cuda.current_stream(self.device).wait_stream(side)
        if n_new > 1:
            tokens.append(tok.clone())
        if n_new > 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            for _ in range(n_new - 2):
                graph.replay()
                tokens.append(tok.clone())
            torch.cuda.synchronize(self.device)
        return torch.cat(tokens, dim=1)
