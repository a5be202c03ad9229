"""The 4-bit cache in a Llama decode loop (``integration.PagedKV4Decoder``): the graph-replayed
tokens are the eager ones, and the logits follow a plain 32-bit model on the CPU that attends
over keys and values quantised by the definition (oracle/kv4.py).

Bound on the logits: a bf16 forward rounds each of about ten intermediates of a layer by at
most u = 2^-8 (u / sqrt(3) on average), sqrt(2 * 10) u / sqrt(3) ~ 0.010 over two layers; a
number whose rounding moved it across the middle of a step stores another code, which for the
few affected of 16 levels adds noise of the same size.  Three times their sum is 0.06."""
from __future__ import annotations

import pytest
import torch

from integration import PagedKV4Decoder, build_llama3_8b
from oracle import kv4 as ref
from transformers import LlamaConfig, LlamaForCausalLM

pytestmark = pytest.mark.gpu


def _tiny(dtype=torch.bfloat16):
    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, vocab_size=512, max_position_embeddings=256)
    return LlamaForCausalLM(cfg).to(dtype).cuda().eval()


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _plain_logits(model, ids, dtype):
    """fp32 CPU logits at every position of one sequence, keys and values through the 4-bit format."""
    m = model.float().cpu()
    core, cfg = m.model, m.config
    D, n_q, n_kv = core.layers[0].self_attn.head_dim, cfg.num_attention_heads, cfg.num_key_value_heads
    norm = lambda x, n: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + n.variance_epsilon) * n.weight  # noqa: E731
    x = core.embed_tokens(ids)
    cos, sin = core.rotary_emb(x[None], torch.arange(len(ids))[None])
    for layer in core.layers:
        a = layer.self_attn
        h = norm(x, layer.input_layernorm)
        q = _rotate(a.q_proj(h).view(-1, n_q, D), cos[0][:, None], sin[0][:, None])
        k = _rotate(a.k_proj(h).view(-1, n_kv, D), cos[0][:, None], sin[0][:, None])
        v = a.v_proj(h).view(-1, n_kv, D)
        k, v = (ref.values(*ref.quantise(t.to(dtype), D)) for t in (k, v))
        out, _ = ref.attention(q.double(), k, v, len(ids))
        x = x + a.o_proj(out.float().reshape(len(ids), -1))
        x = x + layer.mlp(norm(x, layer.post_attention_layernorm))
    return m.lm_head(norm(x, core.norm))


@torch.no_grad()
def test_logits_follow_the_plain_model_and_graph_equals_eager():
    model = _tiny()
    prompt = torch.randint(0, 512, (2, 37), generator=torch.Generator().manual_seed(1)).cuda()
    dec = PagedKV4Decoder(model, 2, 96, block_size=16)
    tokens = dec.generate(prompt, 12)
    logits = dec.forced_logits(prompt, tokens)
    assert torch.equal(logits.argmax(-1), tokens)
    assert torch.equal(dec.generate(prompt, 12), tokens)  # the cache and the plan start again
    got = logits.cpu()
    for b in range(2):
        ids = torch.cat([prompt[b], tokens[b]]).cpu()
        want = _plain_logits(model, ids, torch.bfloat16)[36:-1]
        assert (got[b] - want).norm() <= 0.06 * want.norm()


@torch.no_grad()
def test_llama_shaped_loop_is_the_eager_loop():
    model = build_llama3_8b(dtype=torch.bfloat16, device="cuda", num_hidden_layers=2)
    prompt = torch.randint(0, model.config.vocab_size, (3, 50), generator=torch.Generator().manual_seed(2)).cuda()
    dec = PagedKV4Decoder(model, 3, 128)
    tokens = dec.generate(prompt, 16)
    assert torch.equal(dec.forced_logits(prompt, tokens).argmax(-1), tokens)
    with pytest.raises(ValueError):
        dec.generate(prompt, 100)
