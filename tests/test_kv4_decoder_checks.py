"""``PagedKV4Decoder`` refuses what it does not compute, before any kernel runs.  CPU only."""
from __future__ import annotations

import pytest
import torch

from integration import PagedKV4Decoder
from transformers import LlamaConfig, LlamaForCausalLM


def _model(**kw):
    return LlamaForCausalLM(LlamaConfig(hidden_size=128, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
                                        num_key_value_heads=1, head_dim=64, vocab_size=32, **kw)).to(torch.bfloat16)


@pytest.mark.parametrize("only", ["q_proj", "k_proj", "v_proj"])
def test_attention_bias_is_refused(only):
    model = _model(attention_bias=True)
    for layer in model.model.layers:
        for name in ("q_proj", "k_proj", "v_proj"):
            if name != only:
                getattr(layer.self_attn, name).bias = None
    with pytest.raises(ValueError, match="bias"):
        PagedKV4Decoder(model, 1, 32)


def test_sequences_past_the_cache_are_refused():
    """Teacher forcing appends the prompt and all forced tokens but the last."""
    dec = object.__new__(PagedKV4Decoder)
    dec.batch, dec.max_len = 2, 16
    ids = torch.zeros(2, 12, dtype=torch.long)
    for prompt, tokens in ((ids, ids[:, :6]), (ids[:1], ids[:1, :2]), (ids, ids[:1, :2]), (ids[:, :0], ids[:, :2]),
                           (ids, ids[:, :0])):
        with pytest.raises(ValueError):
            dec.forced_logits(prompt, tokens)
    for prompt, n_new in ((ids, 5), (ids[:1], 1), (ids[:, :0], 3), (ids, 0)):
        with pytest.raises(ValueError):
            dec.generate(prompt, n_new)
