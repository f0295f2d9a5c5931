"""Speculative decoding refuses models and tokens that do not fit one another before anything is computed."""

from __future__ import annotations

import pytest


def _model(vocab: int):  # noqa: ANN202
    from transformers import LlamaConfig, LlamaForCausalLM

    return LlamaForCausalLM(LlamaConfig(hidden_size=16, intermediate_size=16, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1, head_dim=16,
                                        vocab_size=vocab))


@pytest.mark.parametrize("target,draft,first,message", [(32, 40, 1, "vocabularies"), (40, 32, 1, "vocabularies"), (32, 32, 32, "first_token"), (32, 32, -1, "first_token")])
def test_tokens_that_one_of_the_models_does_not_know(target: int, draft: int, first: int, message: str) -> None:
    """A token past an embedding's end would be read out of range on the device."""
    from lazykv_b200.cache import FullGPUCache
    from lazykv_b200.generate import speculative_decode

    caches = [FullGPUCache(1, 16) for _ in range(2)]
    with pytest.raises(ValueError, match=message):
        speculative_decode(_model(target), caches[0], _model(draft), caches[1], first, 4, 2)
    assert all(c.get_seq_length() == 0 for c in caches)


def test_one_cache_for_both_models() -> None:
    from lazykv_b200.cache import FullGPUCache
    from lazykv_b200.generate import speculative_decode

    cache, model = FullGPUCache(1, 16), _model(32)
    with pytest.raises(ValueError, match="a cache each"):
        speculative_decode(model, cache, model, cache, 1, 4, 2)
    assert cache.get_seq_length() == 0
