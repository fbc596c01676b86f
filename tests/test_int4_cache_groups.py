"""A 4-bit cache for a model whose decode steps could not read it is refused when it is made."""
import pytest
from transformers import Qwen3Config

from threadcut_b200 import kv
from threadcut_b200.attention import NAME


def config(heads, kv_heads, attention=NAME):
    cfg = Qwen3Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, head_dim=64)
    cfg._attn_implementation = attention
    return cfg


@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (64, 2)])
def test_more_than_16_query_heads_a_kv_head(heads, kv_heads):
    with pytest.raises(ValueError, match="16 query heads"):
        kv.new_cache(config(heads, kv_heads), paged=True, bits=4)
    try:
        kv.use_paged_cache(bits=4)
        with pytest.raises(ValueError, match="16 query heads"):
            kv.new_cache(config(heads, kv_heads))
    finally:
        kv.use_paged_cache(False)
    # other attentions read the rows back
    assert kv.new_cache(config(heads, kv_heads, "sdpa"), paged=True, bits=4).layers[0].state.bits == 4


@pytest.mark.parametrize("heads,kv_heads", [(16, 1), (32, 8), (4, 4)])
def test_as_many_as_there_may_be(heads, kv_heads):
    assert kv.new_cache(config(heads, kv_heads), paged=True, bits=4).layers[0].state.bits == 4
    assert kv.new_cache(config(34, 2), paged=True).layers[0].state.bits == 16
