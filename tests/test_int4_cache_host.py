"""The 4-bit cache's and weights' options, checked without a GPU."""
import pytest
import torch
from transformers import Qwen3Config, Qwen3ForCausalLM

from threadcut_b200 import kv, tp
from threadcut_b200.paged import PagedKVInt4


def config():
    return Qwen3Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
                       num_key_value_heads=1, head_dim=64)


@pytest.mark.parametrize("args", [dict(d=96), dict(dtype=torch.float32), dict(d=32)])
def test_rows_that_have_no_4_bit_form(args):
    with pytest.raises(ValueError, match="64, 128 or 256"):
        PagedKVInt4(1, 2, **(dict(d=128, max_tokens=10) | args))


def test_the_store_needs_a_gpu():
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVInt4(1, 2, 128, max_tokens=10, device="cpu")


def test_bits_of_a_new_cache():
    cfg = config()
    assert kv.new_cache(cfg, paged=True, bits=4).layers[0].state.bits == 4
    assert kv.new_cache(cfg, paged=True).layers[0].state.bits == 16
    assert isinstance(kv.new_cache(cfg, bits=16).layers[0], kv.GrowingLayer)
    for bad in (dict(bits=8, paged=True), dict(bits=4), dict(bits=4, paged=False)):
        with pytest.raises(ValueError, match="bits"):
            kv.new_cache(cfg, **bad)
    with pytest.raises(ValueError, match="bits"):
        kv.use_paged_cache(bits=5)
    try:
        kv.use_paged_cache(bits=4)
        assert kv.new_cache(cfg).layers[1].state.bits == 4
        assert kv.new_cache(cfg, bits=16).layers[1].state.bits == 16
        assert isinstance(kv.new_cache(cfg, paged=False).layers[0], kv.GrowingLayer)
    finally:
        kv.use_paged_cache(False)
    assert isinstance(kv.new_cache(cfg).layers[0], kv.GrowingLayer)


def test_bits_of_the_decoder_s_weights():
    model = Qwen3ForCausalLM(config()).eval()
    with pytest.raises(ValueError, match="bits"):
        tp.TPDecoder(model, "cpu", world=1, rank=0, weight_bits=8)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        tp.TPDecoder(model, "cpu", world=1, rank=0, weight_bits=4)
    dec = tp.TPDecoder(model.to(torch.bfloat16), "cpu", world=1, rank=0, weight_bits=4)
    assert (dec.lm_head.n, dec.lm_head.k) == (64, 64) and dec.layers_w[0].wqkv.n == 256 and not dec.use_peer_sums
