"""The fused step with 4-bit weights: captured, on a stream of its own, and over a 4-bit cache whose pool is full."""
import pytest
import torch
from transformers import AutoModelForCausalLM, Qwen3Config

from threadcut_b200 import _lib, int4, tp
from threadcut_b200 import attention as tc_attention
from threadcut_b200 import kv as tc_kv
from threadcut_b200.match import Split

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def tiny(dtype=BF):
    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=520, hidden_size=256, intermediate_size=544, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=8192)
    return AutoModelForCausalLM.from_config(cfg, dtype=dtype, attn_implementation=tc_attention.NAME).to(DEV).eval()


@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("n", [1, 2048])
def test_a_captured_step_is_the_eager_one(dtype, n):
    model = tiny(dtype)
    gen = torch.Generator(device=DEV).manual_seed(1)
    with torch.no_grad():
        dec = tp.TPDecoder(model, DEV, world=1, rank=0, weight_bits=4)
        for i in range(2):
            dec.load(i, *(torch.randn(1, 2, n, 128, generator=gen, device=DEV).to(dtype) for _ in range(2)))
        token = torch.tensor([7], device=DEV)
        graph, out = dec.capture(token, n)
        for t in (7, 100, 519):
            token.fill_(t)
            graph.replay()
            torch.cuda.synchronize()
            got = int(out)
            dec.crop(n)
            logits = dec.logits(token, n)
            assert torch.isfinite(logits).all() and got == int(logits.argmax())
            dec.crop(n)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                other = dec.logits(token, n)
            s.synchronize()
            assert torch.equal(other, logits)
            dec.crop(n)
        del graph


def test_a_step_over_a_full_pool_packs_it_first():
    model = tiny()
    inv = model.model.rotary_emb.inv_freq
    ids = torch.randint(0, 520, (1, 60), generator=torch.Generator().manual_seed(4)).to(DEV)
    caches = [tc_kv.new_cache(model.config, paged=True, max_tokens=m, page_rows=32, bits=4) for m in (64, 6400)]
    k = torch.randn(1, 2, 33, 128, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    with torch.no_grad():
        for cache in caches:
            model(input_ids=ids[:, :40], past_key_values=cache, use_cache=True)
        small = caches[0].layers[0].state.kv
        packed = []
        compact = small.compact
        small.compact = lambda: (packed.append(1), compact())
        dec = tp.accelerate(model, weight_bits=4)
        try:
            while len(small.table.free) > 1:  # spans that leave a page with a row or two, until no page is free
                for cache in caches:
                    for layer in cache.layers:
                        layer.update(k, k)
                    n = cache.get_seq_length()
                    tc_kv.splice(cache, Split(n - 33, n - 2, 2), inv)
            while small.table.free or small.table.runs[-1][1] + small.table.runs[-1][2] < 32:
                for cache in caches:
                    for layer in cache.layers:
                        layer.update(k[:, :, :1], k[:, :, :1])
            for layer in caches[0].layers + caches[1].layers:
                layer._flush()
            assert not packed and tp._fusable(caches[0], dec)
            n = caches[0].get_seq_length()
            a, b = (model(input_ids=ids[:, 40:41], past_key_values=c, use_cache=True).logits.float().flatten() for c in caches)
            assert packed == [1] and caches[0].get_seq_length() == n + 1
            for layer in range(2):
                for x, y in zip(small.gather(layer), caches[1].layers[0].state.kv.gather(layer)):
                    # the new row of the first layer is the token's own
                    assert torch.equal(x[:, :n + 1 - layer], y[:, :n + 1 - layer])
            # packed, the rows lie in other tiles and are added up in another order: the attention's outputs may round the other
            # way, at most 2^-8 of each, one of the some 10 such roundings a layer that leave a correlation of 0.9999
            assert torch.corrcoef(torch.stack([a, b]))[0, 1].item() > 0.999
        finally:
            tp.restore(model)
    assert caches[0].get_seq_length() == caches[1].get_seq_length()


def test_an_empty_cache_decodes_to_zeros():
    q = torch.randn(3, 2, 4, 128, device=DEV).to(BF)
    k = torch.zeros(3, 2, 64, int4.row_bytes(128), dtype=torch.uint8, device=DEV)
    assert not int4.decode_attention_int4(q, k[:, :, :0], k[:, :, :0], 0.1).any()
    assert not int4.decode_attention_int4(q[0], k[0, :, :0], k[0, :, :0], 0.1).any()
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert not int4.decode_attention_int4(q, k[:, :, :0], k[:, :, :0], 0.1, lens).any()
