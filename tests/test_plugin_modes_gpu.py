"""The attention plugin on a B200 under torch.inference_mode(), against the same calls under no_grad."""
import pytest
import torch
from transformers import AutoModelForCausalLM, Qwen3Config

from threadcut_b200 import _lib
from threadcut_b200 import attention as tc_attention
from threadcut_b200.kv import new_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def window_mask(lq, lk, w):
    at = (lk - lq + torch.arange(lq, device=DEV))[:, None]
    j = torch.arange(lk, device=DEV)
    return ((j <= at) & (j > at - w))[None, None]


@pytest.mark.parametrize("lq,lk,w", [(1, 50, 20), (30, 50, 7), (50, 50, 49), (5, 9, 100)])
def test_a_window_mask_in_inference_mode(lq, lk, w):
    gen = torch.Generator(device=DEV).manual_seed(lk)
    q, k, v = (torch.randn(1, h, n, 128, generator=gen, device=DEV).to(torch.bfloat16)
               for h, n in ((8, lq), (2, lk), (2, lk)))
    with torch.no_grad():
        want, _ = tc_attention.attention(None, q, k, v, window_mask(lq, lk, w), scaling=0.1, sliding_window=w)
    with torch.inference_mode():
        got, _ = tc_attention.attention(None, q, k, v, window_mask(lq, lk, w), scaling=0.1, sliding_window=w)
        other, _ = tc_attention.attention(None, q, k, v, window_mask(lq, lk, w), scaling=0.1, sliding_window=w + 1)
    assert torch.equal(got, want)
    assert torch.isfinite(other).all()


@pytest.mark.parametrize("paged", [False, True])
def test_a_model_with_sliding_layers_in_inference_mode(paged):
    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=256, hidden_size=128, intermediate_size=256, num_hidden_layers=3, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=4096, use_sliding_window=True,
                      sliding_window=24, layer_types=["sliding_attention", "full_attention", "sliding_attention"])
    model = AutoModelForCausalLM.from_config(cfg, dtype=torch.bfloat16, attn_implementation=tc_attention.NAME).to(DEV).eval()
    ids = torch.randint(0, 256, (1, 100), generator=torch.Generator().manual_seed(2)).to(DEV)
    runs = []
    for mode in (torch.no_grad, torch.inference_mode):
        cache, at, out = new_cache(model.config, paged=paged, max_tokens=500), 0, []
        with mode():
            for n in (70, 20, 1, 1):
                out.append(model(input_ids=ids[:, at:at + n], position_ids=torch.arange(at, at + n, device=DEV)[None],
                                 past_key_values=cache, use_cache=True).logits.clone())
                at += n
        runs.append(out)
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d,hq", [(128, 8), (64, 6)])
def test_a_recorded_call_of_a_sliding_layer_has_gradients(d, hq):
    """The gradients of SDPA over the same mask, for each input that asks for them; without recording, the same
    windowed result as ever."""
    gen = torch.Generator(device=DEV).manual_seed(d)
    x = [torch.randn(1, h, n, d, generator=gen, device=DEV).to(torch.bfloat16) for h, n in ((hq, 30), (2, 60), (2, 60))]
    mask = window_mask(30, 60, 12)
    up = torch.randn(1, 30, hq, d, generator=gen, device=DEV).to(torch.bfloat16)

    def ours(*a):
        return tc_attention.attention(None, *a, mask, scaling=0.1, sliding_window=12)[0]

    def sdpa(*a):
        return torch.nn.functional.scaled_dot_product_attention(*a, attn_mask=mask, scale=0.1, enable_gqa=True).transpose(1, 2)

    plain = ours(*x)
    assert plain.grad_fn is None
    for asks in ((0, 1, 2), (0,), (1,), (2,)):
        grads = []
        for fn in (ours, sdpa):
            leaves = [t.clone().requires_grad_(i in asks) for i, t in enumerate(x)]
            out = fn(*leaves)
            out.backward(up)
            grads.append([out.detach()] + [t.grad for t in leaves if t.requires_grad])
        assert len(grads[0]) == 1 + len(asks)
        for a, b in zip(*grads):  # the same pass twice; fp32 sums in another order may move a rounding by one step
            assert torch.allclose(a.float(), b.float(), rtol=torch.finfo(torch.bfloat16).eps, atol=1e-5)
        with torch.no_grad():
            assert torch.equal(ours(*leaves), plain)


@pytest.mark.parametrize("lq", [1, 40])
def test_a_sliding_layer_with_values_of_another_head_size(lq):
    gen = torch.Generator(device=DEV).manual_seed(lq)
    q, k, v = (torch.randn(1, h, n, d, generator=gen, device=DEV).to(torch.bfloat16)
               for h, n, d in ((8, lq, 128), (2, 100, 128), (2, 100, 64)))
    mask = window_mask(lq, 100, 33)
    out, _ = tc_attention.attention(None, q, k, v, mask, scaling=0.1, sliding_window=33)
    want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=0.1, enable_gqa=True)
    assert torch.equal(out, want.transpose(1, 2))
