"""Sliding-window layers through the transformers plugin on a B200: the windowed kernels run when the mask is
exactly the window, against float64 attention (bounds of attn_bounds) and against the same model with
transformers' SDPA attention."""
import pytest
import torch
from transformers import AutoModelForCausalLM, DynamicCache, Qwen3Config

from attn_bounds import P_SINGLE, P_SPLIT, assert_within, attend64
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


@pytest.fixture
def calls(monkeypatch):
    """Names of the windowed entry points that the plugin called."""
    seen = []
    for mod, name in ((tc_attention, "decode_attention_window"), (tc_attention._prefill, "prefill_attention_window")):
        fn = getattr(mod, name)
        monkeypatch.setattr(mod, name, lambda *a, _f=fn, _n=name, **k: (seen.append(_n), _f(*a, **k))[1])
    return seen


@pytest.mark.parametrize("lq,lk,w", [(1, 50, 20), (1, 50, 1), (30, 50, 7), (50, 50, 49), (200, 900, 130), (5, 9, 100)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 3, 64)])
def test_a_window_mask_runs_the_windowed_kernels(calls, lq, lk, w, hq, hkv, d):
    gen = torch.Generator(device=DEV).manual_seed(lk)
    q, k, v = (torch.randn(1, h, n, d, generator=gen, device=DEV).to(torch.bfloat16)
               for h, n in ((hq, lq), (hkv, lk), (hkv, lk)))
    mask = window_mask(lq, lk, w)
    out, _ = tc_attention.attention(None, q, k, v, mask, scaling=0.1, sliding_window=w)
    assert calls == ["decode_attention_window" if lq == 1 else "prefill_attention_window"]
    kk, vv = (x[0].repeat_interleave(hq // hkv, 0) for x in (k, v))
    ref, tol = attend64(q[0], kk, vv, 0.1, mask[0], (P_SPLIT if lq == 1 else P_SINGLE)[torch.bfloat16])
    assert out.shape == (1, lq, hq, d) and out.is_contiguous()
    assert_within(out[0].transpose(0, 1), ref, tol)


def test_any_other_mask_keeps_the_sdpa_branch(calls):
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(1, h, n, 128, generator=gen, device=DEV).to(torch.bfloat16)
               for h, n in ((8, 30), (2, 60), (2, 60)))
    base = window_mask(30, 60, 12)
    holes = base.clone()
    holes[0, 0, 3, 28] = ~holes[0, 0, 3, 28]
    for mask, kw in ((holes, dict(sliding_window=12)), (base, dict(sliding_window=13)), (base, {}),
                     (base, dict(sliding_window=None)), (base, dict(sliding_window=12, softcap=30.0))):
        out, _ = tc_attention.attention(None, q, k, v, mask, scaling=0.1, **kw)
        want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=0.1, enable_gqa=True)
        assert torch.equal(out, want.transpose(1, 2))
    assert calls == []
    base[0, 0, 3, 28] = ~base[0, 0, 3, 28]  # a mask changed in place is compared anew
    tc_attention.attention(None, q, k, v, base, scaling=0.1, sliding_window=12)
    assert calls == []


def sliding_model(impl):
    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=256, hidden_size=128, intermediate_size=256, num_hidden_layers=3, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=4096, use_sliding_window=True,
                      sliding_window=24, layer_types=["sliding_attention", "full_attention", "sliding_attention"])
    return AutoModelForCausalLM.from_config(cfg, dtype=torch.bfloat16, attn_implementation=impl).to(DEV).eval()


@pytest.mark.parametrize("paged", [False, True])
def test_a_model_with_sliding_layers_matches_sdpa(calls, monkeypatch, paged):
    """A 70-token prompt, a chunk and steps: logits within the bf16 tolerance of the engine tests."""
    from threadcut_b200.paged import PagedKV
    windows = []
    for name in ("decode", "prefill"):
        fn = getattr(PagedKV, name)
        monkeypatch.setattr(PagedKV, name,
                            lambda self, *a, _f=fn, _n=name, **k: (windows.append((_n, k.get("window"))), _f(self, *a, **k))[1])
    ours, ref = sliding_model(tc_attention.NAME), sliding_model("sdpa")
    ref.load_state_dict(ours.state_dict())
    c0 = new_cache(ours.config, paged=paged, max_tokens=500)
    c1 = DynamicCache()
    ids = torch.randint(0, 256, (1, 100), generator=torch.Generator().manual_seed(2)).to(DEV)
    at = 0
    with torch.no_grad():
        for n in (70, 20, 1, 1, 1):
            x = ids[:, at:at + n]
            pos = torch.arange(at, at + n, device=DEV)[None]
            a = ours(input_ids=x, position_ids=pos, past_key_values=c0, use_cache=True).logits
            b = ref(input_ids=x, position_ids=pos, past_key_values=c1, use_cache=True).logits
            assert torch.allclose(a.float(), b.float(), atol=3e-2, rtol=0)
            at += n
    if paged:
        assert [x for x in windows if x[1] == 24] == [("prefill", 24)] * 4 + [("decode", 24)] * 6
    else:
        assert calls == ["prefill_attention_window"] * 4 + ["decode_attention_window"] * 6
