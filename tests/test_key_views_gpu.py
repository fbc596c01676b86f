"""Keys and values whose rows do not start on 16-byte boundaries, in the windowed prefill and in the plugin's
sliding-window layers on a B200: the results of the tensor-core kernel, to the bit."""
import pytest
import torch

from threadcut_b200 import _lib, attention, prefill

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("dtype,d,pad", [(BF16, 128, 1), (BF16, 128, 4), (F16, 64, 3)])
def test_rows_off_their_boundaries(monkeypatch, binding, dtype, d, pad):
    if not binding:
        monkeypatch.setattr(_lib, "host", lambda: None)
    gen = torch.Generator(device=DEV).manual_seed(pad)
    q = torch.randn(1, 8, 60, d, generator=gen, device=DEV).to(dtype)
    k, v = (torch.randn(1, 2, 700, d + pad, generator=gen, device=DEV).to(dtype)[..., pad:] for _ in range(2))
    kc, vc = k.contiguous(), v.contiguous()
    want = prefill.prefill_attention_window(q, kc, vc, 0.1, 100, 7)
    for a, b in ((k, v), (k, vc), (kc, v)):
        assert torch.equal(prefill.prefill_attention_window(q, a, b, 0.1, 100, 7), want)
    at = (640 + torch.arange(60, device=DEV))[:, None]
    j = torch.arange(700, device=DEV)
    mask = ((j <= at) & (j > at - 100))[None, None]
    want = prefill.prefill_attention_window(q, kc, vc, 0.1, 100)
    out, _ = attention.attention(None, q, k, v, mask, scaling=0.1, sliding_window=100)
    assert torch.equal(out, want)
