"""Visible keys that score -inf, in runs that fill whole groups and tiles, for the windowed and shared-prefix operators
on a B200: such a key has weight 0 and no influence, wherever it lies; a row that sees nothing else gives zeros.
Against float64 attention without those keys, tolerances as derived in attn_bounds."""
import pytest
import torch

from attn_bounds import P_SINGLE, P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention_shared, decode_attention_window
from threadcut_b200.prefill import prefill_attention_window

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SPANS = [(0, 32), (0, 140), (32, 64), (250, 300), (0, 299), (10, 290), (0, 300)]


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def make(lq, d, dtype, span, hkv=2, g=2, n=300):
    """Positive queries, so that a key of -inf elements scores -inf; also returns the keys that count."""
    gen = torch.Generator(device=DEV).manual_seed(d + span[0])
    q = (torch.rand(1, hkv * g, lq, d, generator=gen, device=DEV) + 0.1).to(dtype)
    k, v = (torch.randn(1, hkv, n, d, generator=gen, device=DEV).to(dtype) for _ in range(2))
    k[:, :, span[0]:span[1]] = -float("inf")
    counts = torch.ones(n, dtype=torch.bool, device=DEV)
    counts[span[0]:span[1]] = False
    return q, k, v, counts


def reference(q, k, v, counts, seen, bits):
    g = q.shape[1] // k.shape[1]
    kk = k.masked_fill(~counts[None, None, :, None], 0.0).repeat_interleave(g, 1)
    return attend64(q, kk, v.repeat_interleave(g, 1), 0.1, seen & counts, bits[q.dtype])


@pytest.mark.parametrize("span", SPANS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 96), (F32, 64), (F32, 128)])
def test_window_prefill(dtype, d, span):
    q, k, v, counts = make(40, d, dtype, span)
    at = (260 + torch.arange(40, device=DEV))[:, None]
    j = torch.arange(300, device=DEV)
    for window, sinks in ((1000, 0), (200, 40)):
        seen = (j <= at) & ((j < sinks) | (j > at - window))
        out = prefill_attention_window(q, k, v, 0.1, window, sinks).transpose(1, 2)
        assert_within(out, *reference(q, k, v, counts, seen, P_SINGLE))


@pytest.mark.parametrize("span", SPANS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 96), (F32, 64), (F32, 128)])
def test_shared_decode(dtype, d, span):
    q, k, v, counts = make(1, d, dtype, span)
    qq = q.reshape(1, 2, 2, d)
    for n in (0, 64, 200, 300):  # the run lies in the prefix, in the suffix, or in both
        out = decode_attention_shared(qq, k[0, :, :n], v[0, :, :n], k[:, :, n:], v[:, :, n:], 0.1)
        assert_within(out.reshape(q.shape), *reference(q, k, v, counts, torch.ones(300, dtype=torch.bool, device=DEV), P_SINGLE))
