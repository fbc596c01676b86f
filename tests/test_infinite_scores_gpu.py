"""Visible keys that score -inf, in runs that fill whole groups and tiles, for the windowed and shared-prefix operators
on a B200: such a key has weight 0 and no influence, wherever it lies; a row that sees nothing else gives zeros.
Against float64 attention without those keys, tolerances as derived in attn_bounds. And a NaN that a windowed decode
sees shows in its result."""
import pytest
import torch

from attn_bounds import P_SINGLE, P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention, decode_attention_shared, decode_attention_window
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


@pytest.mark.parametrize("span", SPANS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 64), (BF16, 32)])
def test_window_decode(dtype, d, span):
    q, k, v, counts = make(1, d, dtype, span)
    j = torch.arange(300, device=DEV)
    for window, sinks in ((1000, 0), (200, 40)):
        for splits in (None, 1, 3, 10):
            out = decode_attention_window(q.reshape(1, 2, 2, d), k, v, 0.1, window, sinks, splits=splits)
            seen = (j < sinks) | (j >= 300 - window)
            assert_within(out.reshape(q.shape), *reference(q, k, v, counts, seen, P_SPLIT))


@pytest.mark.parametrize("span", SPANS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 64)])
def test_decode_of_the_whole_cache(dtype, d, span):
    q, k, v, counts = make(1, d, dtype, span)
    for splits in (None, 1, 3):
        out = decode_attention(q.reshape(2, 2, d), k[0], v[0], 0.1, splits=splits)
        assert_within(out.reshape(q.shape), *reference(q, k, v, counts, torch.ones_like(counts), P_SPLIT))


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("at", [3, 260])
def test_a_nan_that_is_seen_is_not_hidden(dtype, d, splits, at):
    """A NaN in a query row gives NaN in that row; one in a key or value that is seen in every row of its head; one in
    a hidden key or value in none."""
    q, k, v, _ = make(1, d, dtype, (0, 0))
    q = q.reshape(1, 2, 2, d)

    def run(q, k, v, **kw):
        return decode_attention_window(q, k, v, 0.1, 200, 40, splits=splits, **kw)

    want = run(q, k, v)
    assert torch.isfinite(want).all()
    bad = q.clone()
    bad[0, 1, 0, 5] = float("nan")
    got = run(bad, k, v)
    assert got[0, 1, 0].isnan().all() and torch.equal(got[0, 1, 1], want[0, 1, 1]) and torch.equal(got[0, 0], want[0, 0])
    for which in (0, 1):
        for row, seen in ((at, True), (70, False)):
            kv = [k.clone(), v.clone()]
            kv[which][0, 1, row] = float("nan")
            got = run(q, *kv)
            assert torch.equal(got[0, 0], want[0, 0])
            assert got[0, 1].isnan().all() if seen else torch.equal(got, want)
    # nothing is seen: zeros, whatever the tensors hold
    none = torch.zeros(1, device=DEV, dtype=torch.int32)
    assert (run(torch.full_like(q, float("nan")), torch.full_like(k, float("nan")), v, lengths=none) == 0).all()
