"""Queries that a tensor map cannot describe (rows off a 16-byte boundary, broadcast, an odd stride of an extent of
one) in the windowed prefill and the shared-prefix decode on a B200: the results of the tensor-core kernel, to the bit,
not those of the plain one that takes the other tensors' odd layouts."""
import pytest
import torch

from threadcut_b200 import _lib, flash_decode, prefill

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


@pytest.fixture(params=[True, False], ids=["binding", "checked"])
def binding(request, monkeypatch):
    """Through the compiled binding, and through the checked Python path."""
    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: None)


def views(q):
    """Views with q's shape, and what they hold."""
    b, h, r, d = q.shape
    pad = torch.zeros(b, h, r, d + 1, device=DEV, dtype=q.dtype)
    pad[..., 1:] = q
    yield pad[..., 1:]                                 # rows off their boundary, odd strides
    yield q[:1].expand(b, -1, -1, -1)
    yield q[:, :1].expand(-1, h, -1, -1)
    yield q[:, :, :1].expand(-1, -1, r, -1)
    yield q.transpose(2, 3).contiguous().transpose(2, 3)  # last dimension not contiguous


def rand(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256)])
def test_shared_decode(binding, dtype, d):
    gen = torch.Generator(device=DEV).manual_seed(d)
    q, kp, vp = rand(gen, dtype, 3, 2, 4, d), rand(gen, dtype, 2, 500, d), rand(gen, dtype, 2, 500, d)
    k, v = rand(gen, dtype, 3, 2, 70, d), rand(gen, dtype, 3, 2, 70, d)
    for x in views(q):
        want = flash_decode.decode_attention_shared(x.contiguous(), kp, vp, k, v, 0.1)
        assert torch.equal(flash_decode.decode_attention_shared(x, kp, vp, k, v, 0.1), want)
    one = q[:1, :, :1]
    want = flash_decode.decode_attention_shared(one.contiguous(), kp, vp, k[:1], v[:1], 0.1)
    odd = one.as_strided(one.shape, [5, one.stride(1), 3, 1])
    assert torch.equal(flash_decode.decode_attention_shared(odd, kp, vp, k[:1], v[:1], 0.1), want)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_window_prefill(binding, dtype, d):
    gen = torch.Generator(device=DEV).manual_seed(d)
    q, k, v = rand(gen, dtype, 2, 8, 50, d), rand(gen, dtype, 2, 2, 300, d), rand(gen, dtype, 2, 2, 300, d)
    for x in views(q):
        want = prefill.prefill_attention_window(x.contiguous(), k, v, 0.1, 100, 7)
        assert torch.equal(prefill.prefill_attention_window(x, k, v, 0.1, 100, 7), want)
    one = q[:1, :, :1]
    want = prefill.prefill_attention_window(one.contiguous(), k[:1], v[:1], 0.1, 100, 7)
    odd = one.as_strided(one.shape, [5, one.stride(1), 3, 1])
    assert torch.equal(prefill.prefill_attention_window(odd, k[:1], v[:1], 0.1, 100, 7), want)
