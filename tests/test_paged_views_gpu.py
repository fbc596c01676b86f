"""Broadcast and oddly strided views as queries and suffixes of the operators over a paged cache, on a B200: the same
results as from contiguous copies of them."""
import pytest
import torch

from threadcut_b200 import _lib
from threadcut_b200.paged import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HKV, G = 2, 4


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


@pytest.fixture
def gen():
    return torch.Generator(device=DEV).manual_seed(11)


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV).to(torch.bfloat16)


def cache(gen, d, n=333):
    kv = PagedKV(1, HKV, d, max_tokens=500, device=DEV)
    kv.reserve(n)
    kv.write(0, rand(gen, HKV, n, d), rand(gen, HKV, n, d))
    return kv


def unit_stride(x, stride):
    """x with extents of 1 stepped by `stride` elements, which no access uses."""
    return x.as_strided(x.shape, [stride if n == 1 else s for n, s in zip(x.shape, x.stride())])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_shared_decode_takes_broadcast_views(gen, d):
    kv = cache(gen, d)
    q, k, v = rand(gen, 3, HKV, G, d), rand(gen, 3, HKV, 40, d), rand(gen, 3, HKV, 40, d)
    for args in ((q[:1].expand(3, -1, -1, -1), k, v), (q[:, :1].expand(-1, HKV, -1, -1), k, v),
                 (q[:, :, :1].expand(-1, -1, G, -1), k, v), (q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)),
                 (q, k[:, :1].expand(-1, HKV, -1, -1), v), (q, k, v[:, :, :1].expand(-1, -1, 40, -1))):
        want = kv.decode_shared(0, *(x.contiguous() for x in args), 0.1)
        assert torch.equal(kv.decode_shared(0, *args, 0.1), want)


def test_shared_decode_takes_any_stride_of_an_extent_of_one(gen):
    kv = cache(gen, 128)
    q, k, v = rand(gen, 1, HKV, 1, 128), rand(gen, 1, HKV, 1, 128), rand(gen, 1, HKV, 1, 128)
    want = kv.decode_shared(0, q, k, v, 0.1)
    for stride in (0, 1, 131):
        assert torch.equal(kv.decode_shared(0, *(unit_stride(x, stride) for x in (q, k, v)), 0.1), want)


@pytest.mark.parametrize("d", [64, 128])
def test_window_prefill_takes_broadcast_and_odd_views(gen, d):
    kv = cache(gen, d)
    q = rand(gen, 1, HKV * G, 30, d)
    for x in (q[:, :1].expand(-1, HKV * G, -1, -1), q[:, :, :1].expand(-1, -1, 30, -1), unit_stride(q[:, :, :1], 3)):
        want = kv.prefill(0, x.clone(memory_format=torch.contiguous_format), 0.1, window=50, sinks=3)
        assert torch.equal(kv.prefill(0, x, 0.1, window=50, sinks=3), want)
