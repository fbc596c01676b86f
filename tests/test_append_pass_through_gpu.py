"""What lies past the rotated elements of a paged append (append_rope with rot < d) on a B200: without a norm weight
it passes through to the bit, whatever its neighbours hold, for rows that are whole 16-byte chunks on their
boundaries (the wide kernel) and for rows that are not."""
import pytest
import torch

from threadcut_b200 import _lib
from threadcut_b200.paged import append_rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
BITS = {BF16: torch.int16, F16: torch.int16, F32: torch.int32}


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def rows(gen, h, t, d, dtype, aligned):
    x = torch.randn(h, t, d + (0 if aligned else 3), generator=gen, device=DEV).to(dtype)
    return x if aligned else x[..., 1:d + 1]


def call(q, k, v, rot, dtype, gen, **kw):
    hkv, t, d = k.shape
    ang = torch.rand(t, rot, generator=gen, device=DEV)
    pools = [torch.zeros(1, hkv, 64, d, device=DEV, dtype=dtype) for _ in range(2)]
    slots = torch.stack((torch.zeros(t), torch.arange(t)), 1).to(DEV, torch.int32)
    out = append_rope(k, v, ang.cos().to(dtype), ang.sin().to(dtype), *pools, slots, q=q, **kw)
    return out, pools[0][0, :, :t]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("d,rot", [(64, 32), (128, 32), (128, 96), (256, 64)])
def test_values_pass_through_to_the_bit(dtype, aligned, d, rot):
    """Infinities, NaN and zeros of either sign, each alone in its row: a neighbour keeps its value."""
    gen = torch.Generator(device=DEV).manual_seed(d + rot)
    q, k, v = (rows(gen, h, d - rot, d, dtype, aligned) for h in (4, 2, 2))
    t = d - rot  # token i: element rot + i is special
    for x in (q, k):
        for h, special in zip(range(x.shape[0]), (float("inf"), float("nan"), -0.0, float("-inf"))):
            x[h, torch.arange(t), rot + torch.arange(t)] = special
    t = min(t, 64)
    q, k, v = q[:, :t], k[:, :t], v[:, :t]
    out, keys = call(q, k, v, rot, dtype, gen)
    for got, x in ((out, q), (keys, k)):
        got, want = got[..., rot:].contiguous(), x[..., rot:].contiguous()
        assert torch.equal(got.view(BITS[dtype]), want.view(BITS[dtype]))


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_with_a_weight_only_the_norm_acts(dtype, aligned):
    """z = x r w past rot, r and w positive: an infinite rotated element (r = 0) makes those zeros of their sign, and
    a zero keeps its sign; neither meets another element of the row."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    d, rot, t = 128, 32, 9
    q, k, v = (rows(gen, h, t, d, dtype, aligned) for h in (2, 2, 2))
    w = torch.full((d,), 1.5, device=DEV, dtype=dtype)
    for x in (q, k):
        x[:, 0, 3] = float("inf")   # rotated: r = rsqrt(inf) = 0
        x[:, 1, rot::2] = -0.0
        x[:, 2, rot::2] = 0.0
    out, keys = call(q, k, v, rot, dtype, gen, q_norm=w, k_norm=w)
    for got, x in ((out, q), (keys, k)):
        got, x = got[..., rot:], x[..., rot:]
        assert torch.isfinite(got).all()
        assert (got[:, 0] == 0).all()
        assert torch.equal(torch.signbit(got), torch.signbit(x))
