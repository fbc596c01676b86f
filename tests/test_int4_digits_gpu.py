"""One and two tokens of a 4-bit projection, which enter as whole numbers: of any size, and with NaN and infinities."""
import pytest
import torch

from test_int4_gemv_gpu import BF, HF, check, randn
from threadcut_b200.int4 import gemv_int4, quantize_weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("power", [-115, -110, -101, -100, -90, -81, -80, -65, -64, -63, -40, 40, 100])
def test_tokens_of_any_size(group, power):
    w = quantize_weight(randn(70, 640, dtype=BF, seed=1), group)
    x = randn(2, 640, dtype=BF, seed=2) * 2.0 ** power
    for t in (x, x[:1], torch.stack((x[0], randn(640, dtype=BF, seed=3)))):
        check(gemv_int4(t, w), t, w)
    x[0, 64:128] *= 2.0 ** -5  # blocks on both sides of a limit
    x[1, 320:] = 0
    check(gemv_int4(x, w), x, w)


def test_the_smallest_numbers():
    # bf16's subnormal tokens times weights of about 2^60; fp16's smallest
    for dtype, unit, size in ((BF, 2.0 ** -133, 2.0 ** 60), (HF, 2.0 ** -24, 1.0)):
        w = quantize_weight(randn(40, 128, dtype=dtype, seed=1, scale=size), 64)
        x = (torch.randint(-100, 101, (2, 128), generator=torch.Generator().manual_seed(1)).double() * unit).to(dtype).cuda()
        assert x.any()
        check(gemv_int4(x, w), x, w)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_infinite_and_nan_tokens_show_in_their_rows_alone(dtype, group, bad):
    w = quantize_weight(randn(40, 200, dtype=dtype, seed=1, scale=0.02), group)
    x = randn(2, 200, dtype=dtype, seed=2)
    good = gemv_int4(x, w)
    for at in (0, 31, 32, 63, 100, 130, 199):  # either half of a block, a block that ends inside
        one = x[:1].clone()
        one[0, at] = bad
        assert not torch.isfinite(gemv_int4(one, w)).any()
        for token in (0, 1):
            two = x.clone()
            two[token, at] = bad
            out = gemv_int4(two, w)
            assert not torch.isfinite(out[token]).any() and torch.equal(out[1 - token], good[1 - token])
