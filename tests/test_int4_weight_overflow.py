"""Weights whose group's scale or offset has no finite number: they read back as NaN throughout, as cache rows do."""
import pytest
import torch

from threadcut_b200 import int4


@pytest.mark.parametrize("dtype,values", [(torch.float16, (-60000.0, -50000.0)), (torch.float16, (-60000.0, 60000.0)),
                                          (torch.bfloat16, (-3e38, -1e38)), (torch.bfloat16, (-3e38, 3e38)),
                                          (torch.float16, (float("inf"), 1.0)), (torch.bfloat16, (-float("inf"), 1.0)),
                                          (torch.bfloat16, (float("nan"), 1.0))])
@pytest.mark.parametrize("group", [32, 128])
def test_groups_without_a_finite_scale(dtype, values, group):
    m = torch.ones(18, 2 * group, dtype=dtype)
    m[3, 5], m[3, 6], m[3, 7:group] = values[0], values[1], values[1]
    w = int4.dequantize_weight(int4.quantize_weight(m, group))
    assert torch.isnan(w[3, :group]).all()
    w[3, :group] = 1
    assert (w == 1).all()
