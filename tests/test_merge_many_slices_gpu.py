"""Decode attention split into many slices, whose merge takes a slice of the output columns a CTA: groups of every size, odd ones
among them, over 4-bit, 16-bit and fp32 rows, against float64."""
import pytest
import torch

import int4_ref as ref
from attn_bounds import P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention, decode_attention_batched
from threadcut_b200.int4 import decode_attention_int4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def randn(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def check(out, q, k, v, scale):
    assert_within(out, *attend64(q, k, v, scale, None, P_SPLIT[q.dtype]))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("g", range(1, 17))
def test_4_bit_rows(d, g):
    dtype = BF if g % 2 else HF
    q = randn(2, 2, g, d, dtype=dtype)
    k, v = (ref.rows_of(randn(2, 2, 3000, d, dtype=dtype, seed=s)) for s in (1, 2))
    kk, vv = (ref.values_of(x, d, dtype) for x in (k, v))
    for splits in (23, 40, 94):  # a slice a tile at most
        check(decode_attention_int4(q, k, v, 0.1, splits=splits), q, kk, vv, 0.1)


@pytest.mark.parametrize("hkv,g,n", [(1, 3, 8000), (2, 5, 20000), (4, 3, 10000), (8, 3, 8000), (2, 7, 40000), (1, 13, 70000)])
def test_4_bit_rows_as_planned(hkv, g, n):
    """One sequence of heads of 64: 32 to 80 slices of 8 warps, 74 and more of 16."""
    q = randn(1, hkv, g, 64, dtype=BF)
    k, v = (ref.rows_of(randn(1, hkv, n, 64, dtype=BF, seed=s)) for s in (1, 2))
    check(decode_attention_int4(q, k, v, 0.125), q, *(ref.values_of(x, 64, BF) for x in (k, v)), 0.125)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("g", [1, 3, 5, 7, 11, 13, 15, 16])
def test_16_bit_and_fp32_rows(dtype, d, g):
    q, k, v = randn(2, g, d, dtype=dtype), randn(2, 3000, d, dtype=dtype, seed=1), randn(2, 3000, d, dtype=dtype, seed=2)
    for splits in (11, 30, 94):
        check(decode_attention(q, k, v, 0.1, splits=splits), q, k, v, 0.1)
    qb, kb, vb = (x[None].expand(3, *x.shape).contiguous() for x in (q, k, v))
    check(decode_attention_batched(qb, kb, vb, 0.1, splits=30), qb, kb, vb, 0.1)
