"""Decode attention over one long sequence of 4-bit rows, which takes kernels of 16 warps a CTA where a few rows take 8: every head
size and group that has them, in pages and contiguous, with and without gaps between the rows; against float64."""
import pytest
import torch

import int4_ref as ref
from attn_bounds import P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.int4 import decode_attention_int4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def randn(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def check(out, q, k, v, scale):
    kk, vv = (ref.values_of(x, q.shape[-1], q.dtype) for x in (k, v))
    assert_within(out, *attend64(q, kk, vv, scale, None, P_SPLIT[q.dtype]))


GROUPS = [(64, 1), (64, 4), (64, 7), (64, 8), (64, 16), (128, 1), (128, 3), (128, 5), (128, 8)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,g", GROUPS)
@pytest.mark.parametrize("hkv,n", [(8, 9001), (2, 34000), (1, 70001)])  # by 1 and 2 KV heads: more than 48 slices a head
def test_contiguous(dtype, d, g, hkv, n):
    q = randn(1, hkv, g, d, dtype=dtype)
    k, v = (ref.rows_of(randn(1, hkv, n, d, dtype=dtype, seed=s)) for s in (1, 2))
    out = decode_attention_int4(q, k, v, d ** -0.5)
    check(out, q, k, v, d ** -0.5)
    for some in (n - 17, 5, 0):  # slices of rows that the sequence does not have
        lens = torch.tensor([some], dtype=torch.int32, device=DEV)
        got = decode_attention_int4(q, k, v, d ** -0.5, lens)
        if some:
            check(got, q, k[:, :, :some], v[:, :, :some], d ** -0.5)
        else:
            assert not got.any()
    assert torch.equal(decode_attention_int4(q, k, v, d ** -0.5), out)  # the workspace was left as it was found


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,g", GROUPS)
def test_rows_with_gaps_and_heads_within_rows(dtype, d, g):
    hkv, n = 8, 9001
    q = randn(hkv, g, d, dtype=dtype)
    wide = [torch.full((hkv, n, ref.row_bytes(d) + 16), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    k, v = (w[..., :ref.row_bytes(d)] for w in wide)
    for s, x in enumerate((k, v)):
        x.copy_(ref.rows_of(randn(hkv, n, d, dtype=dtype, seed=s + 1)))
    check(decode_attention_int4(q, k, v, 0.1), q, k, v, 0.1)
    k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    check(decode_attention_int4(q, k, v, 0.1), q, k, v, 0.1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,g", GROUPS)
@pytest.mark.parametrize("hkv,n,page_rows", [(8, 9001, 64), (1, 67003, 100)])
def test_pages(dtype, d, g, hkv, n, page_rows):
    tiles, where, total = ref.pages(n, page_rows, torch.Generator().manual_seed(n), cuts=6)
    kp, vp = (ref.rows_of(randn(total, hkv, page_rows, d, dtype=dtype, seed=s)) for s in (1, 2))
    q = randn(hkv, g, d, dtype=dtype)
    k, v = (x[where[:, 0], :, where[:, 1]].transpose(0, 1) for x in (kp, vp))
    check(decode_attention_int4(q, kp, vp, d ** -0.5, tiles=tiles), q, k, v, d ** -0.5)
