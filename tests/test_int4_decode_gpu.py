"""Decode attention over 4-bit rows against float64 over the values that the rows stand for."""
import pytest
import torch

import int4_ref as ref
from attn_bounds import P_SPLIT, assert_within, attend64
from threadcut_b200.int4 import decode_attention_int4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def randn(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def rows(*shape, dtype, seed):
    return ref.rows_of(randn(*shape, dtype=dtype, seed=seed))


def check(out, q, k, v, scale, seen=None):
    d = q.shape[-1]
    want, tol = attend64(q, ref.values_of(k, d, q.dtype), ref.values_of(v, d, q.dtype), scale, seen, P_SPLIT[q.dtype])
    assert out.dtype == q.dtype and out.shape == q.shape
    assert_within(out, want, tol)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hkv,g,n", [(1, 1, 1, 1), (2, 3, 4, 31), (1, 8, 4, 32), (3, 2, 8, 33), (1, 2, 16, 257),
                                       (5, 1, 9, 700), (1, 4, 7, 4096), (40, 2, 3, 65)])
def test_all_rows(dtype, d, b, hkv, g, n):
    q, k, v = randn(b, hkv, g, d, dtype=dtype), rows(b, hkv, n, d, dtype=dtype, seed=1), rows(b, hkv, n, d, dtype=dtype, seed=2)
    check(decode_attention_int4(q, k, v, d ** -0.5), q, k, v, d ** -0.5)


@pytest.mark.parametrize("splits", [1, 2, 7, 24, 25, 128, 1000])
@pytest.mark.parametrize("g", [4, 12])
def test_any_number_of_slices(splits, g):
    q, k, v = randn(2, 2, g, 128, dtype=BF), rows(2, 2, 5000, 128, dtype=BF, seed=1), rows(2, 2, 5000, 128, dtype=BF, seed=2)
    check(decode_attention_int4(q, k, v, 0.1, splits=splits), q, k, v, 0.1)


@pytest.mark.parametrize("d,n", [(64, 100), (128, 3000), (256, 500)])
def test_lengths_are_clamped_and_the_rest_is_not_seen(d, n):
    lens = torch.tensor([n, 0, 1, 32, -7, n + 9, 33, n - 1], dtype=torch.int32, device=DEV)
    b = lens.shape[0]
    q, k, v = randn(b, 2, 5, d, dtype=HF), rows(b, 2, n, d, dtype=HF, seed=1), rows(b, 2, n, d, dtype=HF, seed=2)
    seen = torch.arange(n, device=DEV) < lens.clamp(0, n)[:, None]
    # what lies behind a sequence may be anything: all bits set are NaN
    k = torch.where(seen[:, None, :, None], k, torch.full_like(k, 255))
    v = torch.where(seen[:, None, :, None], v, torch.full_like(v, 255))
    out = decode_attention_int4(q, k, v, d ** -0.5, lens)
    kk = torch.where(seen[:, None, :, None], k, torch.zeros_like(k))
    vv = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    check(out, q, kk, vv, d ** -0.5, seen[:, None, None])
    assert not out[1].any() and not out[4].any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hkv,g,n,page_rows", [(128, 8, 4, 1, 64), (64, 2, 7, 100, 32), (128, 1, 16, 1000, 100),
                                                 (256, 2, 2, 333, 64), (128, 8, 4, 20000, 64)])
def test_pages(dtype, d, hkv, g, n, page_rows):
    tiles, where, total = ref.pages(n, page_rows, torch.Generator().manual_seed(n), cuts=6)
    kp, vp = (rows(total, hkv, page_rows, d, dtype=dtype, seed=s) for s in (1, 2))
    q = randn(hkv, g, d, dtype=dtype)
    k, v = (x[where[:, 0], :, where[:, 1]].transpose(0, 1) for x in (kp, vp))
    for tab in (tiles, tiles[:, :3].contiguous()):
        check(decode_attention_int4(q, kp, vp, d ** -0.5, tiles=tab), q, k, v, d ** -0.5)


def test_tiles_outside_the_pool_are_skipped():
    d = 128
    kp, vp = (rows(2, 2, 40, d, dtype=BF, seed=s) for s in (1, 2))
    tiles = torch.tensor([[2, 0, 32], [0, 38, 32], [-1, 0, 4], [1, 40, 3], [1, -1, 3], [1, 5, 4], [0, 0, 0], [0, 3, -2]],
                         dtype=torch.int32, device=DEV)
    q = randn(2, 4, d, dtype=BF)
    k, v = (torch.cat((x[0, :, 38:40], x[1, :, 5:9]), 1) for x in (kp, vp))
    check(decode_attention_int4(q, kp, vp, 0.1, tiles=tiles), q, k, v, 0.1)
    assert not decode_attention_int4(q, kp, vp, 0.1, tiles=tiles[:0]).any()
    assert not decode_attention_int4(q, kp, vp, 0.1, tiles=tiles[:1]).any()


@pytest.mark.parametrize("d", [64, 128])
def test_views(d):
    b, hkv, g, n = 3, 2, 4, 90
    big = [rows(b, hkv + 1, n + 20, d, dtype=BF, seed=s) for s in (1, 2)]
    q = randn(b, g, hkv, d, dtype=BF).transpose(1, 2)
    k, v = (x[:, 1:, 3:n + 3] for x in big)
    check(decode_attention_int4(q, k, v, 0.1), q, k, v, 0.1)
    wide = randn(b, hkv, g, 2 * d, dtype=BF)[..., ::2]
    check(decode_attention_int4(wide, k, v, 0.1), wide, k, v, 0.1)
    # one cache for every sequence, rows between two boundaries, one sequence without its batch dimension
    one = k[:1].expand(b, -1, -1, -1)
    check(decode_attention_int4(q, one, one, 0.1), q, one, one, 0.1)
    odd = torch.empty(b * hkv * n * ref.row_bytes(d) + 5, dtype=torch.uint8, device=DEV)[5:].view(b, hkv, n, -1).copy_(k)
    check(decode_attention_int4(q, odd, v, 0.1), q, odd, v, 0.1)
    check(decode_attention_int4(q[0], k[0], v[0], 0.1), q[0], k[0], v[0], 0.1)


def test_scale_zero_negative_and_large_scores():
    q, k, v = randn(1, 2, 4, 128, dtype=BF), rows(1, 2, 300, 128, dtype=BF, seed=1), rows(1, 2, 300, 128, dtype=BF, seed=2)
    for scale in (0.0, -0.2, 30.0):
        check(decode_attention_int4(q, k, v, scale), q, k, v, scale)


def test_a_nan_that_is_seen_shows():
    x = randn(1, 1, 64, 128, dtype=BF, seed=1)
    x[0, 0, 40, 3] = float("nan")
    q, v = randn(1, 1, 4, 128, dtype=BF), rows(1, 1, 64, 128, dtype=BF, seed=2)
    assert torch.isnan(decode_attention_int4(q, ref.rows_of(x), v, 0.1)).all()
    lens = torch.tensor([40], dtype=torch.int32, device=DEV)
    assert torch.isfinite(decode_attention_int4(q, ref.rows_of(x), v, 0.1, lens)).all()
    out = decode_attention_int4(q, v, ref.rows_of(x), 0.1)  # in the values: its own group of 32
    assert torch.isnan(out[..., :32]).all() and torch.isfinite(out[..., 32:]).all()


def test_repeats_to_the_bit_on_streams_and_in_graphs():
    lens = torch.tensor([3000, 77, 0, 1500], dtype=torch.int32, device=DEV)
    q, k, v = randn(4, 2, 4, 128, dtype=BF), rows(4, 2, 3000, 128, dtype=BF, seed=1), rows(4, 2, 3000, 128, dtype=BF, seed=2)
    first = decode_attention_int4(q, k, v, 0.1, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(decode_attention_int4(q, k, v, 0.1, lens), first)
    s.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, neither with the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = decode_attention_int4(q, k, v, 0.1, lens)
        graphs.append((graph, out))
    for l in ([3000, 77, 0, 1500], [5, 3000, 2999, 0]):
        lens.copy_(torch.tensor(l, dtype=torch.int32))
        want = decode_attention_int4(q, k, v, 0.1, lens)
        for graph, out in graphs:
            graph.replay()
            assert torch.equal(out, want)
    lens.fill_(2)
    graphs[0][0].replay()
    graphs[1][0].replay()
    check(graphs[1][1], q, k[:, :, :2], v[:, :, :2], 0.1)
