"""4-bit projections against float64 over the matrix that the codes stand for."""
import pytest
import torch

from threadcut_b200.int4 import Int4Weight, dequantize_weight, gemv_int4, quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def randn(*shape, dtype, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def bound(x, w, out):
    """Sums of products are off by 2^-23 of what has been added up (|x| (2 S + |z|) at most) for each of their steps: 16 or
    64 columns, then groups, then up to 16 parts. One or two tokens enter as whole numbers of at most 1 / 524,288 of the
    largest of each 64 columns: half of that off, for an S of 15/16. One rounding to the output's type."""
    half = torch.finfo(out.dtype).eps / 2
    p = w.params.double().permute(0, 3, 2, 1, 4).reshape(-1, w.params.shape[1], 2)[:w.n]
    scale = p[..., 0].repeat_interleave(w.group, 1)[:, :w.k]
    size = 2 * scale + p[..., 1].abs().repeat_interleave(w.group, 1)[:, :w.k]
    tiny = 2.0 ** -25 if out.dtype == HF else 0.0
    x = x.double().abs()
    pad = torch.nn.functional.pad(x, (0, -w.k % 64)).view(x.shape[0], -1, 64)
    step = (pad.amax(-1, keepdim=True) / 524288).expand_as(pad).reshape(x.shape[0], -1)[:, :w.k]
    off = (w.k / 8 + 64) * 2.0 ** -23 * (x @ size.t()) + (step / 2) @ scale.t()
    return off * (1 + half) + half * out.double().abs() * 1.01 + tiny


def check(got, x, w):
    want = x.double() @ dequantize_weight(w).double().t()
    # the fp32 matrix of dequantize_weight is itself off by two roundings
    assert got.dtype == x.dtype and got.shape == want.shape
    assert ((got.double() - want).abs() <= bound(x, w, got)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 64), (2, 17, 65), (1, 100, 2560), (3, 2561, 31), (8, 333, 1000), (9, 48, 130),
                                   (16, 1000, 257), (17, 40, 640), (32, 129, 2000), (33, 64, 128), (70, 33, 500)])
def test_against_float64(dtype, group, m, n, k):
    w = quantize_weight(randn(n, k, dtype=dtype, seed=1, scale=0.02), group)
    x = randn(m, k, dtype=dtype, seed=2)
    check(gemv_int4(x, w), x, w)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_long_rows_take_fewer_tokens_a_launch(group):
    w = quantize_weight(randn(40, 12288, dtype=BF, seed=1, scale=0.02), group)
    x = randn(20, 12288, dtype=BF, seed=2)
    check(gemv_int4(x, w), x, w)
    w = quantize_weight(randn(20, 60001, dtype=BF, seed=1, scale=0.02), group)
    x = randn(3, 60001, dtype=BF, seed=2)
    check(gemv_int4(x, w), x, w)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_tokens_of_very_different_sizes(dtype):
    w = quantize_weight(randn(300, 640, dtype=dtype, seed=1, scale=0.02), 64)
    x = randn(2, 640, dtype=dtype, seed=2)
    x[0, 5], x[0, 300] = 3000.0, -900.0
    x[1] *= 2.0 ** -12
    x[1, 64:128] = 0
    x[1, 200] = 1.0
    for t in (x, x[:1], x[1:]):
        check(gemv_int4(t, w), t, w)
    x = x * 0
    assert not gemv_int4(x[:1], w).any()


def test_many_rows():
    w = quantize_weight(randn(70001, 192, dtype=BF, seed=1, scale=0.02), 64)
    for m in (1, 5, 20):
        x = randn(m, 192, dtype=BF, seed=m)
        check(gemv_int4(x, w), x, w)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,k", [(1, 640), (3, 100), (1, 9728), (20, 72), (2, 33)])
def test_swiglu(dtype, m, k):
    w = quantize_weight(randn(90, k, dtype=dtype, seed=1, scale=0.02), 64)
    gu = randn(m, 2 * k, dtype=dtype, seed=2, scale=2.0)
    # silu and its product with up are rounded to T each: the tokens may be off by a step of T where the two exp differ
    act = (torch.nn.functional.silu(gu[:, :k].float()).to(dtype).float() * gu[:, k:].float()).to(dtype)
    got = gemv_int4(gu, w, swiglu=True)
    want = act.double() @ dequantize_weight(w).double().t()
    step = 2 * torch.finfo(dtype).eps
    extra = (step * act.double().abs() + 2.0 ** -23) @ dequantize_weight(w).double().abs().t()
    assert ((got.double() - want).abs() <= bound(act, w, got) + extra).all()


def test_views_of_tokens():
    w = quantize_weight(randn(50, 128, dtype=BF, seed=1, scale=0.02), 64)
    x = randn(2, 3, 128, dtype=BF)
    check(gemv_int4(x, w).view(6, 50), x.view(6, 128), w)
    assert gemv_int4(x, w).shape == (2, 3, 50)
    assert torch.equal(gemv_int4(x[0, 0], w), gemv_int4(x[0, :1], w)[0])
    for view in (randn(4, 200, dtype=BF)[:, 1:129], randn(4, 256, dtype=BF)[:, ::2], randn(1, 128, dtype=BF).expand(4, -1),
                 randn(128, 4, dtype=BF).t(), randn(4, 131, dtype=BF)[:, :128]):
        check(gemv_int4(view, w), view, w)
    assert gemv_int4(x[:0], w).shape == (0, 3, 50)


def test_infinite_and_nan_tokens_show_only_in_their_rows():
    w = quantize_weight(randn(40, 256, dtype=BF, seed=1, scale=0.02), 64)
    x = randn(4, 256, dtype=BF, seed=2)
    bad = x.clone()
    bad[1, 7], bad[2, 200] = float("nan"), float("inf")
    out = gemv_int4(bad, w)
    assert torch.equal(out[0], gemv_int4(x, w)[0]) and torch.equal(out[3], gemv_int4(x, w)[3])
    assert not torch.isfinite(out[1]).any() and not torch.isfinite(out[2]).any()


def test_quantised_weights_are_the_nearest_levels():
    for dtype in (BF, HF):
        for group in (32, 64, 128):
            m = randn(37, 200, dtype=dtype, seed=3, scale=0.05)
            m[5] = 0.25
            w = quantize_weight(m, group)
            assert w.codes.device == m.device and w.params.dtype == dtype
            p = w.params.double().permute(0, 3, 2, 1, 4).reshape(-1, w.params.shape[1], 2)[:37]
            s, z = (p[..., i].repeat_interleave(group, 1)[:, :200] for i in (0, 1))
            # half a level, and z's rounding at the ends of the range
            most = s / 32 * 1.001 + torch.finfo(dtype).eps / 2 * (z.abs() + 2 * s) + (2.0 ** -24 if dtype == HF else 0)
            assert ((dequantize_weight(w).double() - m.double()).abs() <= most).all()
            assert torch.equal(dequantize_weight(w)[5], m[5].float())
            on_cpu = quantize_weight(m.cpu(), group)
            assert torch.equal(on_cpu.codes, w.codes.cpu()) and torch.equal(on_cpu.params, w.params.cpu())


def test_graph_and_stream():
    w = quantize_weight(randn(500, 640, dtype=BF, seed=1, scale=0.02), 64)
    x = randn(1, 640, dtype=BF, seed=2)
    first = gemv_int4(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(gemv_int4(x, w), first)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemv_int4(x, w)
    x.copy_(randn(1, 640, dtype=BF, seed=9))
    graph.replay()
    assert torch.equal(y, gemv_int4(x, w))
    assert isinstance(w, Int4Weight)
