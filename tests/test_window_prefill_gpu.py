"""Prefill attention with a sliding window and sinks (prefill_attention_window) on a B200 against float64
attention over the visible keys; tolerances as derived in attn_bounds (weights rounded to 16 bits)."""
import pytest
import torch

from attn_bounds import assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.match import Split
from threadcut_b200.paged import PagedKV
from threadcut_b200.prefill import prefill_attention, prefill_attention_window

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def visible(lq, lk, window, sinks):
    at = (lk - lq + torch.arange(lq, device=DEV))[:, None]
    j = torch.arange(lk, device=DEV)
    return (j <= at) & ((j < sinks) | (j > at - window))


def reference(q, k, v, scale, window, sinks):
    g = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    ref, tol = attend64(q, kk, vv, scale, visible(q.shape[2], k.shape[2], window, sinks))
    return ref.transpose(1, 2), tol.transpose(1, 2)


def make(b, hkv, g, lq, lk, d, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(b, lq, hkv * g, d, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    k, v = (torch.randn(b, hkv, lk + 8, d, generator=gen, device=DEV).to(dtype)[:, :, :lk] for _ in range(2))
    return q, k, v


def check(b, hkv, g, lq, lk, d, dtype, window, sinks, splits=None, scale=None, seed=0):
    q, k, v = make(b, hkv, g, lq, lk, d, dtype, seed)
    scale = d ** -0.5 if scale is None else scale
    out = prefill_attention_window(q, k, v, scale, window, sinks, splits=splits)
    assert out.shape == (b, lq, hkv * g, d) and out.is_contiguous() and out.dtype == dtype
    assert_within(out, *reference(q, k, v, scale, window, sinks))


WINDOWS = [(1, 0), (1, 1), (1, 200), (63, 0), (64, 4), (128, 128), (129, 127), (300, 33), (4000, 5), (10 ** 12, 0)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 700), (33, 33), (130, 700), (700, 700), (257, 1031)])
def test_windows(lq, lk, window, sinks):
    check(1, 2, 4, lq, lk, 128, BF16, window, sinks)


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64), (F16, 64), (F32, 128), (F32, 64), (BF16, 256), (F16, 80),
                                     (BF16, 1), (F32, 255)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 7)])
def test_types_and_head_sizes(dtype, d, window, sinks):
    check(2, 2, 2, 150, 411, d, dtype, window, sinks)


@pytest.mark.parametrize("g", [1, 2, 3, 5, 6, 7, 8, 16, 24, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_head_groups(g, d):
    check(2, 2, g, 70, 200, d, BF16, 50, 3)


@pytest.mark.parametrize("splits", [1, 2, 3, 16])
@pytest.mark.parametrize("lq", [1, 100])
def test_forced_splits(splits, lq):
    check(2, 2, 4, lq, 2000, 128, BF16, 900, 130, splits=splits)
    check(1, 2, 4, lq, 2000, 64, F16, 2000, 0, splits=splits)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_other_scales(scale):
    check(1, 2, 4, 90, 300, 128, BF16, 60, 9, scale=scale)


def test_long_chunks():
    check(1, 1, 4, 300, 40000, 128, BF16, 4096, 4)
    check(1, 1, 2, 3000, 3000, 64, F16, 512, 0)


def test_a_window_over_everything_is_the_causal_prefill():
    q, k, v = make(1, 2, 4, 200, 900, 128, BF16)
    a = prefill_attention_window(q, k, v, 0.1, 10 ** 9)
    assert_within(a, *reference(q, k, v, 0.1, 10 ** 9, 0))
    b = prefill_attention(q, k, v, 0.1)
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7  # two roundings of values below 2


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("lq,lk,window,sinks", [(100, 2000, 256, 5), (300, 2000, 33, 130), (1, 700, 1, 0), (40, 500, 60, 0)])
def test_keys_that_no_query_of_the_call_sees_may_hold_anything(dtype, d, lq, lk, window, sinks):
    """Also where they share a key tile with keys that are seen."""
    q, k, v = make(1, 2, 4, lq, lk, d, dtype)
    want = prefill_attention_window(q, k, v, 0.1, window, sinks)
    first = lk - lq + 1 - window
    assert first > sinks
    for bad in (float("nan"), float("inf"), float("-inf")):
        for x in (k, v):
            x[:, :, sinks:first] = bad
            x._base[:, :, lk:] = bad
        assert torch.equal(prefill_attention_window(q, k, v, 0.1, window, sinks), want)


def test_broadcast_keys():
    """Keys and values expanded over sequences or heads (stride 0)."""
    q, k, v = make(2, 4, 2, 50, 300, 128, BF16)
    for kk, vv in ((k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)),
                   (k[:, :1].expand(-1, 4, -1, -1), v[:, :1].expand(-1, 4, -1, -1))):
        assert_within(prefill_attention_window(q, kk, vv, 0.1, 60, 3), *reference(q, kk, vv, 0.1, 60, 3))


@pytest.mark.parametrize("d,pad", [(128, 8), (128, 1), (64, 3)])
def test_strided_and_unaligned_inputs(d, pad):
    gen = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn(2, 8, 60, d + pad, generator=gen, device=DEV).to(BF16)[..., pad:]
    k, v = (torch.randn(2, 200, 2, d + pad, generator=gen, device=DEV).to(BF16).transpose(1, 2)[..., pad:]
            for _ in range(2))
    assert_within(prefill_attention_window(q, k, v, 0.1, 70, 3), *reference(q, k, v, 0.1, 70, 3))
    qt = q.contiguous().transpose(2, 3).contiguous().transpose(2, 3)  # last dimension not contiguous
    assert_within(prefill_attention_window(qt, k, v, 0.1, 70, 3), *reference(q, k, v, 0.1, 70, 3))


def test_another_stream_and_two_replayed_graphs():
    q, k, v = make(1, 2, 4, 40, 3000, 128, BF16)
    wants = [prefill_attention_window(q, k, v, 0.1, w, 4) for w in (700, 2500)]
    graphs = []
    for w in (700, 2500):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = prefill_attention_window(q, k, v, 0.1, w, 4)
        graphs.append((gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, w, (gr, _) in zip(streams, (700, 2500), graphs):
            with torch.cuda.stream(st):
                gr.replay()
                got.append(prefill_attention_window(q, k, v, 0.1, w, 4))
        torch.cuda.synchronize()
        for want, x, (_, y) in zip(wants, got, graphs):
            assert torch.equal(want, x) and torch.equal(want, y)


@pytest.mark.parametrize("dtype,d,g", [(BF16, 128, 4), (F16, 64, 2), (BF16, 128, 7), (F16, 64, 1)])
@pytest.mark.parametrize("page_rows,splice", [(64, None), (32, (101, 250, 555)), (100, (33, 34, 500))])
@pytest.mark.parametrize("window,sinks", [(1, 0), (60, 4), (129, 200), (10 ** 12, 0)])
def test_a_paged_cache(dtype, d, g, page_rows, splice, window, sinks):
    hkv = 2
    gen = torch.Generator(device=DEV).manual_seed(5)
    kv = PagedKV(1, hkv, d, max_tokens=2500, page_rows=page_rows, dtype=dtype, device=DEV)
    for t in (700, 5, 200):
        kv.reserve(t)
        kv.write(0, *(torch.randn(hkv, t, d, generator=gen, device=DEV).to(dtype) for _ in range(2)))
    if splice:
        kv.splice(Split(*splice), 1e4 ** (-torch.arange(0, d, 2).float() / d))
    for lq in (1, 77, 300):
        kv.reserve(lq)
        kv.write(0, *(torch.randn(hkv, lq, d, generator=gen, device=DEV).to(dtype) for _ in range(2)))
        q = torch.randn(1, lq, hkv * g, d, generator=gen, device=DEV).to(dtype).transpose(1, 2)
        k, v = kv.gather(0)
        want = reference(q, k[None], v[None], 0.1, window, sinks)
        for splits in (None, 3):
            assert_within(kv.prefill(0, q, 0.1, window=window, sinks=sinks, splits=splits), *want)
    # rows that no run lists, or that no query sees, may hold anything
    out = kv.prefill(0, q, 0.1, window=window, sinks=sinks)
    live = torch.zeros(kv.table.num_pages, page_rows, dtype=torch.bool, device=DEV)
    pos = torch.from_numpy(kv.table.positions()).to(DEV)
    seen = visible(lq, kv.n, window, sinks).any(0)
    live[pos[seen, 0], pos[seen, 1]] = True
    for pool in (kv.k[0], kv.v[0]):
        pool.transpose(1, 2)[~live] = float("nan")
    assert torch.equal(kv.prefill(0, q, 0.1, window=window, sinks=sinks), out)


def test_a_window_and_sinks_over_a_paged_cache_need_a_fitting_call():
    kv = PagedKV(1, 2, 128, max_tokens=64, device=DEV)
    kv.reserve(20)
    q = torch.zeros(1, 8, 5, 128, device=DEV, dtype=BF16)
    for bad in (dict(window=0), dict(window=3, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            kv.prefill(0, q, 0.1, **bad)
    with pytest.raises(ValueError):
        kv.prefill(0, q, -0.1, window=3)
    with pytest.raises(ValueError):
        kv.prefill(0, q[:, :7], 0.1, window=3)
    with pytest.raises(ValueError):
        kv.prefill(0, torch.zeros(1, 8, 21, 128, device=DEV, dtype=BF16), 0.1, window=3)


def test_refusals():
    q, k, v = make(1, 2, 4, 8, 20, 128, BF16)
    for bad in (dict(window=0), dict(window=3, sinks=-1)):
        with pytest.raises(ValueError):
            prefill_attention_window(q, k, v, 0.1, **bad)
    with pytest.raises(ValueError):  # more queries than keys
        prefill_attention_window(q, k[:, :, :7], v[:, :, :7], 0.1, 4)
    with pytest.raises(ValueError):  # query heads not a multiple of the KV heads
        prefill_attention_window(q[:, :7], k, v, 0.1, 4)
    with pytest.raises(ValueError):
        prefill_attention_window(q, k[..., :64], v[..., :64], 0.1, 4)
    with pytest.raises(TypeError):
        prefill_attention_window(q, k.half(), v.half(), 0.1, 4)
    q, k, v = make(1, 1, 1, 4, 9, 257, BF16)
    with pytest.raises(_lib.TCError):
        prefill_attention_window(q, k, v, 0.1, 4)
