"""Decode attention with a sliding window and sinks (decode_attention_window, PagedKV.decode(window=)) on a
B200 against float64 attention over the visible rows; tolerances as derived in attn_bounds."""
import pytest
import torch

from attn_bounds import P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention_batched, decode_attention_window
from threadcut_b200.match import Split
from threadcut_b200.paged import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def visible(lengths, n, window, sinks):
    j = torch.arange(n, device=DEV)
    ln = lengths.long()[:, None]
    return ((j < ln) & ((j < sinks) | (j >= ln - window)))[:, None, None]


def check(b, hkv, g, d, n, lengths, window, sinks, dtype, seed=0, cap=None, splits=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cap = n if cap is None else cap
    q = torch.randn(b, hkv, g, d, generator=gen, device=DEV).to(dtype)
    kb, vb = (torch.randn(b, hkv, cap, d, generator=gen, device=DEV).to(dtype) for _ in range(2))
    k, v = kb[:, :, :n], vb[:, :, :n]
    lens = torch.full((b,), n) if lengths is None else torch.tensor(lengths)
    lens = lens.to(DEV, torch.int32)
    out = decode_attention_window(q, k, v, d ** -0.5, window, sinks, None if lengths is None else lens, splits=splits)
    ref, tol = attend64(q, k, v, d ** -0.5, visible(lens, n, window, sinks), P_SPLIT[dtype])
    assert out.shape == q.shape and out.dtype == dtype
    assert_within(out, ref, tol)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 128), (F32, 16), (F16, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 32), (100, 33), (64, 500), (5000, 3)])
def test_windows(dtype, d, window, sinks):
    check(2, 2, 4, d, 700, [700, 131], window, sinks, dtype)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130])
@pytest.mark.parametrize("window,sinks", [(1, 0), (32, 1), (64, 64), (65, 63)])
def test_short_sequences(n, window, sinks):
    check(1, 4, 4, 128, n, None, window, sinks, BF16)


@pytest.mark.parametrize("g", [1, 2, 3, 7, 8, 9, 16])
def test_head_groups(g):
    check(3, 2, g, 64, 300, [300, 17, 200], 50, 5, F16)


def test_ragged_batch_with_an_empty_sequence():
    check(9, 4, 4, 128, 2000, [2000, 0, 1, 40, 39, 41, 1999, 7, 512], 36, 4, BF16)


def test_lengths_outside_the_tensor_are_clamped():
    check(1, 2, 4, 128, 100, None, 30, 2, BF16)
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(2, 2, x, 128, generator=gen, device=DEV).to(BF16) for x in (4, 100, 100))
    got = decode_attention_window(q, k, v, 0.1, 30, 2, torch.tensor([1000, -3], device=DEV, dtype=torch.int32))
    want = decode_attention_window(q, k, v, 0.1, 30, 2, torch.tensor([100, 0], device=DEV, dtype=torch.int32))
    assert torch.equal(got, want) and not want[1].any()


@pytest.mark.parametrize("splits", [1, 2, 7, 40, 128])
def test_forced_splits(splits):
    check(2, 2, 4, 128, 9000, [9000, 4097], 4096, 16, BF16, splits=splits)


def test_a_long_cache_and_many_sequences():
    check(1, 8, 4, 128, 100000, None, 4096, 4, BF16)
    check(80, 4, 2, 64, 900, [(37 * i) % 901 for i in range(80)], 128, 8, F16)


def test_rows_past_32_bit_element_offsets():
    """The last sequence's rows lie beyond 2^31 elements of the batch tensor."""
    b, hkv, n, d = 9, 2, 1 << 20, 128  # 9 * 2 * 2^20 * 128 = 2.4e9 elements
    k = torch.zeros(b, hkv, n, d, device=DEV, dtype=BF16)
    v = torch.zeros(b, hkv, n, d, device=DEV, dtype=BF16)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(b, hkv, 4, d, generator=gen, device=DEV).to(BF16)
    for x in (k, v):
        x[-1, :, -300:] = torch.randn(hkv, 300, d, generator=gen, device=DEV).to(BF16)
        x[-1, :, :40] = torch.randn(hkv, 40, d, generator=gen, device=DEV).to(BF16)
    out = decode_attention_window(q, k, v, 0.09, 300, 40)
    rows = torch.cat((torch.arange(40), torch.arange(n - 300, n))).to(DEV)
    ref, tol = attend64(q[-1], k[-1][:, rows], v[-1][:, rows], 0.09, p_bits=P_SPLIT[BF16])
    assert_within(out[-1], ref, tol)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 64)])
def test_what_is_hidden_may_hold_anything(dtype, d):
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(2, 2, x, d, generator=gen, device=DEV).to(dtype) for x in (4, 500, 500))
    lens = torch.tensor([480, 100], device=DEV, dtype=torch.int32)
    want = decode_attention_window(q, k, v, 0.1, 77, 5, lens)
    for i, ln in enumerate((480, 100)):
        for bad, x in ((float("nan"), k), (float("inf"), k), (float("nan"), v), (float("-inf"), v)):
            x[i, :, 5:ln - 77] = bad
            x[i, :, ln:] = bad
            assert torch.equal(decode_attention_window(q, k, v, 0.1, 77, 5, lens), want)


def test_a_window_over_everything_is_the_plain_decode():
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(3, 2, x, 128, generator=gen, device=DEV).to(BF16) for x in (4, 777, 777))
    lens = torch.tensor([777, 5, 400], device=DEV, dtype=torch.int32)
    assert torch.equal(decode_attention_window(q, k, v, 0.1, 10 ** 12, 0, lens),
                       decode_attention_batched(q, k, v, 0.1, lens))


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_strided_views_unaligned_rows_and_one_sequence_without_batch(dtype, d):
    gen = torch.Generator(device=DEV).manual_seed(7)
    q = torch.randn(2, 4, 2, d + 1, generator=gen, device=DEV).to(dtype).transpose(1, 2)[..., 1:]
    for pad in (8, 1):  # rows 16-byte aligned, then not
        kb, vb = (torch.randn(2, 300, 2, d + pad, generator=gen, device=DEV).to(dtype) for _ in range(2))
        k, v = (x.transpose(1, 2)[..., pad:] for x in (kb, vb))
        out = decode_attention_window(q, k, v, 0.1, 100, 3)
        ref, tol = attend64(q, k, v, 0.1, visible(torch.tensor([300, 300], device=DEV), 300, 100, 3), P_SPLIT[dtype])
        assert_within(out, ref, tol)
        assert torch.equal(decode_attention_window(q[1], k[1], v[1], 0.1, 100, 3), out[1])


def test_two_streams_and_two_replayed_graphs():
    gen = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = (torch.randn(4, 4, x, 128, generator=gen, device=DEV).to(BF16) for x in (4, 6000, 6000))
    wants = [decode_attention_window(q, k, v, 0.1, w, 4) for w in (1500, 5000)]
    graphs = []
    for w in (1500, 5000):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = decode_attention_window(q, k, v, 0.1, w, 4)
        graphs.append((gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, w in zip(streams, (1500, 5000)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(decode_attention_window(q, k, v, 0.1, w, 4))
        for st, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for want, x, (_, y) in zip(wants, got, graphs):
            assert torch.equal(want, x) and torch.equal(want, y)


@pytest.mark.parametrize("page_rows", [32, 64, 100])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (333, 70), (5000, 2)])
def test_paged_windows_after_a_splice(page_rows, window, sinks):
    hkv, g, d = 2, 4, 128
    gen = torch.Generator(device=DEV).manual_seed(9)
    kv = PagedKV(1, hkv, d, max_tokens=1500, page_rows=page_rows, device=DEV)
    inv = 1e4 ** (-torch.arange(0, d, 2).float() / d)
    for t in (600, 7, 300):
        kv.reserve(t)
        kv.write(0, *(torch.randn(hkv, t, d, generator=gen, device=DEV).to(BF16) for _ in range(2)))
    kv.splice(Split(101, 250, 555), inv)
    for step in range(70):  # fused one-token steps across page ends
        kv.reserve(1)
        q = torch.randn(hkv, g, d, generator=gen, device=DEV).to(BF16)
        kn, vn = (torch.randn(hkv, d, generator=gen, device=DEV).to(BF16) for _ in range(2))
        out = kv.decode(0, q, 0.1, k_new=kn, v_new=vn, window=window, sinks=sinks)
        if step % 9 == 0:
            k, v = kv.gather(0)
            assert torch.equal(k[:, -1], kn)
            seen = visible(torch.tensor([kv.n], device=DEV), kv.n, window, sinks)[0]
            ref, tol = attend64(q, k, v, 0.1, seen, P_SPLIT[BF16])
            assert_within(out, ref, tol)
            assert torch.equal(out, kv.decode(0, q, 0.1, window=window, sinks=sinks))
            other = visible(torch.tensor([kv.n], device=DEV), kv.n, window + 7, sinks + 1)[0]  # layers may differ
            assert_within(kv.decode(0, q, 0.1, window=window + 7, sinks=sinks + 1),
                          *attend64(q, k, v, 0.1, other, P_SPLIT[BF16]))
            assert torch.equal(out, kv.decode(0, q, 0.1, window=window, sinks=sinks))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_an_empty_cache_gives_zeros(d, dtype):
    q = torch.ones(2, 2, 4, d, device=DEV, dtype=dtype)
    k = torch.empty(2, 2, 0, d, device=DEV, dtype=dtype)
    assert not decode_attention_window(q, k, k, 0.1, 5, 1).any()
    assert not decode_attention_window(q, k, k, 0.1, 5, 1, torch.tensor([0, 3], device=DEV, dtype=torch.int32)).any()


def test_broadcast_keys():
    """Keys and values expanded over sequences or heads (stride 0)."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn(3, 4, x, 128, generator=gen, device=DEV).to(BF16) for x in (4, 200, 200))
    seen = visible(torch.full((3,), 200, device=DEV), 200, 60, 3)
    for kk, vv in ((k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)),
                   (k[:, :1].expand(-1, 4, -1, -1), v[:, :1].expand(-1, 4, -1, -1))):
        ref, tol = attend64(q, kk, vv, 0.1, seen, P_SPLIT[BF16])
        assert_within(decode_attention_window(q, kk, vv, 0.1, 60, 3), ref, tol)


def test_refusals():
    x = torch.zeros(2, 2, 8, 128, device=DEV, dtype=BF16)
    for bad in (dict(window=0), dict(window=-1), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            decode_attention_window(x, x, x, 0.1, **bad)
    with pytest.raises(ValueError):
        decode_attention_window(x, x, x, 0.1, 4, lengths=torch.zeros(3, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError):
        decode_attention_window(x, x[:1], x[:1], 0.1, 4)
    with pytest.raises(TypeError):
        decode_attention_window(x, x.half(), x.half(), 0.1, 4)
    with pytest.raises(_lib.TCError):  # more than 16 query heads a KV head
        decode_attention_window(torch.zeros(2, 2, 17, 128, device=DEV, dtype=BF16), x, x, 0.1, 4)
    kv = PagedKV(1, 2, 128, max_tokens=64, device=DEV)
    with pytest.raises(ValueError):
        kv.decode(0, x[0, :, :4], 0.1, sinks=3)
    with pytest.raises(ValueError):
        kv.decode(0, x[0, :, :4], 0.1, window=0)
