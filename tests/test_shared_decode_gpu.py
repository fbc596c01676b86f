"""Decode attention over a shared prefix and per-sequence suffixes (decode_attention_shared) on a B200
against float64 attention; tolerances as derived in attn_bounds (weights rounded to 16 bits)."""
import pytest
import torch

from attn_bounds import assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention_batched, decode_attention_shared
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


def make(b, hkv, g, d, n, m, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(b, hkv, g, d, generator=gen, device=DEV).to(dtype)
    kp, vp = (torch.randn(hkv, n + 16, d, generator=gen, device=DEV).to(dtype)[:, :n] for _ in range(2))
    k, v = (torch.randn(b, hkv, m + 3, d, generator=gen, device=DEV).to(dtype)[:, :, :m] for _ in range(2))
    return q, kp, vp, k, v


def reference(q, kp, vp, k, v, scale, lengths):
    b, hkv, g, d = q.shape
    n, m = kp.shape[1], k.shape[2]
    kk = torch.cat((kp.expand(b, -1, -1, -1), k), 2)
    vv = torch.cat((vp.expand(b, -1, -1, -1), v), 2)
    j = torch.arange(n + m, device=DEV)
    ln = lengths.to(DEV).long().clamp(0, m)[:, None]
    return attend64(q, kk, vv, scale, (j < n + ln)[:, None, None])


def check(b, hkv, g, d, n, m, dtype, lengths=None, scale=None, seed=0):
    q, kp, vp, k, v = make(b, hkv, g, d, n, m, dtype, seed)
    scale = d ** -0.5 if scale is None else scale
    lens = torch.full((b,), m) if lengths is None else torch.tensor(lengths)
    out = decode_attention_shared(q, kp, vp, k, v, scale, None if lengths is None else lens.to(DEV, torch.int32))
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    assert_within(out, *reference(q, kp, vp, k, v, scale, lens))


@pytest.mark.parametrize("n", [0, 1, 31, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("m", [0, 1, 40, 64, 65, 200])
def test_lengths(n, m):
    check(3, 2, 4, 128, n, m, BF16)


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64), (F16, 64), (BF16, 256), (F16, 256), (F32, 128), (F32, 256),
                                     (BF16, 80), (F16, 1), (F32, 255)])
def test_types_and_head_sizes(dtype, d):
    check(5, 2, 4, d, 777, 130, dtype, [130, 0, 1, 64, 99])


@pytest.mark.parametrize("b", [1, 2, 31, 32, 33, 65, 130])
@pytest.mark.parametrize("g", [1, 4, 7])
def test_batches_and_head_groups(b, g):
    check(b, 2, g, 128, 300, 70, BF16, [(13 * i) % 71 for i in range(b)])


@pytest.mark.parametrize("g", [2, 3, 5, 8, 16, 40, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_wide_groups(g, d):
    check(6, 1, g, d, 500, 90, F16, [90, 0, 5, 64, 65, 89])


def test_nothing_to_see():
    check(2, 2, 4, 128, 0, 0, BF16)
    check(3, 2, 4, 128, 0, 50, BF16, [0, 50, 7])
    check(2, 2, 4, 128, 70, 50, BF16, [0, 0])


def test_lengths_outside_the_tensor_are_clamped():
    q, kp, vp, k, v = make(3, 2, 4, 128, 100, 50, BF16)
    got = decode_attention_shared(q, kp, vp, k, v, 0.1, torch.tensor([99, -7, 50], device=DEV, dtype=torch.int32))
    want = decode_attention_shared(q, kp, vp, k, v, 0.1, torch.tensor([50, 0, 50], device=DEV, dtype=torch.int32))
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_other_scales(scale):
    check(4, 2, 4, 128, 300, 40, BF16, scale=scale)


def test_long_prefixes():
    check(2, 8, 4, 128, 50001, 33, BF16, [33, 2])
    check(40, 2, 4, 128, 20000, 500, F16, [(97 * i) % 501 for i in range(40)])
    check(1, 1, 1, 64, 30000, 1, BF16)


def test_one_long_suffix_among_short_ones():
    check(6, 2, 4, 128, 100, 9000, BF16, [3, 9000, 0, 1, 64, 4000])


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 64)])
def test_rows_behind_a_suffix_may_hold_anything(dtype, d):
    q, kp, vp, k, v = make(3, 2, 4, d, 200, 150, dtype)
    lens = torch.tensor([149, 0, 65], device=DEV, dtype=torch.int32)
    want = decode_attention_shared(q, kp, vp, k, v, 0.1, lens)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for x in (k, v):
            for i, ln in enumerate(lens.tolist()):
                x[i, :, ln:] = bad
            assert torch.equal(decode_attention_shared(q, kp, vp, k, v, 0.1, lens), want)


def test_rows_behind_a_prefix_view_may_hold_anything():
    q, kp, vp, k, v = make(3, 2, 4, 128, 201, 30, BF16)
    want = decode_attention_shared(q, kp, vp, k, v, 0.1)
    for x in (kp, vp):
        x._base[:, 201:] = float("nan")
    assert torch.equal(decode_attention_shared(q, kp, vp, k, v, 0.1), want)


def test_a_batch_equals_its_sequences_and_the_plain_decode():
    """Against decode_attention_batched over the copied-out concatenation, within both bounds."""
    q, kp, vp, k, v = make(4, 2, 4, 128, 333, 60, BF16)
    got = decode_attention_shared(q, kp, vp, k, v, 0.1)
    kk = torch.cat((kp.expand(4, -1, -1, -1), k), 2)
    vv = torch.cat((vp.expand(4, -1, -1, -1), v), 2)
    ref, tol = reference(q, kp, vp, k, v, 0.1, torch.full((4,), 60))
    assert_within(got, ref, tol)
    assert_within(decode_attention_batched(q, kk, vv, 0.1), ref, tol)
    for i in range(4):
        one = decode_attention_shared(q[i:i + 1], kp, vp, k[i:i + 1], v[i:i + 1], 0.1)
        assert_within(one, ref[i:i + 1], tol[i:i + 1])


@pytest.mark.parametrize("pad", [8, 1])
def test_strided_views_and_unaligned_rows(pad):
    gen = torch.Generator(device=DEV).manual_seed(4)

    def rand(*s):
        return torch.randn(*s, generator=gen, device=DEV).to(BF16)

    q = rand(3, 4, 2, 128 + pad).transpose(1, 2)[..., pad:]
    kp, vp = (rand(150, 2, 128 + pad).transpose(0, 1)[..., pad:] for _ in range(2))
    k, v = (rand(40, 3, 2, 128 + pad).permute(1, 2, 0, 3)[..., pad:] for _ in range(2))
    assert_within(decode_attention_shared(q, kp, vp, k, v, 0.1), *reference(q, kp, vp, k, v, 0.1, torch.full((3,), 40)))


def test_broadcast_tensors():
    """A prefix expanded over heads, suffixes expanded over sequences, one query for every sequence (stride 0)."""
    q, kp, vp, k, v = make(3, 4, 2, 128, 150, 40, BF16)
    for args in ((q, kp[:1].expand(4, -1, -1), vp[:1].expand(4, -1, -1), k, v),
                 (q, kp, vp, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)),
                 (q[:1].expand(3, -1, -1, -1), kp, vp, k, v)):
        assert_within(decode_attention_shared(*args, 0.1), *reference(*args, 0.1, torch.full((3,), 40)))


def test_prefix_rows_past_32_bit_element_offsets():
    hkv, n, d = 9, 1 << 21, 128  # 9 * 2^21 * 128 = 2.4e9 elements
    kp = torch.zeros(hkv, n, d, device=DEV, dtype=BF16)
    vp = torch.zeros(hkv, n, d, device=DEV, dtype=BF16)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(2, hkv, 4, d, generator=gen, device=DEV).to(BF16)
    k, v = (torch.randn(2, hkv, 5, d, generator=gen, device=DEV).to(BF16) for _ in range(2))
    # the last head: keys far along q for its last rows, so that they carry the softmax
    kp[-1, -20:] = (3 * q[:, -1, :, :].reshape(8, d).float().mean(0)).to(BF16)
    vp[-1, -20:] = torch.randn(20, d, generator=gen, device=DEV).to(BF16)
    out = decode_attention_shared(q, kp, vp, k, v, 0.5)
    ref, tol = reference(q[:, -1:], kp[-1:], vp[-1:], k[:, -1:], v[:, -1:], 0.5, torch.full((2,), 5))
    assert_within(out[:, -1:], ref, tol)


def test_another_stream_and_two_replayed_graphs():
    q, kp, vp, k, v = make(4, 2, 4, 128, 3000, 300, BF16)
    lens = torch.tensor([300, 1, 20, 0], device=DEV, dtype=torch.int32)
    sets = [(kp, vp), (kp[:, :700], vp[:, :700])]
    wants = [decode_attention_shared(q, a, c, k, v, 0.1, lens) for a, c in sets]
    graphs = []
    for a, c in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = decode_attention_shared(q, a, c, k, v, 0.1, lens)
        graphs.append((gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, (a, c), (gr, _) in zip(streams, sets, graphs):
            with torch.cuda.stream(st):
                gr.replay()
                got.append(decode_attention_shared(q, a, c, k, v, 0.1, lens))
        torch.cuda.synchronize()
        for want, x, (_, y) in zip(wants, got, graphs):
            assert torch.equal(want, x) and torch.equal(want, y)


def test_new_lengths_reach_a_replayed_graph():
    q, kp, vp, k, v = make(2, 2, 4, 128, 500, 300, BF16)
    lens = torch.tensor([10, 20], device=DEV, dtype=torch.int32)
    decode_attention_shared(q, kp, vp, k, v, 0.1, lens)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = decode_attention_shared(q, kp, vp, k, v, 0.1, lens)
    for a, c in ((11, 0), (300, 150), (1, 299)):
        lens.copy_(torch.tensor([a, c], dtype=torch.int32))
        gr.replay()
        assert_within(out, *reference(q, kp, vp, k, v, 0.1, torch.tensor([a, c])))


def paged_prefix(hkv, d, dtype, page_rows, gen, pieces, splice=None):
    kv = PagedKV(2, hkv, d, max_tokens=sum(pieces) + 500, page_rows=page_rows, dtype=dtype, device=DEV)
    for t in pieces:
        kv.reserve(t)
        for layer in range(2):
            kv.write(layer, *(torch.randn(hkv, t, d, generator=gen, device=DEV).to(dtype) for _ in range(2)))
    if splice:
        kv.splice(Split(*splice), 1e4 ** (-torch.arange(0, d, 2).float() / d))
    return kv


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256)])
@pytest.mark.parametrize("page_rows,pieces,splice", [
    (64, (1,), None), (64, (500,), None), (32, (33, 1, 90), None), (100, (700, 5, 1), None),
    (64, (900, 3), (101, 250, 555)), (40, (600, 40, 7), (33, 34, 500)), (64, (2000,), (70, 1500, 500))])
@pytest.mark.parametrize("b", [1, 5, 40])
def test_a_paged_prefix(dtype, d, page_rows, pieces, splice, b):
    hkv, g, m = 2, 4, 90
    gen = torch.Generator(device=DEV).manual_seed(b)
    kv = paged_prefix(hkv, d, dtype, page_rows, gen, pieces, splice)
    q, _, _, k, v = make(b, hkv, g, d, 1, m, dtype)
    lens = torch.tensor([(29 * i) % (m + 1) for i in range(b)], device=DEV, dtype=torch.int32)
    for layer in range(2):
        kp, vp = kv.gather(layer)
        out = kv.decode_shared(layer, q, k, v, 0.1, lens)
        assert_within(out, *reference(q, kp, vp, k, v, 0.1, lens.cpu()))
    # rows of the pages that no run lists may hold anything
    live = torch.zeros(kv.table.num_pages, page_rows, dtype=torch.bool, device=DEV)
    pos = torch.from_numpy(kv.table.positions()).to(DEV)
    live[pos[:, 0], pos[:, 1]] = True
    for pool in (kv.k[1], kv.v[1]):
        pool.transpose(1, 2)[~live] = float("nan")
    assert torch.equal(kv.decode_shared(1, q, k, v, 0.1, lens), out)


def test_an_empty_paged_prefix_and_unaligned_suffixes():
    gen = torch.Generator(device=DEV).manual_seed(1)
    kv = PagedKV(1, 2, 128, max_tokens=64, device=DEV)
    q, kp, vp, k, v = make(3, 2, 4, 128, 0, 20, BF16)
    assert_within(kv.decode_shared(0, q, k, v, 0.1), *reference(q, kp, vp, k, v, 0.1, torch.full((3,), 20)))
    kv = paged_prefix(2, 128, BF16, 64, gen, (77,))
    kp, vp = kv.gather(0)
    odd = torch.randn(3, 2, 21, 130, generator=gen, device=DEV).to(BF16)[:, :, 1:, 1:129]
    assert_within(kv.decode_shared(0, q, odd, odd, 0.1), *reference(q, kp, vp, odd, odd, 0.1, torch.full((3,), 20)))
    empty = k[:, :, :0]
    assert_within(kv.decode_shared(0, q, empty, empty, 0.1), *reference(q, kp, vp, empty, empty, 0.1, torch.zeros(3)))


def test_table_entries_outside_the_pool_count_as_empty():
    gen = torch.Generator(device=DEV).manual_seed(2)
    kv = paged_prefix(2, 128, BF16, 64, gen, (300,))
    q, _, _, k, v = make(2, 2, 4, 128, 1, 20, BF16)
    kp, vp = kv.gather(0)
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    tiles, _ = kv._tiles()  # the device copy: entries 1, 4 and 6 are made bad
    for i, bad in ((1, (-1, 0, 32)), (4, (kv.table.num_pages, 0, 32)), (6, (0, 40, 32))):
        keep[32 * i:32 * i + 32] = False
        tiles[i] = torch.tensor(bad, dtype=torch.int32)
    out = kv.decode_shared(0, q, k, v, 0.1)
    assert_within(out, *reference(q, kp[:, keep], vp[:, keep], k, v, 0.1, torch.full((2,), 20)))


def test_refusals():
    kv = PagedKV(1, 2, 128, max_tokens=64, device=DEV)
    q, kp, vp, k, v = make(2, 2, 4, 128, 20, 10, BF16)
    for bad in ((q, k[:1], v[:1], 0.1), (q, k, v[:, :, :3], 0.1), (q[..., :64], k, v, 0.1), (q, k, v, 0.0), (q, k, v, -1.0),
                (q, k, v, 0.1, torch.zeros(3, device=DEV, dtype=torch.int32))):
        with pytest.raises(ValueError):
            kv.decode_shared(0, *bad)
    with pytest.raises(TypeError):
        kv.decode_shared(0, q.half(), k.half(), v.half(), 0.1)
    q, kp, vp, k, v = make(2, 2, 4, 128, 20, 10, BF16)
    with pytest.raises(ValueError):
        decode_attention_shared(q, kp[:1], vp[:1], k, v, 0.1)
    with pytest.raises(ValueError):
        decode_attention_shared(q, kp, vp, k[:1], v[:1], 0.1)
    with pytest.raises(ValueError):
        decode_attention_shared(q, kp, vp[:, :5], k, v, 0.1)
    with pytest.raises(ValueError):
        decode_attention_shared(q, kp, vp, k, v, 0.1, torch.zeros(3, device=DEV, dtype=torch.int32))
    with pytest.raises(TypeError):
        decode_attention_shared(q, kp, vp, k.half(), v.half(), 0.1)
    with pytest.raises(_lib.TCError):
        decode_attention_shared(*make(1, 1, 129, 64, 5, 5, BF16), 0.1)
