"""Argument checks of the serving operators without a GPU: the C entries refuse bad arguments (and accept
empty work) before touching CUDA, and the Python wrappers refuse CPU tensors."""
import ctypes

import pytest
import torch

from threadcut_b200 import _lib
from threadcut_b200.paged import append_rope

P = ctypes.c_void_p(256)  # an aligned address that is never read: every call below ends before a launch
N = None


def append_status(q=P, k=P, v=P, qo=P, kp=P, vp=P, hq=8, hkv=2, d=64, t=4, eps=1e-6, cos=P, sin=P, rot=64, table=2,
                  rows=64, pages=4, slots=P, dtype=2):
    return _lib.lib().tc_paged_append_rope(q, k, v, qo, kp, vp, hq, hkv, d, t, *[64] * 8, N, N, eps, cos, sin, rot, 64,
                                           64, table, rows, pages, 4096, 64, 64, slots, dtype, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=9), 3), (dict(table=1), 3), (dict(dtype=0, table=2), 3), (dict(d=63, rot=32), 1), (dict(d=514), 1),
    (dict(d=0), 1), (dict(rot=66), 1), (dict(rot=3), 1), (dict(rot=0), 1), (dict(hkv=0), 1), (dict(hq=-1), 1),
    (dict(t=-1), 1), (dict(rows=0), 1), (dict(pages=0), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(q=N), 1), (dict(qo=N), 1), (dict(k=N), 1), (dict(v=N), 1), (dict(kp=N), 1), (dict(vp=N), 1), (dict(cos=N), 1),
    (dict(sin=N), 1), (dict(slots=N), 1)])
def test_append_refuses(bad, status):
    assert append_status(**bad) == status


def test_append_of_no_tokens_does_nothing():
    assert append_status(t=0) == 0
    assert append_status(t=0, q=N, qo=N, hq=0) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_rope(x, x, x[0], x[0], x[None], x[None], torch.zeros(4, 2, dtype=torch.int32))


def window_status(q=P, k=P, v=P, out=P, b=2, hkv=2, g=4, d=128, n=100, window=10, sinks=2, scale=0.1, dtype=2, ws=P,
                  nb=1 << 30):
    return _lib.lib().tc_decode_attention_window(q, k, v, out, b, hkv, g, d, n, N, window, sinks, *[128] * 12, scale, 0,
                                                 dtype, ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=5), 3), (dict(window=0), 1), (dict(window=-4), 1), (dict(sinks=-1), 1), (dict(g=17), 1), (dict(g=0), 1),
    (dict(b=0), 1), (dict(hkv=0), 1), (dict(n=-1), 1), (dict(n=1 << 31), 1), (dict(q=N), 1), (dict(out=N), 1),
    (dict(k=N), 1), (dict(v=N), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(d=48), 1),
    (dict(dtype=0, d=256), 2)])
def test_window_decode_refuses(bad, status):
    assert window_status(**bad) == status


def test_window_workspace_follows_the_window_not_the_cache():
    size = _lib.lib().tc_decode_attention_window_workspace_size
    assert size(1, 8, 4, 128, 1 << 20, 2048, 16, 0, 2) == size(1, 8, 4, 128, 1 << 24, 2048, 16, 0, 2) > 0
    assert size(64, 8, 4, 128, 1 << 20, 2048, 16, 0, 2) == 0  # one slice per head: nothing to join
    assert size(64, 8, 4, 128, 1 << 20, 0, 16, 0, 2) == 0 and size(64, 8, 4, 128, 100, 5, -1, 0, 2) == 0


def prefill_status(q=P, k=P, v=P, out=P, b=1, hq=8, hkv=2, lq=4, lk=100, d=128, window=10, sinks=2, scale=0.1, splits=0,
                   dtype=2, ws=N, nb=0):
    return _lib.lib().tc_prefill_attention_window(q, k, v, out, b, hq, hkv, lq, lk, d, window, sinks, *[128] * 12, scale,
                                                  splits, dtype, ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=5), 3), (dict(window=0), 1), (dict(sinks=-1), 1), (dict(hq=7), 1), (dict(hq=1), 1), (dict(hkv=0), 1),
    (dict(b=0), 1), (dict(b=65536), 1), (dict(lq=0), 1), (dict(lk=3), 1), (dict(d=0), 1), (dict(d=257), 1),
    (dict(splits=-1), 1), (dict(q=N), 1), (dict(k=N), 1), (dict(v=N), 1), (dict(out=N), 1),
    (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1)])
def test_window_prefill_refuses(bad, status):
    assert prefill_status(**bad) == status


def shared_status(q=P, kp=P, vp=P, k=P, v=P, out=P, b=2, hkv=2, g=4, d=128, n=100, m=10, scale=0.1, dtype=2, ws=N, nb=0):
    return _lib.lib().tc_decode_attention_shared(q, kp, vp, k, v, out, b, hkv, g, d, n, m, N, *[128] * 16, scale, dtype,
                                                 ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=5), 3), (dict(b=0), 1), (dict(b=65536), 1), (dict(hkv=0), 1), (dict(g=0), 1), (dict(g=129), 1),
    (dict(d=0), 1), (dict(d=257), 1), (dict(n=-1), 1), (dict(m=-1), 1), (dict(n=1 << 31), 1), (dict(m=1 << 31), 1),
    (dict(q=N), 1), (dict(out=N), 1), (dict(kp=N), 1), (dict(vp=N), 1), (dict(k=N), 1), (dict(v=N), 1),
    (dict(scale=float("nan")), 1), (dict(scale=float("-inf")), 1)])
def test_shared_decode_refuses(bad, status):
    assert shared_status(**bad) == status


def shared_paged_status(q=P, kp=P, vp=P, k=P, v=P, out=P, b=2, hkv=2, g=4, d=128, rows=64, pages=4, page_stride=64, tiles=P,
                        nt=3, m=10, scale=0.1, dtype=2, ws=N, nb=0, qs=128):
    return _lib.lib().tc_decode_attention_shared_paged(q, kp, vp, k, v, out, b, hkv, g, d, rows, pages, page_stride, 64, 64,
                                                       tiles, nt, m, N, qs, *[128] * 11, scale, dtype, ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(b=0), 1), (dict(hkv=0), 1), (dict(g=0), 1), (dict(g=129), 1), (dict(d=96), 1),
    (dict(rows=31), 1), (dict(pages=0), 1), (dict(tiles=N), 1), (dict(nt=-1), 1), (dict(m=-1), 1), (dict(q=N), 1),
    (dict(out=N), 1), (dict(kp=N), 1), (dict(vp=N), 1), (dict(k=N), 1), (dict(v=N), 1), (dict(scale=0.0), 1),
    (dict(scale=float("nan")), 1), (dict(page_stride=65), 2), (dict(qs=127), 2), (dict(q=ctypes.c_void_p(8)), 2)])
def test_shared_paged_decode_refuses(bad, status):
    assert shared_paged_status(**bad) == status


def prefill_paged_status(q=P, kp=P, vp=P, out=P, hq=8, hkv=2, lq=4, lk=100, d=128, rows=64, pages=4, page_stride=64,
                         ktab=P, n_sub=4, qb=P, sink_tiles=1, window=10, sinks=2, qs=128, scale=0.1, splits=0, dtype=2):
    return _lib.lib().tc_prefill_attention_window_paged(q, kp, vp, out, hq, hkv, lq, lk, d, rows, pages, page_stride, 64,
                                                        64, ktab, n_sub, qb, sink_tiles, window, sinks, qs, 128, 128, 128,
                                                        scale, splits, dtype, N, 0, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(hq=7), 1), (dict(hkv=0), 1), (dict(hq=258), 1), (dict(lq=0), 1), (dict(lk=3), 1),
    (dict(d=256), 1), (dict(rows=31), 1), (dict(pages=0), 1), (dict(n_sub=0), 1), (dict(sink_tiles=-1), 1),
    (dict(window=0), 1), (dict(sinks=-1), 1), (dict(scale=0.0), 1), (dict(scale=float("nan")), 1), (dict(splits=-1), 1),
    (dict(q=N), 1), (dict(kp=N), 1), (dict(vp=N), 1), (dict(out=N), 1), (dict(ktab=N), 1), (dict(qb=N), 1),
    (dict(page_stride=65), 2), (dict(qs=127), 2), (dict(ktab=ctypes.c_void_p(8)), 2)])
def test_window_paged_prefill_refuses(bad, status):
    assert prefill_paged_status(**bad) == status


def test_window_sizes_take_any_window():
    most = (1 << 63) - 1
    prefill = _lib.lib().tc_prefill_window_workspace_size
    for args in ((1, 32, 8, 512, 98304, 128), (2, 8, 4, 777, 5001, 64), (1, 8, 2, 1, 1, 128)):
        assert prefill(*args, most, 0, 3) == prefill(*args, args[4], 0, 3)
        assert prefill(*args, 100, most, 3) == prefill(*args, 100, args[4], 3)
    assert prefill(1, 32, 8, 512, 98304, 128, 0, 0, 0) == 0 and prefill(1, 7, 2, 5, 9, 128, 4, 0, 0) == 0
    decode = _lib.lib().tc_decode_attention_window_workspace_size
    assert decode(1, 8, 4, 128, 4000, most, most, 0, 2) == decode(1, 8, 4, 128, 4000, 4000, 0, 0, 2)
