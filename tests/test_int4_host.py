"""Argument checks of the 4-bit operators without a GPU: the C entries refuse bad arguments (and accept empty work) before
touching CUDA, and the Python functions refuse what does not fit."""
import ctypes

import pytest
import torch

import int4_ref as ref
from threadcut_b200 import _lib, int4

P = ctypes.c_void_p(256)  # an aligned address that is never read: every call below ends before a launch
ODD = ctypes.c_void_p(260)
N = None


def append(q=P, k=P, v=P, qo=P, kp=P, vp=P, hq=8, hkv=2, d=64, t=4, eps=1e-6, cos=P, sin=P, rot=64, table=2, rows=64, pages=4,
           sp=5120, sh=2560, sr=40, slots=P, dtype=2):
    return _lib.lib().tc_int4_append_rope(q, k, v, qo, kp, vp, hq, hkv, d, t, *[64] * 8, N, N, eps, cos, sin, rot, 64, 64,
                                          table, rows, pages, sp, sh, sr, slots, dtype, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(dtype=9), 3), (dict(table=1), 3), (dict(d=96), 1), (dict(d=0), 1), (dict(d=512), 1),
    (dict(rot=66), 1), (dict(rot=3), 1), (dict(rot=-2), 1), (dict(hkv=0), 1), (dict(hkv=65536), 1), (dict(hq=-1), 1),
    (dict(t=-1), 1), (dict(t=1 << 31), 1), (dict(rows=0), 1), (dict(pages=0), 1), (dict(eps=-1.0), 1),
    (dict(eps=float("nan")), 1), (dict(q=N), 1), (dict(qo=N), 1), (dict(k=N), 1), (dict(v=N), 1), (dict(kp=N), 1),
    (dict(vp=N), 1), (dict(cos=N), 1), (dict(sin=N), 1), (dict(slots=N), 1), (dict(kp=ODD), 2), (dict(vp=ODD), 2),
    (dict(sp=5124), 2), (dict(sh=2564), 2), (dict(sr=44), 2), (dict(d=128, sr=40), 2)])
def test_append_refuses(bad, status):
    assert append(**bad) == status


def test_empty_work_is_done():
    assert append(t=0) == 0 and append(t=0, q=N, qo=N, hq=0, rot=0, cos=N, sin=N) == 0
    assert gather(n=0) == 0 and gather(nt=0, tiles=N) == 0
    assert rotate(nt=0, tiles=N) == 0
    assert gemv(m=0) == 0 and gemv(n=0) == 0


def gather(kp=P, vp=P, ko=P, vo=P, hkv=2, d=128, n=10, oh=1280, on=128, rows=64, pages=4, sr=80, tiles=P, nt=1, dtype=1):
    return _lib.lib().tc_int4_gather(kp, vp, ko, vo, hkv, d, n, oh, on, rows, pages, 10240, 5120, sr, tiles, nt, dtype, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(hkv=0), 1), (dict(d=80), 1), (dict(n=-1), 1), (dict(nt=-1), 1), (dict(rows=0), 1),
    (dict(pages=0), 1), (dict(kp=N), 1), (dict(vp=N), 1), (dict(ko=N), 1), (dict(vo=N), 1), (dict(tiles=N), 1),
    (dict(kp=ODD), 2), (dict(vp=ODD), 2), (dict(ko=ODD), 2), (dict(vo=ODD), 2), (dict(tiles=ODD), 2), (dict(sr=88), 2),
    (dict(oh=1284), 2), (dict(on=132), 2)])
def test_gather_refuses(bad, status):
    assert gather(**bad) == status


def rotate(pool=256, layers=1, hkv=2, d=128, rows=64, pages=4, sr=80, tiles=P, cols=4, nt=1, table=True, dtype=2, pools=True):
    ptrs = (ctypes.c_void_p * 1)(pool) if pools else None
    tab = (ctypes.c_float * 256)()
    return _lib.lib().tc_int4_rotate_keys(ptrs, layers, hkv, d, rows, pages, 10240, 5120, sr, tiles, cols, nt,
                                          ctypes.cast(tab, ctypes.POINTER(ctypes.c_float)) if table else None, dtype, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(layers=0), 1), (dict(layers=129), 1), (dict(hkv=0), 1), (dict(d=192), 1), (dict(rows=0), 1),
    (dict(pages=0), 1), (dict(nt=-1), 1), (dict(cols=2), 1), (dict(tiles=N), 1), (dict(pool=None), 1), (dict(pools=False), 1),
    (dict(table=False), 1), (dict(pool=264), 2), (dict(sr=72), 2)])
def test_rotate_refuses(bad, status):
    assert rotate(**bad) == status


def decode(q=P, k=P, v=P, out=P, b=2, hkv=2, g=4, d=128, n=5000, kb=160000, kh=80000, kn=80, scale=0.1, splits=0, dtype=2,
           ws=N, nb=0):
    return _lib.lib().tc_decode_attention_int4(q, k, v, out, b, hkv, g, d, n, N, 1024, 512, 128, kb, kh, kn, kb, kh, kn, 1024,
                                               512, 128, scale, splits, dtype, ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(b=0), 1), (dict(b=65536), 1), (dict(hkv=0), 1), (dict(g=0), 1), (dict(g=17), 1), (dict(d=96), 1),
    (dict(n=-1), 1), (dict(n=1 << 31), 1), (dict(splits=-1), 1), (dict(q=N), 1), (dict(k=N), 1), (dict(v=N), 1),
    (dict(out=N), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(k=ODD), 2), (dict(v=ODD), 2),
    (dict(kb=160008), 2), (dict(kh=80008), 2), (dict(kn=88), 2), (dict(), 4), (dict(ws=P, nb=100), 4),
    (dict(ws=ODD, nb=1 << 30), 2)])
def test_decode_refuses(bad, status):
    assert decode(**bad) == status


def paged(q=P, k=P, v=P, out=P, hkv=2, g=4, d=128, rows=64, pages=4, sr=80, tiles=P, cols=4, nt=200, scale=0.1, splits=0,
          dtype=2, ws=N, nb=0):
    return _lib.lib().tc_decode_attention_int4_paged(q, k, v, out, hkv, g, d, rows, pages, 10240, 5120, sr, tiles, cols, nt,
                                                     512, 128, 512, 128, scale, splits, dtype, ws, nb, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(hkv=0), 1), (dict(g=17), 1), (dict(d=96), 1), (dict(rows=0), 1), (dict(pages=0), 1),
    (dict(tiles=N), 1), (dict(cols=2), 1), (dict(nt=-1), 1), (dict(nt=1 << 26), 1), (dict(q=N), 1), (dict(k=N), 1),
    (dict(v=N), 1), (dict(out=N), 1), (dict(splits=-1), 1), (dict(scale=float("-inf")), 1), (dict(k=ODD), 2),
    (dict(v=ODD), 2), (dict(sr=88), 2), (dict(), 4)])
def test_paged_decode_refuses(bad, status):
    assert paged(**bad) == status


def test_decode_workspace():
    size = _lib.lib().tc_decode_attention_int4_workspace_size
    assert size(1, 8, 4, 128, 98304, 0) > size(1, 8, 4, 128, 1536, 0) > 0
    assert size(1, 8, 4, 128, 256, 0) == 0 == size(1, 8, 4, 128, 0, 0)  # one slice a head: nothing to join
    assert size(0, 8, 4, 128, 98304, 0) == 0 == size(1, 8, 17, 128, 98304, 0) == size(1, 8, 4, 96, 98304, 0)
    assert size(1, 8, 4, 128, 98304, -1) == 0 == size(1, 8, 4, 128, -1, 0)
    assert size(1, 8, 4, 128, 98304, 1 << 20) == size(1, 8, 4, 128, 98304, 128)


def gemv(x=P, codes=P, params=P, out=P, n=32, k=128, m=1, group=64, swiglu=0, dtype=2):
    return _lib.lib().tc_gemv_int4(x, codes, params, out, n, k, m, group, k, n, swiglu, dtype, N)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=0), 3), (dict(n=-1), 1), (dict(n=1 << 31), 1), (dict(k=0), 1), (dict(k=65537), 1), (dict(m=-1), 1),
    (dict(group=16), 1), (dict(group=0), 1), (dict(x=N), 1), (dict(codes=N), 1), (dict(params=N), 1), (dict(out=N), 1),
    (dict(codes=ODD), 2), (dict(params=ODD), 2)])
def test_gemv_refuses(bad, status):
    assert gemv(**bad) == status


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(1, 2, 32, 40, dtype=torch.uint8)
    slots = torch.zeros(4, 2, dtype=torch.int32)
    tiles = torch.zeros(1, 4, dtype=torch.int32)
    for call in (lambda: int4.write_int4(x, x, pool, pool, slots),
                 lambda: int4.append_rope_int4(x, x, x[0], x[0], pool, pool, slots, q=x),
                 lambda: int4.gather_int4(pool, pool, tiles, 4, torch.bfloat16),
                 lambda: int4.rotate_keys_int4([pool], tiles, 1, torch.ones(32), torch.bfloat16),
                 lambda: int4.decode_attention_int4(x[None], pool, pool, 0.1),
                 lambda: int4.decode_attention_int4(x, pool, pool, 0.1, tiles=tiles),
                 lambda: int4.gemv_int4(x[0], int4.quantize_weight(torch.ones(16, 64, dtype=torch.bfloat16)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_quantised_weights_on_the_host():
    for dtype in (torch.bfloat16, torch.float16):
        m = (0.02 * torch.randn(33, 130, generator=torch.Generator().manual_seed(0))).to(dtype)
        w = int4.quantize_weight(m, 32)
        assert w.codes.shape == (3, 3, 512) and w.params.shape == (3, 5, 8, 2, 2) and (w.n, w.k, w.group) == (33, 130, 32)
        pad = torch.cat((m, m[:, -1:].expand(-1, 30)), 1)
        codes, s, z = ref.quantise64(pad)
        want = s.double().repeat_interleave(32, 1) * (1 + codes.double() / 16) + z.double().repeat_interleave(32, 1)
        assert (int4.dequantize_weight(w).double() - want[:, :130]).abs().max() <= 2.0 ** -24
        # what lies behind the matrix is zero
        big = int4.Int4Weight(w.codes, w.params, 48, 192, 32)
        assert not big.codes[2].view(3, 8, 4, 2, 2, 4)[:, 1:, :, :, :].any() and not w.params[2, :, 1:].any()


@pytest.mark.parametrize("bad", [dict(w=torch.ones(4, dtype=torch.bfloat16)), dict(group=48),
                                 dict(w=torch.ones(0, 8, dtype=torch.bfloat16))])
def test_quantize_weight_refuses(bad):
    args = dict(w=torch.ones(4, 8, dtype=torch.bfloat16), group=64) | bad
    with pytest.raises(ValueError):
        int4.quantize_weight(**args)


def test_quantize_weight_refuses_other_types():
    with pytest.raises(TypeError):
        int4.quantize_weight(torch.ones(4, 8))
