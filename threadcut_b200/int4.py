"""KV cache rows and projection weights held in 4 bits.

threadcut keeps its cache and its weights in 16 bits; at long contexts a decode step is bound by exactly
those bytes (threadcut/engine.py:66-73, one model call a token). Here a group of neighbouring elements shares a
scale S and an offset z of the 16-bit type, and each element is a code of 0..15 that stands for
S (1 + code / 16) + z: 16 levels from the group's least element to its greatest, each element at the nearest one.

Cache: a row of d elements is `row_bytes(d)` = 5 d / 8 bytes: d / 2 bytes of codes (element e in byte e / 2, the
even one in the low half), then (S, z) of each 32 elements. Its values are rounded to the 16-bit type. Pools and
buffers are uint8 tensors [pages or batch, hkv, rows, row_bytes(d)], d 64, 128 or 256.

  append_rope_int4, write_int4   a step's keys and values into their slots (and its queries rotated)
  gather_int4                    rows back as contiguous 16-bit keys and values
  decode_attention_int4          attention of one query token a sequence over such rows
  rotate_keys_int4               a splice's re-rotation of keys, where they lie (threadcut/kv.py:28-41)

A group that holds an infinity or a NaN, or in fp16 magnitudes above 20,000, reads back as NaN.

Weights: `quantize_weight` lays a matrix out once as an Int4Weight, `gemv_int4` multiplies a few tokens with it.

Kernels: csrc/int4.cuh, csrc/int4_attn.cuh, csrc/int4_gemv.cuh. CUDA only."""
import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, cos_sin_table, dtype_code, lib, require_cuda, stream_ptr

__all__ = ["Int4Weight", "append_rope_int4", "decode_attention_int4", "dequantize_weight", "gather_int4", "gemv_int4",
           "quantize_weight", "rotate_keys_int4", "row_bytes", "write_int4"]

GROUP = 32  # elements of a cache row that share a scale
HEAD_SIZES = (64, 128, 256)
MAX_LAYERS = 128  # of a rotation's launch


def row_bytes(d):
    """Bytes of a cache row of d elements."""
    return d // 2 + d // 8


def _code16(dtype, what):
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"threadcut_b200.{what}: needs bf16 or fp16, got {dtype}")
    return _lib.DTYPE_CODE[dtype]


def _head_size(rows, what):
    for d in HEAD_SIZES:
        if rows.shape[-1] == row_bytes(d):
            return d
    raise ValueError(f"{what}: rows of {rows.shape[-1]} bytes; head sizes 64, 128 and 256 have "
                     f"{', '.join(str(row_bytes(d)) for d in HEAD_SIZES)}")


def _aligned(x, d):
    """Whether every row of x starts on a whole unit of copies (16 bytes, 8 for heads of 64)."""
    unit = 8 if d == 64 else 16
    return x.stride(-1) == 1 and x.data_ptr() % unit == 0 and all(s % unit == 0 for s in x.stride()[:-1])


def _pools(k_pool, v_pool, hkv, d, what):
    """The pools as they are written or read by slot: [pages, hkv, page_rows, row_bytes(d)], of equal strides."""
    if k_pool.dtype != torch.uint8 or v_pool.dtype != torch.uint8:
        raise TypeError(f"threadcut_b200.{what}: 4-bit pools are uint8, got {k_pool.dtype} and {v_pool.dtype}")
    if d not in HEAD_SIZES:
        raise ValueError(f"{what}: head size {d}: 4-bit rows have 64, 128 or 256 elements")
    if (k_pool.dim() != 4 or k_pool.shape[1] != hkv or k_pool.shape[3] != row_bytes(d) or v_pool.shape != k_pool.shape):
        raise ValueError(f"{what}: pools must be [pages, {hkv}, page_rows, {row_bytes(d)}], got {tuple(k_pool.shape)}, "
                         f"{tuple(v_pool.shape)}")
    if v_pool.stride() != k_pool.stride() or not _aligned(k_pool, d) or not _aligned(v_pool, d):
        raise ValueError(f"{what}: the pools must have equal strides and rows on {8 if d == 64 else 16}-byte boundaries")


def _tiles(tiles, cols, device, what):
    if tiles.device != device or tiles.dtype != torch.int32 or tiles.dim() != 2 or not tiles.is_contiguous():
        raise ValueError(f"{what}: tiles must be a contiguous int32 [tiles, {cols}] tensor on {device}")


def append_rope_int4(k, v, cos, sin, k_pool, v_pool, slots, *, q=None, q_norm=None, k_norm=None, eps=1e-6):
    """paged.append_rope into pools of 4-bit rows, in one launch (tc_int4_append_rope): normalises (optional) and
    rotates a step's queries and keys, rounds them to their type, and writes keys and values, quantised, to
    their slots.

    k, v: [hkv, t, d] (or [1, hkv, t, d]) raw projections, bf16 or fp16; q: [hq, t, d] or None; cos, sin: [t, rot] (or
    [1, t, rot]) of the data's dtype or fp32, rot <= d (elements from rot on pass through); q_norm / k_norm: RMSNorm
    weights [d] or None; any strides (a last dimension with gaps is copied). k_pool, v_pool: uint8 [pages, hkv,
    page_rows, row_bytes(d)]; slots: int32 [t, 2] (page, row), distinct; slots outside the pool are skipped. Returns the
    rotated queries, in q's shape and stored token by token ([t, hq, d]), or None."""
    what = "append_rope_int4"
    if (hb := _lib.host()) is not None:
        done, out = hb.int4_append(k, v, cos, sin, k_pool, v_pool, slots, q, q_norm, k_norm, float(eps))
        if done:
            return out
    return _append(what, k, v, cos, sin, k_pool, v_pool, slots, q, q_norm, k_norm, eps)


def write_int4(k, v, k_pool, v_pool, slots):
    """Writes keys and values k, v [hkv, t, d] (or [1, hkv, t, d]), quantised as they are, to their slots:
    append_rope_int4 without the rotation."""
    if (hb := _lib.host()) is not None:
        done, _ = hb.int4_append(k, v, None, None, k_pool, v_pool, slots, None, None, None, 0.0)
        if done:
            return
    _append("write_int4", k, v, None, None, k_pool, v_pool, slots, None, None, None, 0.0)


def _append(what, k, v, cos, sin, k_pool, v_pool, slots, q, q_norm, k_norm, eps):
    require_cuda(k, v, k_pool, v_pool, slots, *(x for x in (cos, sin, q, q_norm, k_norm) if x is not None), what=what)
    code = _code16(k.dtype, what)
    batched = k.dim() == 4
    if batched:
        if k.shape[0] != 1 or v.dim() != 4 or v.shape[0] != 1 or (q is not None and (q.dim() != 4 or q.shape[0] != 1)):
            raise ValueError(f"{what}: one sequence per call (batch 1)")
        k, v, q = k[0], v[0], q[0] if q is not None else None
    if k.dim() != 3 or v.shape != k.shape or (q is not None and q.dim() != 3):
        raise ValueError(f"{what}: expected k, v [hkv, t, d] and q [hq, t, d]; got {tuple(k.shape)}, {tuple(v.shape)}"
                         + (f", {tuple(q.shape)}" if q is not None else ""))
    hkv, t, d = k.shape
    hq = q.shape[0] if q is not None else 0
    if q is not None and tuple(q.shape) != (hq, t, d):
        raise ValueError(f"{what}: q {tuple(q.shape)} does not match k {tuple(k.shape)}")
    rot = 0
    if cos is not None:
        cos, sin = (x[0] if x.dim() == 3 and x.shape[0] == 1 else x for x in (cos, sin))
        rot = cos.shape[-1]
        if cos.dim() != 2 or cos.shape[0] != t or sin.shape != cos.shape or sin.dtype != cos.dtype:
            raise ValueError(f"{what}: cos/sin must be [{t}, rot] of one dtype, got {tuple(cos.shape)}, {tuple(sin.shape)}")
        if rot % 2 or not 2 <= rot <= d:
            raise ValueError(f"{what}: needs an even rot in [2, {d}], got {rot}")
        if cos.dtype != k.dtype and cos.dtype != torch.float32:
            raise TypeError(f"threadcut_b200.{what}: cos/sin must be {k.dtype} or fp32, got {cos.dtype}")
    _pools(k_pool, v_pool, hkv, d, what)
    if tuple(slots.shape) != (t, 2) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int32 [{t}, 2] tensor")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (tuple(w.shape) != (d,) or w.dtype != k.dtype):
            raise ValueError(f"{what}: {name} must be [{d}] of {k.dtype}")
    for x in (v,) if q is None else (v, q):
        if x.dtype != k.dtype:
            raise TypeError(f"threadcut_b200.{what}: dtype mismatch {k.dtype} vs {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"{what}: needs eps >= 0, got {eps}")
    k, v, q, cos, sin, q_norm, k_norm = (x if x is None or x.stride(-1) == 1 else x.contiguous()
                                         for x in (k, v, q, cos, sin, q_norm, k_norm))
    out = torch.empty((t, hq, d), dtype=k.dtype, device=k.device).transpose(0, 1) if q is not None else None

    def ptr(x):
        return None if x is None else x.data_ptr()

    def strides(x):
        return (0, 0) if x is None else x.stride()[:2]

    with torch.cuda.device(k.device):
        st = lib().tc_int4_append_rope(
            ptr(q), ptr(k), ptr(v), ptr(out), ptr(k_pool), ptr(v_pool), hq, hkv, d, t, *strides(q), *strides(k), *strides(v),
            *strides(out), ptr(q_norm), ptr(k_norm), float(eps), ptr(cos), ptr(sin), rot, strides(cos)[0], strides(sin)[0],
            code if cos is None else _lib.DTYPE_CODE[cos.dtype], k_pool.shape[2], k_pool.shape[0], *k_pool.stride()[:3],
            ptr(slots), code, stream_ptr(k.device))
    check("tc_int4_append_rope", st)
    return out[None] if batched and out is not None else out


def gather_int4(k_pool, v_pool, tiles, n, dtype):
    """Rows of 4-bit pools as contiguous keys and values [hkv, n, d] of `dtype`, the 16-bit type they were written from
    (tc_int4_gather). tiles: int32 [T, 4] (page, first row, rows <= 32, position of the first row in the outputs);
    positions that no tile covers are left unset, and rows outside the pool or the outputs are skipped."""
    what = "gather_int4"
    if (hb := _lib.host()) is not None and (out := hb.int4_gather(k_pool, v_pool, tiles, int(n), dtype)) is not None:
        return out
    require_cuda(k_pool, v_pool, tiles, what=what)
    code = _code16(dtype, what)
    d = _head_size(k_pool, what)
    hkv = k_pool.shape[1] if k_pool.dim() == 4 else 0
    _pools(k_pool, v_pool, hkv, d, what)
    _tiles(tiles, 4, k_pool.device, what)
    if tiles.shape[1] != 4 or tiles.data_ptr() % 16 or n < 0:
        raise ValueError(f"{what}: needs tiles [T, 4] on a 16-byte boundary and n >= 0, got {tuple(tiles.shape)} and {n}")
    k = torch.empty((hkv, n, d), dtype=dtype, device=k_pool.device)
    v = torch.empty_like(k)
    with torch.cuda.device(k_pool.device):
        check("tc_int4_gather", lib().tc_int4_gather(
            k_pool.data_ptr(), v_pool.data_ptr(), k.data_ptr(), v.data_ptr(), hkv, d, n, k.stride(0), k.stride(1),
            k_pool.shape[2], k_pool.shape[0], *k_pool.stride()[:3], tiles.data_ptr(), tiles.shape[0], code,
            stream_ptr(k_pool.device)))
    return k, v


def rotate_keys_int4(k_pools, tiles, delta, inv_freq, dtype):
    """Moves the keys that `tiles` lists by `delta` positions, in place and in every pool (one a layer), in one launch for
    128 layers (tc_int4_rotate_keys): each row's values, rotated as kv.shift_keys rotates them and quantised again. tiles: int32
    [T, >= 3] (page, first row, rows <= 32, ...), no row twice; rows outside the pools are skipped. inv_freq:
    [d / 2]. dtype: the 16-bit type the rows were written from. All pools of one shape and strides."""
    what = "rotate_keys_int4"
    k_pools = list(k_pools)
    if not k_pools:
        return
    if (hb := _lib.host()) is not None and hb.int4_rotate(k_pools, tiles, int(delta), inv_freq, dtype):
        return
    require_cuda(*k_pools, tiles, what=what)
    code = _code16(dtype, what)
    first = k_pools[0]
    d = _head_size(first, what)
    for p in k_pools:
        _pools(first, p, first.shape[1] if first.dim() == 4 else 0, d, what)
    _tiles(tiles, 3, first.device, what)
    if tiles.shape[1] < 3:
        raise ValueError(f"{what}: tiles must have at least 3 columns, got {tuple(tiles.shape)}")
    if inv_freq.numel() * 2 != d:
        raise ValueError(f"{what}: inv_freq has {inv_freq.numel()} entries, keys need {d // 2}")
    tab, tab_ptr = cos_sin_table(int(delta), inv_freq)
    with torch.cuda.device(first.device):
        for i in range(0, len(k_pools), MAX_LAYERS):
            some = k_pools[i:i + MAX_LAYERS]
            check("tc_int4_rotate_keys", lib().tc_int4_rotate_keys(
                (ctypes.c_void_p * len(some))(*[p.data_ptr() for p in some]), len(some), first.shape[1], d, first.shape[2],
                first.shape[0], *first.stride()[:3], tiles.data_ptr(), tiles.shape[1], tiles.shape[0], tab_ptr, code,
                stream_ptr(first.device)))
    del tab  # the table is copied into the launch parameters


def decode_attention_int4(q, k, v, scale, lengths=None, *, tiles=None, splits=None):
    """flash_decode.decode_attention_batched over rows of 4 bits: softmax(scale q k^T) v in fp32 over the values that
    the rows stand for. bf16 or fp16 queries, the type the rows were written from; up to 16 query heads a KV head.

    Contiguous: q [b, hkv, g, d], k, v uint8 [b, hkv, n, row_bytes(d)] (views of larger buffers are fine; rows that do
    not start on 16-byte boundaries, 8 for d = 64, are copied); lengths: int32 CUDA [b], the rows of each sequence that
    count, clamped into [0, n] (None: all). Returns [b, hkv, g, d]; a sequence of no rows gives zeros. q [hkv, g, d] and
    k, v [hkv, n, row_bytes(d)] are one sequence, whose result is [hkv, g, d].
    Paged: q [hkv, g, d], k, v pools [pages, hkv, page_rows, row_bytes(d)], tiles int32 [T, >= 3] (page, first row,
    rows <= 32, ...) in order; tiles outside the pool are skipped. Returns [hkv, g, d].
    splits forces the number of slices a KV head's rows are split into."""
    what = "decode_attention_int4"
    if (hb := _lib.host()) is not None:
        out = hb.int4_decode(q, k, v, float(scale), lengths, tiles, int(splits or 0))
        if out is not None:
            return out
    require_cuda(q, k, v, *(x for x in (lengths, tiles) if x is not None), what=what)
    code = _code16(q.dtype, what)
    if k.dtype != torch.uint8 or v.dtype != torch.uint8:
        raise TypeError(f"threadcut_b200.{what}: rows of 4 bits are uint8, got {k.dtype} and {v.dtype}")
    if not -float("inf") < scale < float("inf"):
        raise ValueError(f"{what}: needs a finite scale, got {scale}")
    if splits is not None and not 0 <= splits <= 65535:
        raise ValueError(f"{what}: needs splits >= 0, got {splits}")
    single = tiles is None and q.dim() == 3
    if single:
        q, k, v = q[None], k[None], v[None]
    if q.dim() != (3 if tiles is not None else 4) or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{what}: expected q [b, hkv, g, d] and k, v [b, hkv, n, bytes], or q [hkv, g, d] with pools and "
                         f"tiles; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    hkv, g, d = q.shape[-3:]
    if d not in HEAD_SIZES or not 1 <= g <= 16:
        raise ValueError(f"{what}: needs heads of 64, 128 or 256 and at most 16 query heads a KV head, got {d} and {g}")
    if k.shape[1] != hkv or k.shape[3] != row_bytes(d) or (tiles is None and k.shape[0] != q.shape[0]):
        raise ValueError(f"{what}: k, v {tuple(k.shape)} do not match q {tuple(q.shape)}")
    q = q if q.stride(-1) == 1 else q.contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out[0] if single else out
    L, s = lib(), int(splits or 0)
    with torch.cuda.device(q.device):
        if tiles is not None:
            if lengths is not None:
                raise ValueError(f"{what}: tiles say which rows count, lengths do not go with them")
            _pools(k, v, hkv, d, what)
            _tiles(tiles, 3, q.device, what)
            if tiles.shape[1] < 3:
                raise ValueError(f"{what}: tiles must have at least 3 columns, got {tuple(tiles.shape)}")
            nt = tiles.shape[0]
            ws = _workspace(1, hkv, g, d, 32 * nt, s, q.device)
            st = L.tc_decode_attention_int4_paged(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), hkv, g, d, k.shape[2], k.shape[0], *k.stride()[:3],
                tiles.data_ptr(), tiles.shape[1], nt, *q.stride()[:2], *out.stride()[:2], float(scale), s, code,
                ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream_ptr(q.device))
            check("tc_decode_attention_int4_paged", st)
            return out
        b, n = q.shape[0], k.shape[2]
        k, v = (x if _aligned(x, d) else x.clone(memory_format=torch.contiguous_format) for x in (k, v))
        if lengths is not None:
            lengths = lengths.to(torch.int32).contiguous()
            if lengths.shape != (b,):
                raise ValueError(f"{what}: lengths must be [{b}]")
        ws = _workspace(b, hkv, g, d, n, s, q.device)
        st = L.tc_decode_attention_int4(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, hkv, g, d, n,
            lengths.data_ptr() if lengths is not None else None, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
            *out.stride()[:3], float(scale), s, code, ws.data_ptr() if ws is not None else None,
            ws.numel() if ws is not None else 0, stream_ptr(q.device))
    check("tc_decode_attention_int4", st)
    return out[0] if single else out


def _workspace(b, hkv, g, d, rows, splits, device):
    nb = lib().tc_decode_attention_int4_workspace_size(b, hkv, g, d, rows, splits)
    return _lib.decode_workspace(b * hkv, device, nb) if nb else None


class Int4Weight(NamedTuple):
    """A weight matrix [n, k] in 4 bits, laid out for gemv_int4: codes uint8 [ceil(n / 16), ceil(k / 64), 512] and
    params [ceil(n / 16), ceil(k / group), 8, 2, 2] of the 16-bit type of the tokens.

    codes: tiles of 16 rows and 64 columns. Bytes 16 (4 r + c) .. + 15 of a tile, r < 8, c < 4, are four little-endian
    words: (row r, columns 8 c .. 8 c + 7), (row r + 8, the same), (row r, columns 32 + 8 c ..), (row r + 8, the same);
    of a word's codes, number j is column 2 j and number 4 + j column 2 j + 1. params: (S, z) of rows r and r + 8.
    Both are 0 behind row n and column k. A code stands for S (1 + code / 16) + z, not rounded further.
    The tensors stay as they are: gemv_int4 may read them while the kernel ahead of it in the stream is still running, so
    weights that change become a new Int4Weight (or wait for the kernel that writes them before the next product)."""
    codes: torch.Tensor
    params: torch.Tensor
    n: int
    k: int
    group: int


_WORD = (0, 4, 1, 5), (2, 6, 3, 7)  # columns in the low and in the high halves of a word's bytes


def quantize_weight(w, group=64):
    """A weight matrix w [n, k] (bf16 or fp16, rows of output features as torch.nn.Linear keeps them) as an Int4Weight
    on w's device, `group` (32, 64 or 128) neighbours of a row sharing a scale: 4.5 bits an element at 64."""
    what = "quantize_weight"
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"{what}: expected a matrix, got {tuple(w.shape)}")
    if group not in (32, 64, 128):
        raise ValueError(f"{what}: groups have 32, 64 or 128 columns, got {group}")
    _code16(w.dtype, what)
    w = w.detach()
    n, k = w.shape
    rows, cols, groups = -(-n // 16), -(-k // 64), -(-k // group)
    codes = torch.empty((rows, cols, 512), dtype=torch.uint8, device=w.device)
    params = torch.zeros((rows, groups, 8, 2, 2), dtype=w.dtype, device=w.device)
    some = max(1, 2 ** 20 // k)
    for r0 in range(0, rows, some):  # pieces: the steps below take about 30 bytes an element
        r1 = min(rows, r0 + some)
        piece = w[16 * r0:16 * r1].float()
        m = piece.shape[0]
        # the last group's extremes are those of its own columns
        pad = groups * group - k
        g = torch.cat((piece, piece[:, -1:].expand(m, pad)), 1).view(m, groups, group)
        lo, hi = g.amin(-1), g.amax(-1)
        scale = ((hi - lo) / torch.full_like(hi, 0.9375)).to(w.dtype)  # (by a number: a product with its reciprocal on CUDA)
        zero = (lo - scale.float()).to(w.dtype)
        scale.masked_fill_(~zero.isfinite(), float("nan"))  # (a finite S would leave infinities that look like data)
        s, z = scale.double().unsqueeze(-1), zero.double().unsqueeze(-1)
        c = ((g.double() - z) / s * 16 - 16).round().clamp(0, 15).masked_fill(s == 0, 0).nan_to_num(0).to(torch.uint8)
        full = torch.zeros((16 * (r1 - r0), 64 * cols), dtype=torch.uint8, device=w.device)
        full[:m, :k] = c.view(m, -1)[:, :k]
        x = full.view(r1 - r0, 2, 8, cols, 2, 4, 8).permute(0, 3, 2, 5, 4, 1, 6)
        codes[r0:r1] = (x[..., _WORD[0]] | (x[..., _WORD[1]] << 4)).reshape(r1 - r0, cols, 512)
        both = torch.zeros((16 * (r1 - r0), groups, 2), dtype=w.dtype, device=w.device)
        both[:m] = torch.stack((scale, zero), -1)
        params[r0:r1] = both.view(r1 - r0, 2, 8, groups, 2).permute(0, 3, 2, 1, 4)
    if w.is_cuda and not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(w.device).synchronize()  # products do not wait for the kernel that wrote their weights
    return Int4Weight(codes, params, n, k, group)


def dequantize_weight(w):
    """The matrix [n, k] that an Int4Weight stands for, in fp32."""
    rows, cols, _ = w.codes.shape
    x = w.codes.view(rows, cols, 8, 4, 2, 2, 4)
    out = torch.empty((rows, cols, 8, 4, 2, 2, 8), dtype=torch.float32, device=w.codes.device)
    out[..., _WORD[0]], out[..., _WORD[1]] = (x & 15).float(), (x >> 4).float()
    codes = out.permute(0, 5, 2, 1, 4, 3, 6).reshape(16 * rows, 64 * cols)[:w.n, :w.k]
    p = w.params.float().permute(0, 3, 2, 1, 4).reshape(16 * rows, -1, 2)[:w.n]
    s, z = (p[..., i].repeat_interleave(w.group, 1)[:, :w.k] for i in (0, 1))
    return s * (1 + codes / 16) + z


def gemv_int4(x, w, *, swiglu=False):
    """x [..., k] times the transpose of an Int4Weight [n, k] -> [..., n] (tc_gemv_int4), sums in fp32: the
    projections of a decode step. x: bf16 or fp16, the type of w's params. Up to 32 tokens read the weights once (as
    many as fit shared memory with their k columns: 28 at 2,560, 7 at 12,288); more are taken in turns, each of which reads
    the weights again: this is for a few tokens, not for a prompt.
    One or two tokens, of a call or left over by its turns, enter as whole numbers of 20 bits: each x is off by at most 2^-20 of the
    largest |x| of its 64 columns. A token's result may so differ in its last bits with how many share its call.
    swiglu: x is [..., 2 k] (gate | up) and the tokens are silu(gate) * up, rounded after each step as
    transformers rounds them, computed on the way."""
    what = "gemv_int4"
    if (hb := _lib.host()) is not None and (out := hb.int4_gemv(x, w.codes, w.params, w.n, w.k, w.group, swiglu)) is not None:
        return out
    require_cuda(x, w.codes, w.params, what=what)
    code = _code16(x.dtype, what)
    if w.params.dtype != x.dtype or w.codes.dtype != torch.uint8:
        raise TypeError(f"threadcut_b200.{what}: {x.dtype} tokens need params of that type and uint8 codes, got "
                        f"{w.params.dtype} and {w.codes.dtype}")
    rows, cols = -(-w.n // 16), -(-w.k // 64)
    if w.k > 65536:
        raise ValueError(f"{what}: rows of at most 65536 columns, got {w.k}")
    if (w.n < 1 or w.k < 1 or w.group not in (32, 64, 128) or tuple(w.codes.shape) != (rows, cols, 512)
            or tuple(w.params.shape) != (rows, -(-w.k // w.group), 8, 2, 2)):
        raise ValueError(f"{what}: codes {tuple(w.codes.shape)} and params {tuple(w.params.shape)} are not those of a matrix "
                         f"[{w.n}, {w.k}] in groups of {w.group}")
    if not w.codes.is_contiguous() or not w.params.is_contiguous() or (w.codes.data_ptr() | w.params.data_ptr()) % 16:
        raise ValueError(f"{what}: codes and params must be contiguous and on 16-byte boundaries")
    wide = 2 * w.k if swiglu else w.k
    if x.dim() < 1 or x.shape[-1] != wide:
        raise ValueError(f"{what}: tokens of {wide} elements expected, got {tuple(x.shape)}")
    x2 = x.reshape(-1, wide)
    x2 = x2 if x2.stride(1) == 1 else x2.contiguous()
    m = x2.shape[0]
    out = torch.empty((*x.shape[:-1], w.n), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        check("tc_gemv_int4", lib().tc_gemv_int4(
            x2.data_ptr(), w.codes.data_ptr(), w.params.data_ptr(), out.data_ptr(), w.n, w.k, m, w.group, x2.stride(0), w.n,
            int(swiglu), code, stream_ptr(x.device)))
    return out
