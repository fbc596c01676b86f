"""GQA prefill attention on the B200 tensor cores (tcgen05) — the prefill branch of
threadcut/attention.py:43-46 without expanding K/V.

`prefill_attention(query, key, value, scale)`: query [1, hq, lq, d], key/value [1, hkv, lk, d] with
hq = 4*hkv and d = 128 (bf16 or fp16, CUDA). Query position p (of the lq newest tokens) attends to
keys [0, lk - lq + p], the causal mask of a prefill over a cache that ends with those tokens.
Returns [1, lq, hq, d] contiguous (the layout the attention plugin returns). `supported()` says
whether the kernel takes the inputs; the plugin keeps torch SDPA for everything else.
"""
import torch

from . import _lib
from ._lib import check, dtype_code, lib, require_cuda, rows16, stream_ptr, workspaces

__all__ = ["prefill_attention", "prefill_attention_window", "supported", "causal_offset_mask"]


def supported(query, key, value):
    return (query.is_cuda and key.is_cuda and value.is_cuda and query.dim() == 4 and key.dim() == 4
            and query.shape[0] == 1 and key.shape[0] == 1 and query.shape[-1] == 128
            and query.dtype in (torch.bfloat16, torch.float16) and key.dtype == query.dtype
            and value.dtype == query.dtype and key.shape[1] * 4 == query.shape[1]
            and value.shape == key.shape and 1 <= query.shape[2] <= key.shape[2])


def causal_offset_mask(lq, lk, device):
    """The boolean SDPA mask [lq, lk] the kernel implements: True where key j <= lk - lq + p."""
    p = torch.arange(lq, device=device)[:, None]
    j = torch.arange(lk, device=device)[None, :]
    return j <= (lk - lq) + p


def prefill_attention(query, key, value, scale, *, splits=None):
    what = "prefill_attention"
    require_cuda(query, key, value, what=what)
    if not supported(query, key, value):
        raise ValueError(f"{what}: needs query [1, 4*hkv, lq, 128], key/value [1, hkv, lk, 128] with lq <= lk, "
                         f"bf16/fp16; got {tuple(query.shape)}, {tuple(key.shape)}, {query.dtype}")
    _, hq, lq, d = query.shape
    hkv, lk = key.shape[1], key.shape[2]
    q, k, v = query[0], key[0], value[0]
    if q.stride(-1) != 1:
        q = q.contiguous()
    if k.stride(-1) != 1:
        k = k.contiguous()
    if v.stride(-1) != 1:
        v = v.contiguous()
    out = torch.empty((1, lq, hq, d), dtype=query.dtype, device=query.device)
    L = lib()
    s = int(splits or 0)
    with torch.cuda.device(query.device):
        nb = L.tc_prefill_workspace_size(hq, hkv, lq, lk, s)
        ws = workspaces.get("prefill", query.device, nb) if nb else None
        st = L.tc_prefill_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), hq, hkv, lq, lk, d, q.stride(0), q.stride(1),
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(1), out.stride(2), float(scale), s,
            _lib.DTYPE_CODE[query.dtype], ws.data_ptr() if ws is not None else None, nb, stream_ptr(query.device))
    check(what, st)
    return out


def prefill_attention_window(query, key, value, scale, window, sinks=0, *, splits=None):
    """Causal attention of a chunk over the cache that ends with it, with a sliding window and sinks: query
    [b, hq, lq, d], key/value [b, hkv, lk, d] (hq a multiple of hkv, d <= 256, any dtype of the package).
    Query position p sees the keys j <= lk - lq + p with j < sinks or j > lk - lq + p - window (window >= 1
    counts the query's own token). Returns [b, lq, hq, d] contiguous. The softmax weights meet the values rounded to the
    16-bit type, as in prefill_attention.

    The tensor cores take 16-bit types, d of 64 or 128, up to 128 query heads per KV head, scale > 0, and keys and values
    that are not broadcast; a tensor whose rows do not start on 16-byte boundaries, and a broadcast query, is copied
    first. Anything else runs on a plain kernel, a CTA a query row, many times slower."""
    what = "prefill_attention_window"
    hb = _lib.host()
    if hb is not None:
        out = hb.window_prefill(query, key, value, float(scale), int(window), int(sinks), int(splits or 0))
        if out is not None:
            return out
    require_cuda(query, key, value, what=what)
    if query.dim() != 4 or key.dim() != 4 or value.shape != key.shape:
        raise ValueError(f"{what}: expected query [b, hq, lq, d], key/value [b, hkv, lk, d]; got {tuple(query.shape)}, "
                         f"{tuple(key.shape)}, {tuple(value.shape)}")
    b, hq, lq, d = query.shape
    hkv, lk = key.shape[1], key.shape[2]
    if key.shape[0] != b or key.shape[3] != d or hkv < 1 or hq % hkv or not 1 <= lq <= lk:
        raise ValueError(f"{what}: key {tuple(key.shape)} does not fit query {tuple(query.shape)} (1 <= lq <= lk, hq a "
                         "multiple of hkv)")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError(f"threadcut_b200.{what}: dtype mismatch {query.dtype} vs {key.dtype}/{value.dtype}")
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"{what}: needs window >= 1 and sinks >= 0, got {window} and {sinks}")
    window, sinks = min(window, lk), min(sinks, lk)
    code = dtype_code(query, what)
    q, (k, v) = rows16(query), (x if x.stride(-1) == 1 else x.contiguous() for x in (key, value))
    if code != _lib.DTYPE_CODE[torch.float32] and d in (64, 128):
        # off a 16-byte boundary: a copy costs its bytes, the plain kernel a hundred times that. A broadcast tensor
        # stays: its copy could be any size.
        k, v = (x if any(s == 0 and n > 1 for n, s in zip(x.shape, x.stride())) else rows16(x) for x in (k, v))
    dev = query.device
    out = torch.empty((b, lq, hq, d), dtype=query.dtype, device=dev)
    L = lib()
    s = int(splits or 0)
    with torch.cuda.device(dev):
        nb = L.tc_prefill_window_workspace_size(b, hq, hkv, lq, lk, d, window, sinks, s)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        st = L.tc_prefill_attention_window(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, hq, hkv, lq, lk, d, window, sinks,
            *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], float(scale), s, code,
            ws.data_ptr() if ws is not None else None, nb, stream_ptr(dev))
    check("tc_prefill_attention_window", st)
    return out
