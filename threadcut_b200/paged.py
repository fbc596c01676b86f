"""Paged K/V cache: the layout threadcut names as its next step (README.md:141-144, "drop B by
freeing pages, rotate C in place with no move").

threadcut's splice (kv.py:28-41, 83-92) turns A.B.C into A.C by copying C's K and V rows down to
position a and re-rotating the keys by -(c0 - a) positions. Here every layer keeps its K and V in
pools of fixed-size pages, and a sequence is an ordered list of runs (page, first row, rows). The
splice then

  * cuts the run list at a, c0 and c0 + c and keeps A's and C's runs, in that order;
  * returns every page that no kept run touches to the free list (B and the stale tail);
  * re-rotates C's keys where they lie (tc_paged_rotate_keys, every layer in one launch).

No row of K or V moves, and V is not touched at all: the splice costs a read and a write of C's
keys instead of a read and a write of C's keys and values. Decode reads the pages through a tile
table (tc_decode_attention_paged); appends write into the free rows after the last run and then
into fresh pages (tc_paged_write, or fused into the decode launch for one token).

The logical order of the runs is always the reference cache's token order, and rows inside a page
are only ever written in that order, so the rows after the last run's end in its page hold no
live token and the next append may take them.
"""
import ctypes

import numpy as np
import torch

from . import _lib, int4
from ._lib import check, dtype_code, lib, require_cuda, rows16, stream_ptr, workspaces
from .match import Split
from .prefill import prefill_attention, prefill_attention_window

__all__ = ["PageTable", "PagedKV", "PagedKVInt4", "TILE_ROWS", "append_rope"]

TILE_ROWS = 32  # rows per tile-table entry (the decode kernel's tile height)


class PageTable:
    """Host bookkeeping of one paged sequence: free pages, the run list, slot allocation, splice and
    the decode tile table. No device work; PagedKV drives the kernels with what this returns.

    Runs are an int64 array [R, 3] (page, first row, rows) and the tile table an int32 array
    [T, 3] kept in step with them in a growable buffer: an append touches only the tail of the
    table (tiles from `dirty` on changed; a one-token append is O(1)), and a splice keeps the tiles
    of every run it does not cut and re-tiles only the runs cut at a, c0 and c0 + c."""

    def __init__(self, num_pages, page_rows):
        if page_rows < TILE_ROWS:
            raise ValueError(f"page_rows must be >= {TILE_ROWS}")
        self.num_pages = int(num_pages)
        self.page_rows = int(page_rows)
        self.free = list(range(self.num_pages - 1, -1, -1))  # stack: page 0 is taken first
        self._runs = np.zeros((0, 3), np.int64)
        self._tbuf = np.zeros((64, 3), np.int32)
        self._nt = 0
        self.n = 0
        self.version = 0  # bumped whenever the run list changes
        self.dirty = 0    # tiles [dirty, T) changed since the last mark_clean()

    @property
    def runs(self):
        return self._runs.tolist()

    def tiles(self):
        return self._tbuf[:self._nt]

    def mark_clean(self):
        self.dirty = self._nt

    def _set_tiles(self, keep, tail):
        """Tile table = the first `keep` tiles + `tail`."""
        need = keep + tail.shape[0]
        if need > self._tbuf.shape[0]:
            buf = np.zeros((max(need, 2 * self._tbuf.shape[0]), 3), np.int32)
            buf[:keep] = self._tbuf[:keep]
            self._tbuf = buf
        self._tbuf[keep:need] = tail
        self._nt = need
        self.dirty = min(self.dirty, keep)

    # ---------------------------------------------------------------- allocation
    def reserve(self, t):
        """Slots (page, row) for t new tokens at the end of the sequence, in order: first the rows
        after the last run in its page, then fresh pages. Returns an int32 array [t, 2]."""
        t = int(t)
        P = self.page_rows
        out = np.empty((t, 2), dtype=np.int32)
        if t == 0:
            return out
        runs = self._runs
        room = P - int(runs[-1, 1] + runs[-1, 2]) if runs.shape[0] else 0
        if t == 1 and room >= 1:
            # one-token step inside the last page: extend the last run and its last tile
            page, r = int(runs[-1, 0]), int(runs[-1, 1] + runs[-1, 2])
            out[0, 0], out[0, 1] = page, r
            runs[-1, 2] += 1
            last = self._tbuf[self._nt - 1]
            if int(last[2]) < TILE_ROWS and int(last[0]) == page and int(last[1] + last[2]) == r:
                last[2] += 1
                self.dirty = min(self.dirty, self._nt - 1)
            else:
                self._set_tiles(self._nt, np.asarray([[page, r, 1]], np.int32))
            self.n += 1
            self.version += 1
            return out
        first = min(room, t)
        n_new = -(-(t - first) // P)
        if n_new > len(self.free):
            raise MemoryError("PagedKV: no free page left in the pool")
        retile_run = runs.shape[0]  # runs from this index on are (re)tiled below
        keep = self._nt             # tiles before this index stay as they are
        if first > 0:
            page, r0 = int(runs[-1, 0]), int(runs[-1, 1] + runs[-1, 2])
            out[:first, 0] = page
            out[:first, 1] = np.arange(r0, r0 + first, dtype=np.int32)
            keep = self._nt - int(-(-runs[-1, 2] // TILE_ROWS))  # the last run's tiles are redone
            retile_run = runs.shape[0] - 1
            runs[-1, 2] += first
        if n_new:
            pages = [self.free.pop() for _ in range(n_new)]
            counts = np.full(n_new, P, np.int64)
            counts[-1] = (t - first) - P * (n_new - 1)
            new = np.stack([np.asarray(pages, np.int64), np.zeros(n_new, np.int64), counts], axis=1)
            out[first:, 0] = np.repeat(np.asarray(pages, np.int32), P)[:t - first]
            out[first:, 1] = np.tile(np.arange(P, dtype=np.int32), n_new)[:t - first]
            self._runs = np.concatenate((runs, new))
        self._set_tiles(keep, self.tiles_of(self._runs[retile_run:]))
        self.n += t
        self.version += 1
        return out

    # ---------------------------------------------------------------- splice
    def _index(self):
        cnt = self._runs[:, 2]
        end = np.cumsum(cnt)
        nt = (cnt + TILE_ROWS - 1) // TILE_ROWS
        tile0 = np.concatenate(([0], np.cumsum(nt)))
        return end, end - cnt, tile0

    def _span(self, lo, hi, end, start, tile0):
        """Runs covering logical tokens [lo, hi) cut at the ends, and their tiles: the tiles of runs
        kept whole are copied from the current table, cut runs are re-tiled."""
        if hi <= lo or self._runs.shape[0] == 0:
            return np.zeros((0, 3), np.int64), np.zeros((0, 3), np.int32)
        i0 = int(np.searchsorted(end, lo, side="right"))
        i1 = int(np.searchsorted(start, hi, side="left"))
        sel = self._runs[i0:i1].copy()
        cut_lo = lo - int(start[i0])
        cut_hi = int(end[i1 - 1]) - hi
        if cut_lo > 0:
            sel[0, 1] += cut_lo
            sel[0, 2] -= cut_lo
        if cut_hi > 0:
            sel[-1, 2] -= cut_hi
        k = sel.shape[0]
        a = 1 if cut_lo > 0 else 0                 # runs [a, b) of sel keep their old tiles
        b = k - 1 if (cut_hi > 0 and k - 1 >= a) else k
        parts = []
        if a:
            parts.append(self.tiles_of(sel[:1]))
        if b > a:
            parts.append(self._tbuf[tile0[i0 + a]:tile0[i0 + b]])
        if b < k:
            parts.append(self.tiles_of(sel[b:]))
        return sel, np.concatenate(parts) if parts else np.zeros((0, 3), np.int32)

    def _cut(self, lo, hi):
        """Runs covering logical tokens [lo, hi), split at the ends (int64 [k, 3])."""
        end, start, tile0 = self._index()
        return self._span(lo, hi, end, start, tile0)[0]

    def splice(self, s: Split):
        """Keep A = [0, a) and C = [c0, c0 + c) (threadcut/kv.py:28-33 semantics, everything after C
        dropped). Returns (C's runs in the new list as [k, 3] int64, pages freed)."""
        a, c0, c = int(s.a), int(s.c0), int(s.c)
        if not (0 <= a <= c0 and c >= 0 and c0 + c <= self.n):
            raise ValueError(f"splice {s} outside a sequence of {self.n} tokens")
        end, start, tile0 = self._index()
        runs_a, tiles_a = self._span(0, a, end, start, tile0)
        runs_c, tiles_c = self._span(c0, c0 + c, end, start, tile0)
        new = np.concatenate((runs_a, runs_c))
        old_used = np.zeros(self.num_pages, bool)
        old_used[self._runs[:, 0]] = True
        old_used[new[:, 0]] = False
        dropped = np.flatnonzero(old_used).tolist()
        self.free.extend(reversed(dropped))
        self._runs = new
        self._set_tiles(0, np.concatenate((tiles_a, tiles_c)))
        self.n = a + c
        self.version += 1
        return runs_c, dropped

    def truncate(self, n):
        """Keep the first n tokens (a crop), freeing pages no longer used."""
        n = int(n)
        if n >= self.n:
            return []
        return self.splice(Split(n, n, 0))[1]

    # ---------------------------------------------------------------- tables
    @staticmethod
    def tiles_of(runs):
        """Tile table [n_tiles, 3] int32 (page, first row, rows <= TILE_ROWS) covering `runs`."""
        runs = np.asarray(runs, np.int64).reshape(-1, 3)
        if runs.shape[0] == 0:
            return np.zeros((0, 3), np.int32)
        nt = (runs[:, 2] + TILE_ROWS - 1) // TILE_ROWS
        idx = np.repeat(np.arange(runs.shape[0]), nt)
        off = (np.arange(idx.shape[0]) - np.repeat(np.cumsum(nt) - nt, nt)) * TILE_ROWS
        sel = runs[idx]
        out = np.empty((idx.shape[0], 3), np.int32)
        out[:, 0] = sel[:, 0]
        out[:, 1] = sel[:, 1] + off
        out[:, 2] = np.minimum(TILE_ROWS, sel[:, 2] - off)
        return out

    def window_tiles(self, window, sinks):
        """Tile table of the rows a windowed decode reads: tokens [0, sinks) and [n - window, n), or every
        token where the two meet."""
        lo = self.n - window
        if lo <= sinks:
            return self.tiles()
        end, start, tile0 = self._index()
        return np.concatenate((self._span(0, sinks, end, start, tile0)[1],
                               self._span(lo, self.n, end, start, tile0)[1]))

    def positions(self):
        """(page, row) of every logical token, int64 [n, 2] (for gathers and checks)."""
        runs = self._runs
        if runs.shape[0] == 0:
            return np.zeros((0, 2), np.int64)
        cnt = runs[:, 2]
        idx = np.repeat(np.arange(runs.shape[0]), cnt)
        k = np.arange(idx.shape[0]) - np.repeat(np.cumsum(cnt) - cnt, cnt)
        return np.stack((runs[idx, 0], runs[idx, 1] + k), axis=1)


def append_rope(k, v, cos, sin, k_pool, v_pool, slots, *, q=None, q_norm=None, k_norm=None, eps=1e-6):
    """Normalises (optional) and rotates a step's queries and keys and writes keys and values to
    their slots of one layer's pools, in one launch (tc_paged_append_rope).

    k, v: [hkv, t, d] (or [1, hkv, t, d]) raw projections; q: [hq, t, d] or None; cos, sin: [t, rot]
    (or [1, t, rot]: transformers' position_embeddings) of the data's dtype or fp32, rot <= d (elements
    from rot on pass through); q_norm / k_norm: RMSNorm weights [d] or None. k_pool, v_pool:
    [pages, hkv, page_rows, d]; slots: int32 [t, 2] (page, row), distinct (PagedKV.reserve). Any
    strides with a contiguous last dimension. Returns the rotated queries, in q's shape and stored
    token by token ([t, hq, d]), or None. fp32 inside, each output rounded once. The rows it writes are not
    stable (stable_tiles of a decode) for the launch that follows it."""
    what = "append_rope"
    if q is not None and (hb := _lib.host()) is not None:
        out = hb.append_rope(k, v, cos, sin, k_pool, v_pool, slots, q, q_norm, k_norm, float(eps))
        if out is not None:
            return out
    require_cuda(k, v, cos, sin, k_pool, v_pool, slots, *(x for x in (q, q_norm, k_norm) if x is not None), what=what)
    batched = k.dim() == 4
    if batched:
        if k.shape[0] != 1 or v.dim() != 4 or v.shape[0] != 1 or (q is not None and (q.dim() != 4 or q.shape[0] != 1)):
            raise ValueError(f"{what}: one sequence per call (batch 1)")
        k, v, q = k[0], v[0], q[0] if q is not None else None
    if cos.dim() == 3 and cos.shape[0] == 1:
        cos = cos[0]
    if sin.dim() == 3 and sin.shape[0] == 1:
        sin = sin[0]
    if k.dim() != 3 or v.shape != k.shape or (q is not None and q.dim() != 3):
        raise ValueError(f"{what}: expected k, v [hkv, t, d] and q [hq, t, d]; got {tuple(k.shape)}, {tuple(v.shape)}"
                         + (f", {tuple(q.shape)}" if q is not None else ""))
    hkv, t, d = k.shape
    hq = q.shape[0] if q is not None else 0
    if q is not None and tuple(q.shape) != (hq, t, d):
        raise ValueError(f"{what}: q {tuple(q.shape)} does not match k {tuple(k.shape)}")
    rot = cos.shape[-1]
    if cos.dim() != 2 or cos.shape[0] != t or sin.shape != cos.shape or sin.dtype != cos.dtype:
        raise ValueError(f"{what}: cos/sin must be [{t}, rot] of one dtype, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    if d % 2 or d > 512 or rot % 2 or not 2 <= rot <= d:
        raise ValueError(f"{what}: needs an even head size <= 512 and an even rot in [2, d], got d = {d}, rot = {rot}")
    if k_pool.dim() != 4 or k_pool.shape[1] != hkv or k_pool.shape[3] != d or v_pool.shape != k_pool.shape:
        raise ValueError(f"{what}: pools must be [pages, {hkv}, page_rows, {d}], got {tuple(k_pool.shape)}")
    if k_pool.stride(-1) != 1 or v_pool.stride() != k_pool.stride():
        raise ValueError(f"{what}: the pools must have equal strides and a contiguous last dimension (they are written)")
    if tuple(slots.shape) != (t, 2) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int32 [{t}, 2] tensor")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (tuple(w.shape) != (d,) or w.dtype != k.dtype):
            raise ValueError(f"{what}: {name} must be [{d}] of {k.dtype}")
    code = dtype_code(k, what)
    for x in (v, k_pool, v_pool) if q is None else (v, k_pool, v_pool, q):
        if x.dtype != k.dtype:
            raise TypeError(f"threadcut_b200.{what}: dtype mismatch {k.dtype} vs {x.dtype}")
    if cos.dtype != k.dtype and cos.dtype != torch.float32:
        raise TypeError(f"threadcut_b200.{what}: cos/sin must be {k.dtype} or fp32, got {cos.dtype}")
    k, v, cos, sin = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v, cos, sin))
    q_norm, k_norm = (w if w is None or w.stride(0) == 1 else w.contiguous() for w in (q_norm, k_norm))
    out = None
    if q is not None:
        q = q if q.stride(-1) == 1 else q.contiguous()
        out = torch.empty((t, hq, d), dtype=q.dtype, device=q.device).transpose(0, 1)
    dev = k.device
    ks, vs, ps = k.stride(), v.stride(), k_pool.stride()
    qs, os = (q.stride(), out.stride()) if q is not None else ((0, 0), (0, 0))
    with torch.cuda.device(dev):
        st = lib().tc_paged_append_rope(
            q.data_ptr() if q is not None else None, k.data_ptr(), v.data_ptr(),
            out.data_ptr() if q is not None else None, k_pool.data_ptr(), v_pool.data_ptr(), hq, hkv, d, t, qs[0],
            qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], q_norm.data_ptr() if q_norm is not None else None,
            k_norm.data_ptr() if k_norm is not None else None, float(eps), cos.data_ptr(), sin.data_ptr(), rot,
            cos.stride(0), sin.stride(0), _lib.DTYPE_CODE[cos.dtype], k_pool.shape[2], k_pool.shape[0], ps[0], ps[1],
            ps[2], slots.data_ptr(), code, stream_ptr(dev))
    check("tc_paged_append_rope", st)
    return out[None] if batched and out is not None else out


class PagedKV:
    """Paged K/V of `layers` attention layers of one sequence on one GPU.

    Pools: k[l], v[l] of shape [pages, hkv, page_rows, d] (16-bit dtypes for decode). A step is
    `reserve(t)` (once, for all layers) followed by `write(l, k, v)` per layer, or, for a one-token
    decode step, `decode(l, q, scale, k_new=..., v_new=...)` per layer, which writes the new row in
    the same launch that reads the cache."""

    def __init__(self, layers, hkv, d, *, max_tokens, page_rows=64, dtype=torch.bfloat16, device=None,
                 spare_pages=2):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dev.type != "cuda":
            raise RuntimeError("PagedKV: needs a CUDA device")
        self.layers, self.hkv, self.d = int(layers), int(hkv), int(d)
        self.page_rows = int(page_rows)
        pages = -(-int(max_tokens) // self.page_rows) + int(spare_pages)
        self.table = PageTable(pages, self.page_rows)
        self.dtype, self.device = dtype, dev
        row, kind = self._row()
        shape = (pages, self.hkv, self.page_rows, row)
        self.k = [torch.zeros(shape, dtype=kind, device=dev) for _ in range(self.layers)]
        self.v = [torch.zeros(shape, dtype=kind, device=dev) for _ in range(self.layers)]
        self._kptrs = (ctypes.c_void_p * self.layers)(*[t.data_ptr() for t in self.k])
        self._slots = None       # device int32 [t, 2] of the step reserved last
        self._tiles_dev = None   # device int32 [capacity, 3]: the tile table, rows [0, n) valid
        self._tiles_ver = -1     # table version the device copy reflects
        self._win = {}           # (window, sinks) -> device int32 [T, 3]: the tiles a windowed decode reads
        self._win_ver = -1       # table version those tables reflect
        self._ktab = None        # device int32 [T, 4]: tiles + logical start, for prefill
        self._ktab_starts = None
        self._ktab_ver = -1

    def _row(self):
        """Elements and type of a pool's row."""
        return self.d, self.dtype

    @property
    def row_bytes(self):
        """Bytes of a token's key (or value) of one head."""
        return self._row()[0] * self._row()[1].itemsize

    @property
    def n(self):
        return self.table.n

    @property
    def n_tiles(self):
        return self.table.tiles().shape[0]

    def _strides(self):
        s = next(t for t in self.k if t is not None).stride()  # compact() frees pools layer by layer
        return s[0], s[1], s[2]

    def _tiles(self):
        """Device tile table and its length, brought up to date by copying only the rows that
        changed since the last call (an append changes the tail; a splice everything)."""
        tab = self.table.tiles()
        nt = tab.shape[0]
        if self._tiles_ver != self.table.version:
            lo = self.table.dirty
            if self._tiles_dev is None or self._tiles_dev.shape[0] < nt:
                cap = max(nt, 2 * (self._tiles_dev.shape[0] if self._tiles_dev is not None else 0), 64)
                self._tiles_dev = torch.empty((cap, 3), dtype=torch.int32, device=self.device)
                lo = 0
            if lo < nt:
                self._tiles_dev[lo:nt].copy_(torch.from_numpy(np.ascontiguousarray(tab[lo:nt])))
            self.table.mark_clean()
            self._tiles_ver = self.table.version
        return (self._tiles_dev if nt else None), nt

    # ---------------------------------------------------------------- step
    def reserve(self, t):
        """Takes t slots at the end of the sequence for the next write/decode of every layer."""
        slots = self.table.reserve(t)
        self._slots = torch.from_numpy(slots).to(self.device)
        return self._slots

    def write(self, layer, k, v):
        """Writes the reserved step's rows of one layer: k, v [hkv, t, d] (or [1, hkv, t, d])."""
        if k.dim() == 4:
            k, v = k[0], v[0]
        require_cuda(k, v, what="PagedKV.write")
        t = k.shape[1]
        if self._slots is None or self._slots.shape[0] != t:
            raise ValueError("PagedKV.write: reserve(t) the step's slots first (same t)")
        if k.shape != (self.hkv, t, self.d) or v.shape != k.shape or k.dtype != self.dtype or v.dtype != self.dtype:
            raise ValueError(f"PagedKV.write: expected [{self.hkv}, t, {self.d}] {self.dtype}, got {tuple(k.shape)} {k.dtype}")
        if k.stride(-1) != 1 or v.stride(-1) != 1:
            k, v = k.contiguous(), v.contiguous()
        sp, sh, sr = self._strides()
        with torch.cuda.device(self.device):
            check("tc_paged_write", lib().tc_paged_write(
                k.data_ptr(), v.data_ptr(), self.k[layer].data_ptr(), self.v[layer].data_ptr(), self.hkv, self.d, t,
                k.stride(0), k.stride(1), v.stride(0), v.stride(1), self.page_rows, self.table.num_pages,
                sp, sh, sr, self._slots.data_ptr(), dtype_code(k, "PagedKV.write"), stream_ptr(self.device)))

    def append(self, layer, k, v, cos, sin, *, q=None, q_norm=None, k_norm=None, eps=1e-6):
        """Rotates the reserved step's raw keys (and queries) of one layer and writes keys and values
        to its slots in one launch: append_rope into this layer's pools. Returns the rotated queries."""
        t = k.shape[-2]
        if self._slots is None or self._slots.shape[0] != t:
            raise ValueError("PagedKV.append: reserve(t) the step's slots first (same t)")
        return append_rope(k, v, cos, sin, self.k[layer], self.v[layer], self._slots, q=q, q_norm=q_norm,
                           k_norm=k_norm, eps=eps)

    def _window_tiles(self, window, sinks):
        """Device tile table of a windowed decode, its length and the tokens it lists; built once per
        window and state of the sequence (once a step for all layers that share a window)."""
        if self._win_ver != self.table.version:
            self._win, self._win_ver = {}, self.table.version
        tab = self._win.get((window, sinks))
        if tab is None:
            # a fresh tensor: an earlier step's launches may still be reading the old one
            tab = torch.from_numpy(np.ascontiguousarray(self.table.window_tiles(window, sinks))).to(self.device)
            self._win[(window, sinks)] = tab
        nt = tab.shape[0]
        return (tab if nt else None), nt, min(self.table.n, window + sinks)

    def decode(self, layer, q, scale, *, k_new=None, v_new=None, splits=None, stable_tiles=0, window=None, sinks=0):
        """Decode attention of q [hkv, g, d] over the whole sequence (threadcut/flash_decode.py:57-69
        semantics). With k_new/v_new [hkv, d] the last reserved row (a one-token step) is written by
        the same launch (fused append). stable_tiles: the leading tiles of the table (see
        `n_tiles`) whose rows no kernel still running writes, which the launch may load before the
        previous one ends (0: none; n_tiles - 1 in a layer-by-layer decode step with fused append,
        where each launch writes only the last row of its own layer). window / sinks: the query sees
        only the first `sinks` and the last `window` tokens (the newest one counted), as
        flash_decode.decode_attention_window; stable_tiles is ignored then."""
        require_cuda(q, what="PagedKV.decode")
        hkv, g, d = q.shape
        if hkv != self.hkv or d != self.d or q.dtype != self.dtype:
            raise ValueError(f"PagedKV.decode: q {tuple(q.shape)} {q.dtype} does not match the cache")
        if (k_new is None) != (v_new is None):
            raise ValueError("PagedKV.decode: k_new and v_new go together")
        if k_new is not None:
            if self._slots is None or self._slots.shape[0] != 1:
                raise ValueError("PagedKV.decode: reserve(1) the step's slot before a fused append")
            if k_new.dim() == 3:
                k_new, v_new = k_new.reshape(hkv, d), v_new.reshape(hkv, d)
            if k_new.shape != (hkv, d) or v_new.shape != (hkv, d):
                raise ValueError("PagedKV.decode: k_new/v_new must be [hkv, d]")
            if k_new.stride(-1) != 1 or v_new.stride(-1) != 1:
                k_new, v_new = k_new.contiguous(), v_new.contiguous()
        if q.stride(-1) != 1:
            q = q.contiguous()
        tiles, nt, n = self._decode_tiles(window, sinks, "PagedKV.decode")
        stable_tiles = 0 if window is not None else stable_tiles
        out = torch.empty((hkv, g, d), dtype=q.dtype, device=q.device)
        code = dtype_code(q, "PagedKV.decode")
        ws = workspaces.get(("decode", hkv), q.device, _lib.decode_workspace_bound(1, hkv, g, d, code))
        sp, sh, sr = self._strides()
        with torch.cuda.device(q.device):
            check("tc_decode_attention_paged", lib().tc_decode_attention_paged(
                q.data_ptr(), self.k[layer].data_ptr(), self.v[layer].data_ptr(), out.data_ptr(), hkv, g, d,
                self.page_rows, self.table.num_pages, sp, sh, sr, tiles.data_ptr() if tiles is not None else None,
                nt, n, k_new.data_ptr() if k_new is not None else None,
                v_new.data_ptr() if v_new is not None else None, k_new.stride(0) if k_new is not None else 0,
                v_new.stride(0) if v_new is not None else 0, q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                float(scale), int(splits or 0), code, int(stable_tiles), ws.data_ptr(), ws.numel(),
                stream_ptr(q.device)))
        return out

    def decode_shared(self, layer, q, k, v, scale, lengths=None):
        """flash_decode.decode_attention_shared with this sequence as the prefix, straight over its pages:
        q [b, hkv, g, d], the continuations' suffixes k/v [b, hkv, m, d] of which the first lengths[i] rows
        count (int32 CUDA [b], clamped into [0, m]; None: all m). 16-bit, d in {64, 128, 256}, g <= 128,
        scale > 0; weights rounded to 16 bits, as there. Returns [b, hkv, g, d]."""
        what = "PagedKV.decode_shared"
        require_cuda(q, k, v, what=what)
        if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"{what}: expected q [b, hkv, g, d], k/v [b, hkv, m, d]; got {tuple(q.shape)}, "
                             f"{tuple(k.shape)}, {tuple(v.shape)}")
        b, hkv, g, d = q.shape
        m = k.shape[2]
        if hkv != self.hkv or d != self.d or k.shape != (b, hkv, m, d):
            raise ValueError(f"{what}: q {tuple(q.shape)} / k {tuple(k.shape)} do not match the cache")
        if q.dtype != self.dtype or k.dtype != self.dtype or v.dtype != self.dtype or self.dtype == torch.float32:
            raise TypeError(f"threadcut_b200.{what}: needs the cache's 16-bit dtype {self.dtype}, got {q.dtype}, "
                            f"{k.dtype}, {v.dtype}")
        if not scale > 0:
            raise ValueError(f"{what}: needs scale > 0, got {scale}")
        q, k, v = (rows16(x) for x in (q, k, v))
        lens_ptr = None
        if lengths is not None:
            if lengths.dtype != torch.int32 or lengths.device != q.device or not lengths.is_contiguous():
                lengths = lengths.to(device=q.device, dtype=torch.int32).contiguous()
            if lengths.shape != (b,):
                raise ValueError(f"{what}: lengths must be [{b}]")
            lens_ptr = lengths.data_ptr()
        tiles, nt = self._tiles()
        out = torch.empty((b, hkv, g, d), dtype=q.dtype, device=q.device)
        L = lib()
        code = dtype_code(q, what)
        sp, sh, sr = self._strides()
        with torch.cuda.device(q.device):
            nb = L.tc_decode_attention_shared_workspace_size(b, hkv, g, d, TILE_ROWS * nt, m, code)
            ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb else None
            st = L.tc_decode_attention_shared_paged(
                q.data_ptr(), self.k[layer].data_ptr(), self.v[layer].data_ptr(), k.data_ptr(), v.data_ptr(),
                out.data_ptr(), b, hkv, g, d, self.page_rows, self.table.num_pages, sp, sh, sr,
                tiles.data_ptr() if tiles is not None else None, nt, m, lens_ptr, *q.stride()[:3], *k.stride()[:3],
                *v.stride()[:3], *out.stride()[:3], float(scale), code, ws.data_ptr() if ws is not None else None, nb,
                stream_ptr(q.device))
        check("tc_decode_attention_shared_paged", st)
        return out

    def _decode_tiles(self, window, sinks, what):
        """Device tile table of a decode, its length and the tokens it lists, for all tokens or a window's."""
        if window is None:
            if sinks:
                raise ValueError(f"{what}: sinks go with a window")
            return (*self._tiles(), self.table.n)
        if window < 1 or sinks < 0:
            raise ValueError(f"{what}: needs window >= 1 and sinks >= 0, got {window} and {sinks}")
        return self._window_tiles(int(window), int(sinks))

    def _prefill_table(self):
        """Device int32 [T, 4] = (page, first row, rows, logical position of the first row) of the
        current tile table, and the host copy of the logical starts."""
        if self._ktab_ver != self.table.version:
            tab = self.table.tiles()
            starts = (np.cumsum(tab[:, 2], dtype=np.int64) - tab[:, 2]).astype(np.int32)
            k4 = np.ascontiguousarray(np.concatenate((tab, starts[:, None]), axis=1))
            self._ktab = torch.from_numpy(k4).to(self.device)
            self._ktab_starts = starts
            self._ktab_ver = self.table.version
        return self._ktab, self._ktab_starts

    def _prefill_window(self, layer, query, scale, window, sinks, splits):
        """prefill with a sliding window and sinks (tc_prefill_attention_window_paged)."""
        what = "PagedKV.prefill"
        _, hq, lq, d = query.shape
        n = self.table.n
        if (query.shape[0] != 1 or d != self.d or d not in (64, 128) or hq % self.hkv or hq // self.hkv > 128
                or query.dtype != self.dtype or query.dtype not in (torch.bfloat16, torch.float16) or not 1 <= lq <= n):
            raise ValueError(f"{what}: query {tuple(query.shape)} {query.dtype} does not fit the cache")
        if window < 1 or sinks < 0 or not scale > 0:
            raise ValueError(f"{what}: needs window >= 1, sinks >= 0 and scale > 0, got {window}, {sinks} and {scale}")
        ktab, starts = self._prefill_table()
        tile_starts = starts[::4]
        block = 2 * (128 // (hq // self.hkv))
        p0 = (n - lq) + block * np.arange(-(-lq // block), dtype=np.int64)
        qb = np.empty((p0.shape[0], 2), np.int32)
        qb[:, 0] = np.searchsorted(tile_starts, np.maximum(p0 + 1 - window, 0), side="right") - 1
        qb[:, 1] = np.searchsorted(tile_starts, np.minimum(p0 + block, n), side="left")
        qb_tiles = torch.from_numpy(qb).to(self.device)
        q = rows16(query[0])
        out = torch.empty((1, lq, hq, d), dtype=query.dtype, device=query.device)
        L = lib()
        n_sub = ktab.shape[0]
        sp, sh, sr = self._strides()
        with torch.cuda.device(query.device):
            nb = L.tc_prefill_window_workspace_size(1, hq, self.hkv, lq, max(lq, 128 * (-(-n_sub // 4))), d,
                                                    min(window, n), min(sinks, n), splits)
            ws = torch.empty(nb, dtype=torch.uint8, device=query.device) if nb else None
            st = L.tc_prefill_attention_window_paged(
                q.data_ptr(), self.k[layer].data_ptr(), self.v[layer].data_ptr(), out.data_ptr(), hq, self.hkv, lq, n, d,
                self.page_rows, self.table.num_pages, sp, sh, sr, ktab.data_ptr(), n_sub, qb_tiles.data_ptr(),
                int(np.searchsorted(tile_starts, min(sinks, n), side="left")), min(window, n), min(sinks, n),
                q.stride(0), q.stride(1), out.stride(1), out.stride(2), float(scale), splits,
                _lib.DTYPE_CODE[query.dtype], ws.data_ptr() if ws is not None else None, nb, stream_ptr(query.device))
        check("tc_prefill_attention_window_paged", st)
        return out

    def prefill(self, layer, query, scale, *, splits=None, window=None, sinks=0):
        """Causal attention of a chunk's queries over the whole paged sequence, whose last lq tokens
        are the chunk (already written): query [1, 4*hkv, lq, 128] (bf16/fp16) -> [1, lq, hq, 128],
        as threadcut_b200.prefill.prefill_attention on the contiguous cache, with no copy of it.
        window / sinks: each query sees only the first `sinks` and the last `window` keys up to its own, as
        prefill.prefill_attention_window; then any number of query heads (up to 128 per KV head) and d of 64
        or 128."""
        require_cuda(query, what="PagedKV.prefill")
        if window is not None:
            return self._prefill_window(layer, query, scale, int(window), int(sinks), int(splits or 0))
        if sinks:
            raise ValueError("PagedKV.prefill: sinks go with a window")
        _, hq, lq, d = query.shape
        n = self.table.n
        if (query.shape[0] != 1 or d != 128 or d != self.d or hq != 4 * self.hkv or query.dtype != self.dtype
                or query.dtype not in (torch.bfloat16, torch.float16) or not 1 <= lq <= n):
            raise ValueError(f"PagedKV.prefill: query {tuple(query.shape)} {query.dtype} does not fit the cache")
        ktab, starts = self._prefill_table()
        n_sub = ktab.shape[0]
        nqb = -(-lq // 64)
        kend = np.minimum(n, (n - lq) + 64 * (np.arange(nqb, dtype=np.int64) + 1))
        qbt = np.maximum(np.searchsorted(starts[::4], kend, side="left"), 1).astype(np.int32)
        qb_tiles = torch.from_numpy(qbt).to(self.device)
        q = query[0]
        if q.stride(-1) != 1:
            q = q.contiguous()
        out = torch.empty((1, lq, hq, d), dtype=query.dtype, device=query.device)
        L = lib()
        sp, sh, sr = self._strides()
        s = int(splits or 0)
        with torch.cuda.device(query.device):
            nb = L.tc_prefill_workspace_size(hq, self.hkv, lq, 128 * (-(-n_sub // 4)), s)
            ws = workspaces.get("prefill", query.device, nb) if nb else None
            st = L.tc_prefill_attention_paged(
                q.data_ptr(), self.k[layer].data_ptr(), self.v[layer].data_ptr(), out.data_ptr(), hq, self.hkv, lq, n,
                d, self.page_rows, self.table.num_pages, sp, sh, sr, ktab.data_ptr(), n_sub, qb_tiles.data_ptr(),
                q.stride(0), q.stride(1), out.stride(1), out.stride(2), float(scale), s, _lib.DTYPE_CODE[query.dtype],
                ws.data_ptr() if ws is not None else None, nb, stream_ptr(query.device))
        check("tc_prefill_attention_paged", st)
        return out

    # ---------------------------------------------------------------- splice
    def splice(self, s: Split, inv_freq):
        """A.B.C -> A.C on every layer (threadcut/kv.py:28-41, 83-92 semantics): B's pages return to
        the pool, C's keys are re-rotated by -(c0 - a) positions where they lie, nothing moves."""
        gap = int(s.c0) - int(s.a)
        self._rotates(s, inv_freq, "PagedKV.splice")
        runs_c, _ = self.table.splice(s)
        if gap == 0 or runs_c.shape[0] == 0:
            return  # the reference clones C onto itself: nothing to rotate
        tab = PageTable.tiles_of(runs_c)
        tiles = torch.from_numpy(tab).to(self.device)
        cs, cs_ptr = _lib.cos_sin_table(-gap, inv_freq)
        sp, sh, sr = self._strides()
        with torch.cuda.device(self.device):
            check("tc_paged_rotate_keys", lib().tc_paged_rotate_keys(
                self._kptrs, self.layers, self.hkv, self.d, self.page_rows, self.table.num_pages, sp, sh, sr,
                tiles.data_ptr(), tab.shape[0], cs_ptr, _lib.DTYPE_CODE[self.dtype], stream_ptr(self.device)))
        del cs  # the table is copied into the launch parameters

    def _rotates(self, s, inv_freq, what):
        """Refuses frequencies that a splice's keys cannot be rotated by, before anything has changed."""
        if s.c0 != s.a and s.c and inv_freq.numel() * 2 != self.d:
            raise ValueError(f"{what}: inv_freq has {inv_freq.numel()} entries, keys need {self.d // 2}")

    def truncate(self, n):
        self.table.truncate(n)

    def compact(self):
        """Re-packs the sequence into pages in logical order (one copy of every layer's K and V into
        fresh pools), for when splices have left so many partly used pages that an append finds no
        free page. Peak memory: the old and the new pools."""
        new = PagedKV(self.layers, self.hkv, self.d, max_tokens=self.table.num_pages * self.page_rows,
                      page_rows=self.page_rows, dtype=self.dtype, device=self.device, spare_pages=0)
        n = self.n
        if n:
            new.reserve(n)
            for l in range(self.layers):
                k, v = self.gather(l)
                new.write(l, k, v)
                self.k[l] = self.v[l] = None  # free the old pools layer by layer
        self.__dict__.update(new.__dict__)

    # ---------------------------------------------------------------- views
    def gather(self, layer):
        """Contiguous copies (K, V) [hkv, n, d] of one layer in logical order (tc_paged_gather), for
        the attention paths that do not read pages and for compact()."""
        n = self.table.n
        k = torch.empty((self.hkv, n, self.d), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        if n == 0:
            return k, v
        ktab, _ = self._prefill_table()
        sp, sh, sr = self._strides()
        with torch.cuda.device(self.device):
            check("tc_paged_gather", lib().tc_paged_gather(
                self.k[layer].data_ptr(), self.v[layer].data_ptr(), k.data_ptr(), v.data_ptr(), self.hkv, self.d, n,
                k.stride(0), k.stride(1), self.page_rows, self.table.num_pages, sp, sh, sr, ktab.data_ptr(),
                ktab.shape[0], _lib.DTYPE_CODE[self.dtype], stream_ptr(self.device)))
        return k, v


class PagedKVInt4(PagedKV):
    """PagedKV whose rows are held in 4 bits (threadcut_b200.int4: 5 d / 8 bytes a row instead of 2 d): the same steps,
    splices and reads over uint8 pools [pages, hkv, page_rows, row_bytes(d)]. dtype (bf16 or fp16) is the type that keys and
    values come in and are read back as; d 64, 128 or 256.

    Keys that a splice rotates are quantised again: each splice that moves a key may move its elements by half a level.
    The shared decode has no form over such rows: gather the context once and use decode_attention_shared."""

    def __init__(self, layers, hkv, d, *, dtype=torch.bfloat16, **kwargs):
        if d not in int4.HEAD_SIZES or dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PagedKVInt4: needs bf16 or fp16 and heads of 64, 128 or 256, got {dtype} and {d}")
        super().__init__(layers, hkv, d, dtype=dtype, **kwargs)

    def _row(self):
        return int4.row_bytes(self.d), torch.uint8

    def _step(self, k, what):
        t = k.shape[-2]
        if self._slots is None or self._slots.shape[0] != t:
            raise ValueError(f"{what}: reserve(t) the step's slots first (same t)")
        if tuple(k.shape[-3:]) != (self.hkv, t, self.d) or k.dtype != self.dtype:
            raise ValueError(f"{what}: expected [{self.hkv}, t, {self.d}] {self.dtype}, got {tuple(k.shape)} {k.dtype}")

    def write(self, layer, k, v):
        """Quantises and writes the reserved step's rows of one layer: k, v [hkv, t, d] (or [1, hkv, t, d])."""
        self._step(k, "PagedKVInt4.write")
        int4.write_int4(k, v, self.k[layer], self.v[layer], self._slots)

    def append(self, layer, k, v, cos, sin, *, q=None, q_norm=None, k_norm=None, eps=1e-6):
        """PagedKV.append with the keys and values quantised: int4.append_rope_int4 into this layer's pools."""
        self._step(k, "PagedKVInt4.append")
        return int4.append_rope_int4(k, v, cos, sin, self.k[layer], self.v[layer], self._slots, q=q, q_norm=q_norm,
                                     k_norm=k_norm, eps=eps)

    def decode(self, layer, q, scale, *, k_new=None, v_new=None, splits=None, stable_tiles=0, window=None, sinks=0):
        """PagedKV.decode over the 4-bit rows (decode_attention_int4): q [hkv, g, d], at most 16 query heads a KV head.
        k_new / v_new [hkv, d] (or [hkv, 1, d]) are written first, in a launch of their own. stable_tiles changes nothing."""
        what = "PagedKVInt4.decode"
        require_cuda(q, what=what)
        if q.dim() != 3 or q.shape[0] != self.hkv or q.shape[2] != self.d or q.dtype != self.dtype:
            raise ValueError(f"{what}: q {tuple(q.shape)} {q.dtype} does not match the cache")
        if (k_new is None) != (v_new is None):
            raise ValueError(f"{what}: k_new and v_new go together")
        if k_new is not None:
            if self._slots is None or self._slots.shape[0] != 1:
                raise ValueError(f"{what}: reserve(1) the step's slot first")
            self.write(layer, k_new.reshape(self.hkv, 1, self.d), v_new.reshape(self.hkv, 1, self.d))
        tiles, nt, _ = self._decode_tiles(window, sinks, what)
        if nt == 0:
            return torch.zeros_like(q)
        return int4.decode_attention_int4(q, self.k[layer], self.v[layer], scale, tiles=tiles[:nt], splits=splits)

    def decode_shared(self, layer, q, k, v, scale, lengths=None):
        raise ValueError("PagedKVInt4.decode_shared: no shared decode over 4-bit rows; gather(layer) the context once and use "
                         "flash_decode.decode_attention_shared")

    def prefill(self, layer, query, scale, *, splits=None, window=None, sinks=0):
        """PagedKV.prefill: the rows that the chunk's queries see are read back as 16-bit keys and values (gather_int4)
        and the contiguous kernels run over them."""
        what = "PagedKVInt4.prefill"
        require_cuda(query, what=what)
        n = self.n
        if (query.dim() != 4 or query.shape[0] != 1 or query.shape[3] != self.d or query.dtype != self.dtype
                or not 1 <= query.shape[2] <= n):
            raise ValueError(f"{what}: query {tuple(query.shape)} {query.dtype} does not fit the cache")
        if window is None:
            if sinks:
                raise ValueError(f"{what}: sinks go with a window")
            k, v = self.gather(layer)
            return prefill_attention(query, k[None], v[None], scale, splits=splits)
        if window < 1 or sinks < 0:
            raise ValueError(f"{what}: needs window >= 1 and sinks >= 0, got {window} and {sinks}")
        first = max(0, n - query.shape[2] - int(window) + 1) if sinks == 0 else 0
        k, v = self.gather(layer, first)
        return prefill_attention_window(query, k[None], v[None], scale, int(window), int(sinks), splits=splits)

    def splice(self, s: Split, inv_freq):
        """A.B.C -> A.C on every layer: B's pages return to the pool, C's keys are rotated by -(c0 - a) positions and
        quantised again where they lie (int4.rotate_keys_int4)."""
        gap = int(s.c0) - int(s.a)
        self._rotates(s, inv_freq, "PagedKVInt4.splice")
        runs_c, _ = self.table.splice(s)
        if gap and runs_c.shape[0]:
            tiles = torch.from_numpy(PageTable.tiles_of(runs_c)).to(self.device)
            int4.rotate_keys_int4(self.k, tiles, -gap, inv_freq, self.dtype)

    def compact(self):
        """PagedKV.compact; the rows' bytes are moved as they are."""
        at = torch.from_numpy(self.table.positions()).to(self.device)
        new = PagedKVInt4(self.layers, self.hkv, self.d, max_tokens=self.table.num_pages * self.page_rows,
                          page_rows=self.page_rows, dtype=self.dtype, device=self.device, spare_pages=0)
        if self.n:
            to = new.reserve(self.n).long()
            for l in range(self.layers):
                for pools, fresh in ((self.k, new.k), (self.v, new.v)):
                    fresh[l][to[:, 0], :, to[:, 1]] = pools[l][at[:, 0], :, at[:, 1]]
                    pools[l] = None  # free the old pools layer by layer
        self.__dict__.update(new.__dict__)

    def gather(self, layer, first=0):
        """Contiguous (K, V) [hkv, n - first, d] of the tokens from `first` on, in logical order and of the cache's dtype."""
        n = self.n
        if first == 0:
            tiles = self._prefill_table()[0] if n else torch.zeros((0, 4), dtype=torch.int32, device=self.device)
        else:
            tab = self.table._span(first, n, *self.table._index())[1]
            start = np.cumsum(tab[:, 2], dtype=np.int64) - tab[:, 2]
            tab = np.concatenate((tab, start[:, None].astype(np.int32)), axis=1)
            tiles = torch.from_numpy(np.ascontiguousarray(tab)).to(self.device)
        return int4.gather_int4(self.k[layer], self.v[layer], tiles, n - first, self.dtype)
