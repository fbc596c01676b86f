"""The block table of a windowed prefill over pages (tc_prefill_attention_window_paged) on a B200: written by
the launch just before, and with values outside the tiles that there are."""
import numpy as np
import pytest
import torch

from attn_bounds import assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.paged import PagedKV, append_rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HKV, G, D, LQ, WINDOW = 2, 4, 128, 512, 300


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def block_table(starts, n, window):
    """[blocks, 2] as the header describes it, from the key tiles' logical starts; 64 queries a block."""
    tile_starts = starts[::4]
    p0 = (n - LQ) + 64 * np.arange(LQ // 64)
    first = np.searchsorted(tile_starts, np.maximum(p0 + 1 - window, 0), side="right") - 1
    return np.stack((first, np.searchsorted(tile_starts, np.minimum(p0 + 64, n), side="left")), 1).astype(np.int32)


def prefill(kv, q, qb):
    n = kv.n
    ktab, starts = kv._prefill_table()
    out = torch.empty(1, LQ, HKV * G, D, device=DEV, dtype=q.dtype)
    page, head, row = kv._strides()
    st = _lib.lib().tc_prefill_attention_window_paged(
        q.data_ptr(), kv.k[0].data_ptr(), kv.v[0].data_ptr(), out.data_ptr(), HKV * G, HKV, LQ, n, D, kv.page_rows,
        kv.table.num_pages, page, head, row, ktab.data_ptr(), ktab.shape[0], qb.data_ptr(), 0, WINDOW, 0, q.stride(0),
        q.stride(1), out.stride(1), out.stride(2), 0.1, 1, 2, None, 0, _lib.stream_ptr(q.device))
    assert st == 0
    return out


def test_a_table_that_the_previous_launch_writes():
    """A paged append, which lets the next launch start early, writes the table as the bits of its last value row; until
    then the table is that of a wider window."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    n, t = 3000, 200000
    kv = PagedKV(1, HKV, D, max_tokens=n, device=DEV)
    kv.reserve(n)
    kv.write(0, *(torch.randn(HKV, n, D, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2)))
    q = torch.randn(HKV * G, LQ, D, generator=gen, device=DEV).to(torch.bfloat16)
    want = kv.prefill(0, q[None], 0.1, window=WINDOW, splits=1)
    starts = kv._prefill_table()[1]
    right, wider = (torch.from_numpy(block_table(starts, n, w)).to(DEV).reshape(16) for w in (WINDOW, n))
    assert not torch.equal(right, wider)
    rows = torch.zeros(1, t, 16, device=DEV)
    rows[0, -1] = right.view(torch.float32)
    cos = torch.ones(t, 16, device=DEV)
    slots = torch.stack((torch.zeros(t), torch.arange(t)), 1).to(DEV, torch.int32)
    k_pool, v_pool = (torch.zeros(1, 1, t, 16, device=DEV) for _ in range(2))
    qb = v_pool[0, 0, -1].view(torch.int32)
    outs = []
    for _ in range(10):
        qb.copy_(wider)
        append_rope(rows, rows, cos, cos, k_pool, v_pool, slots)
        outs.append(prefill(kv, q, qb))
    for out in outs:
        assert torch.equal(out, want)


def test_table_values_outside_the_tiles_are_held_within_them():
    """Each block sees the keys of its window that lie in its tiles, a first tile below 0 being tile 0, an end past the
    last tile that tile's, and no end before the second tile or first tile past the end's."""
    gen = torch.Generator(device=DEV).manual_seed(10)
    n = 1500
    kv = PagedKV(1, HKV, D, max_tokens=n, device=DEV)
    kv.reserve(n)
    kv.write(0, *(torch.randn(HKV, n, D, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2)))
    q = torch.randn(HKV * G, LQ, D, generator=gen, device=DEV).to(torch.bfloat16)
    starts = kv._prefill_table()[1]
    right = block_table(starts, n, WINDOW)
    tiles = -(-len(starts) // 4)
    edges = torch.tensor([int(x) for x in starts[::4]] + [n], device=DEV)
    most = 2 ** 31 - 1
    bad = right.copy()
    bad[0], bad[1, 0], bad[2, 1], bad[3] = (-most - 1, most), -5, 10 ** 6, (0, most)
    bad[4], bad[5], bad[6] = (most, most), (10, 10), (3, -7)
    held = [(0, tiles), (0, right[1, 1]), (right[2, 0], tiles), (0, tiles), (tiles - 1, tiles), (9, 10), (0, 1), tuple(right[7])]
    at = (n - LQ + torch.arange(LQ, device=DEV))[:, None]
    j = torch.arange(n, device=DEV)
    lo, hi = (edges[torch.tensor([int(h[i]) for h in held], device=DEV)].repeat_interleave(64)[:, None] for i in (0, 1))
    k, v = (x.repeat_interleave(G, 0) for x in kv.gather(0))
    seen = (j <= at) & (j > at - WINDOW) & (j >= lo) & (j < hi)
    assert not seen[384:448].any()  # a block without a key gives zeros
    ref, tol = attend64(q, k, v, 0.1, seen)
    assert_within(prefill(kv, q, torch.from_numpy(bad).to(DEV))[0], ref.transpose(0, 1), tol.transpose(0, 1))
