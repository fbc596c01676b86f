"""4-bit rows in calls of thousands of tokens, which take other kernels than a few do, and groups of every offset and size."""
import pytest
import torch

import int4_ref as ref
from threadcut_b200 import int4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def slots_and_rows(t, rows, seed):
    """Slots of t tokens over shuffled pages, some of them outside the pool; (slots, tokens inside, their page and row, pages)."""
    _, where, total = ref.pages(t, rows, torch.Generator().manual_seed(seed))
    slots = where.to(torch.int32).contiguous()
    slots[5::97] = torch.tensor([-1, 3], dtype=torch.int32, device=DEV)
    slots[6::97] = torch.tensor([total, 0], dtype=torch.int32, device=DEV)
    slots[7::97] = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    at = torch.arange(t, device=DEV)
    inside = (at % 97 < 5) | (at % 97 > 7)
    return slots, inside, where[inside], total


@pytest.mark.parametrize("dtype,d,hkv", [(BF, 64, 5), (HF, 128, 3), (BF, 128, 8), (HF, 256, 2)])
def test_many_tokens_written(dtype, d, hkv):
    t = 12007
    x = randn(t, 2 * hkv, d, dtype=dtype).transpose(0, 1)  # views of one projection
    k, v = x[:hkv], x[hkv:]
    slots, inside, where, total = slots_and_rows(t, 48, 1)
    pools = [torch.full((total, hkv, 48, ref.row_bytes(d)), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    int4.write_int4(k, v, *pools, slots)
    for pool, src in zip(pools, (k, v)):
        want = torch.full_like(pool, 0xA5)
        want[where[:, 0], :, where[:, 1]] = ref.rows_of(src[:, inside].contiguous()).transpose(0, 1)
        assert torch.equal(pool, want)


@pytest.mark.parametrize("dtype,d,rot,table", [(BF, 128, 128, "same"), (HF, 64, 32, "f32"), (BF, 256, 256, "f32"),
                                               (HF, 128, 64, "same"), (BF, 64, 64, "same")])
@pytest.mark.parametrize("hq", [5, 0])
def test_many_tokens_rotated(dtype, d, rot, table, hq):
    hkv, t = 3, 12007
    x = randn(t, hq + 2 * hkv, d, dtype=dtype, seed=2).transpose(0, 1)
    q, k, v = x[:hq] if hq else None, x[hq:hq + hkv], x[hq + hkv:]
    angle = randn(t, rot, dtype=F32, seed=4) * 3
    tab = dtype if table == "same" else F32
    cos, sin = angle.cos().to(tab), angle.sin().to(tab)
    slots, inside, where, total = slots_and_rows(t, 64, 2)
    pools = [torch.full((total, hkv, 64, ref.row_bytes(d)), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    out = int4.append_rope_int4(k, v, cos, sin, *pools, slots, q=q)
    assert out is None if q is None else torch.equal(out, ref.rotate32(q, cos, sin))
    for pool, src in zip(pools, (ref.rotate32(k, cos, sin), v)):
        want = torch.full_like(pool, 0xA5)
        want[where[:, 0], :, where[:, 1]] = ref.rows_of(src[:, inside].contiguous()).transpose(0, 1)
        assert torch.equal(pool, want)


@pytest.mark.parametrize("dtype,d,rot", [(BF, 128, 128), (HF, 64, 32), (HF, 256, 128)])
@pytest.mark.parametrize("norms", ["both", "keys"])
def test_many_tokens_normalised_as_a_few_are(dtype, d, rot, norms):
    hq, hkv, t = 6, 3, 12007
    q, k, v = (randn(h, t, d, dtype=dtype, seed=i) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    angle = randn(t, rot, dtype=F32, seed=4) * 3
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    w = dict(q_norm=(1 + 0.1 * randn(d, dtype=F32, seed=5)).to(dtype) if norms == "both" else None,
             k_norm=(1 + 0.1 * randn(d, dtype=F32, seed=6)).to(dtype), eps=1e-6)
    slots, _, _, total = slots_and_rows(t, 64, 3)
    pools, few = ([torch.zeros((total, hkv, 64, ref.row_bytes(d)), dtype=torch.uint8, device=DEV) for _ in range(2)]
                  for _ in range(2))
    out = int4.append_rope_int4(k, v, cos, sin, *pools, slots, q=q, **w)
    for a in range(0, t, 400):
        s = slice(a, min(t, a + 400))
        part = int4.append_rope_int4(k[:, s], v[:, s], cos[s], sin[s], *few, slots[s], q=q[:, s], **w)
        assert torch.equal(out[:, s], part)
    assert all(torch.equal(a, b) and a.any() for a, b in zip(pools, few))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_groups_of_every_offset_and_size(dtype):
    """One token a (offset, size): offsets of up to 40 times the spread, spreads over the type's range; whole numbers, many of
    which lie on a border between two levels; and rotations of them by an angle of nothing, which quantise values again."""
    d, hkv = 128, 2
    offsets = [0.0, 0.5, 1.0, 2.0, 2.9, 3.0, 3.1, 3.9, 4.0, 4.1, 5.0, 8.0, 40.0]
    sizes = [2.0 ** e for e in (range(-122, 120, 9) if dtype == BF else range(-17, 9))]
    cases = [(sign * o, s) for o in offsets for sign in (1, -1) for s in sizes]
    spread, at = torch.tensor([s for _, s in cases], device=DEV), torch.tensor([o for o, _ in cases], device=DEV)
    x = randn(hkv, len(cases), d, dtype=F32).double()
    x = ((x + at.double()[:, None]) * spread.double()[:, None]).to(dtype)
    whole = torch.randint(0, 31, (hkv, 64, d), generator=torch.Generator().manual_seed(1)).to(DEV)
    whole[..., ::32], whole[..., 1::32] = 0, 30
    whole = torch.cat([(whole + o).to(dtype) for o in (0, -15, -31, 40, -90)], 1)
    x = torch.cat((x, whole), 1).contiguous()
    t = x.shape[1]
    tiles, where, total = ref.pages(t, 64, torch.Generator().manual_seed(2))
    pools = [torch.zeros((total, hkv, 64, ref.row_bytes(d)), dtype=torch.uint8, device=DEV) for _ in range(2)]
    int4.write_int4(x, x, *pools, where.to(torch.int32).contiguous())
    rows = ref.rows_of(x)
    for pool in pools:
        assert torch.equal(pool[where[:, 0], :, where[:, 1]].transpose(0, 1), rows)
    values = int4.gather_int4(*pools, tiles, t, dtype)[0]
    assert torch.equal(values, ref.values_of(rows, d, dtype)) and torch.isfinite(values).all()
    int4.rotate_keys_int4([pools[0]], tiles, 0, torch.ones(d // 2), dtype)
    assert torch.equal(pools[0][where[:, 0], :, where[:, 1]].transpose(0, 1), ref.rows_of(values))
