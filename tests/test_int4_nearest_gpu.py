"""Codes of 4-bit rows are those of the nearest levels, also for elements a hair beside a border between two of them, and a row's
bytes do not depend on the rows that are quantised beside it."""
import pytest
import torch

import int4_ref as ref
from threadcut_b200 import int4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def written(x, page_rows=64):
    """Rows x [hkv, t, d] after write_int4 into pages, [hkv, t, row bytes] (keys; the values' are checked to be the same)."""
    hkv, t, d = x.shape
    at = torch.arange(t, device=DEV)
    slots = torch.stack((at // page_rows, at % page_rows), 1).to(torch.int32).contiguous()
    pools = [torch.zeros(-(-t // page_rows), hkv, page_rows, ref.row_bytes(d), dtype=torch.uint8, device=DEV) for _ in range(2)]
    int4.write_int4(x, x, *pools, slots)
    rows = [p[at // page_rows, :, at % page_rows].transpose(0, 1) for p in pools]
    assert torch.equal(*rows)
    return rows[0]


def rows_of(x):
    """x [..., d] as 4-bit rows, codes by comparison with the borders S (33 + 2 j) / 32 + z, which float64 holds exactly (ref.rows_of's
    quotients have 2^-48 of a level at most, and call an element nearer to a border than that one on it)."""
    _, s, z = ref.quantise64(x)
    g, sd, zd = x.unflatten(-1, (-1, 32)).double(), s.double().unsqueeze(-1), z.double().unsqueeze(-1)
    code = torch.zeros(g.shape, dtype=torch.uint8, device=x.device)
    for j in range(15):
        border = sd * ((33 + 2 * j) / 32) + zd
        code += (g > border) | ((g == border) & (j % 2 == 1))
    return ref.pack_rows(code.masked_fill(sd == 0, 0).flatten(-2), s, z)


def codes_of(rows, d):
    return torch.stack((rows[..., :d // 2] & 15, rows[..., :d // 2] >> 4), -1).flatten(-2)


def test_an_element_a_hair_beside_a_border():
    # 6.500003 levels above the lowest
    x = torch.zeros(1, 1, 64, dtype=HF, device=DEV)
    x[..., 0], x[..., 1], x[..., 2] = -1.9833984375, 2.59765625, 0.0008554458618164062
    rows = written(x)
    assert codes_of(rows, 64)[0, 0, 2] == 7 and torch.equal(rows, ref.rows_of(x))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_zero_on_a_border(dtype):
    """Groups from -(j + 1/2) to 14 1/2 - j steps: S = 16 steps, z = -(j + 16 1/2) steps, exactly, and zero lies between levels
    j and j + 1. Whatever is above it, however little, is j + 1; whatever is below j; zero itself the even one."""
    tiny = [2.0 ** -e for e in ((2, 9, 15, 20, 24) if dtype == HF else (2, 9, 15, 20, 30, 60, 100, 133))]
    steps = [1.0, 0.5, 64.0] + ([] if dtype == HF else [2.0 ** 100, 2.0 ** 118, 2.0 ** -90])
    rows, want = [], []
    for j in range(15):
        for step in steps:
            some = [v for v in tiny if v < 0.4 * step]
            x = torch.zeros(64, dtype=torch.float64)
            x[0], x[1] = -(j + 0.5) * step, (14.5 - j) * step
            code = torch.full((64,), j + j % 2)
            code[0], code[1] = 0, 15
            for i, v in enumerate(some):
                x[2 + 2 * i], x[3 + 2 * i] = v, -v
                code[2 + 2 * i], code[3 + 2 * i] = j + 1, j
            x[32:], code[32:] = x[:32], code[:32]
            rows.append(x)
            want.append(code)
    x, want = torch.stack(rows).to(dtype).to(DEV)[None], torch.stack(want).to(DEV)
    assert torch.equal(codes_of(written(x), 64)[0].long(), want)


def close_to_borders(dtype, n, d, seed):
    """Rows of normal elements, a part of them tiny; of whole numbers, some with a tiny rest; and of values spread between ends
    whose border lies near zero."""
    g = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    def some(share):
        return torch.rand(n, d, generator=g) < share

    tiny = normal(n, d) * torch.exp2(-torch.randint(0, 41, (n, d), generator=g).double())
    a = torch.where(some(0.25), tiny, normal(n, d))
    whole = torch.randint(-15, 16, (n, d), generator=g).double()
    b = torch.where(some(0.25), tiny, whole + torch.where(some(0.3), tiny, torch.zeros(())))
    hi = 1 + torch.rand(n, d // 32, 1, generator=g, dtype=torch.float64)
    j = torch.randint(0, 15, (n, d // 32, 1), generator=g).double()
    c = hi / 15 * (15 * torch.rand(n, d // 32, 32, generator=g, dtype=torch.float64) - j - 0.5)
    c[..., :1], c[..., 1:2] = -hi / 15 * (j + 0.5), hi / 15 * (14.5 - j)
    c = torch.where(some(0.3).view(n, -1, 32) & (torch.arange(32) > 1), tiny.view(n, -1, 32), c).flatten(1)
    return torch.cat((a, b, c)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (HF, 64), (BF, 256)])
def test_rows_close_to_borders(dtype, d):
    x = close_to_borders(dtype, 9000, d, 3).view(3, 9000, d)
    want = rows_of(x)
    assert torch.equal(written(x), want)          # many tokens
    for a in range(0, 9000, 3000):                # and few
        assert torch.equal(written(x[:, a:a + 100]), want[:, a:a + 100])
    # values read back and quantised again by a rotation of nothing
    values = ref.values_of(want, d, dtype)
    pool = want.reshape(-1, 1, 50, ref.row_bytes(d)).contiguous()
    tiles = torch.tensor([[p, r, min(32, 50 - r)] for p in range(pool.shape[0]) for r in (0, 32)], dtype=torch.int32, device=DEV)
    int4.rotate_keys_int4([pool], tiles, 0, torch.ones(d // 2), dtype)
    assert torch.equal(pool.view(want.shape), rows_of(values))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 256])
def test_bytes_do_not_depend_on_the_rows_beside(dtype, d):
    x = close_to_borders(dtype, 100, d, 4)[None]
    alone = written(x)
    for other in (float("nan"), 0.0, 1e4):
        mixed = x.clone()
        mixed[:, ::2] = other
        if other == 1e4:  # far from zero for their spread
            mixed[:, ::2, ::3] += 64
        assert torch.equal(written(mixed)[:, 1::2], alone[:, 1::2])
