"""The 4-bit number format in plain torch and float64, for the tests."""
import torch

GROUP = 32


def row_bytes(d):
    return d // 2 + d // 8


def quantise64(x, group=GROUP):
    """x [..., d] of a 16-bit type (d a multiple of group) -> codes uint8 [..., d], S and z [..., d / group]: nearest levels
    in float64, ties to the even code."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.float().amin(-1), g.float().amax(-1)
    # (a tensor of divisors: by a number, torch's CUDA division is a product with its rounded reciprocal, which turned an S of
    # exactly 0x1.9dp87 into 0x1.9ep87 in bf16, where the even neighbour is 0x1.9cp87)
    s = ((hi - lo) / torch.full_like(hi, 0.9375)).to(x.dtype)
    z = (lo - s.float()).to(x.dtype)
    sd, zd = s.double().unsqueeze(-1), z.double().unsqueeze(-1)
    c = ((g.double() - zd) / sd * 16 - 16).round().clamp(0, 15).masked_fill(sd == 0, 0).nan_to_num(0)
    return c.to(torch.uint8).flatten(-2), s, z


def pack_rows(codes, s, z):
    return torch.cat((codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack((s, z), -1).flatten(-2).view(torch.uint8)), -1)


def rows_of(x):
    """x [..., d] as 4-bit rows uint8 [..., row_bytes(d)]."""
    return pack_rows(*quantise64(x))


def values_of(rows, d, dtype):
    """The values of 4-bit rows, of `dtype`: one rounding of the exact S (1 + code/16) + z."""
    codes = torch.stack((rows[..., :d // 2] & 15, rows[..., :d // 2] >> 4), -1).flatten(-2).double()
    p = rows[..., d // 2:].contiguous().view(dtype).double().unflatten(-1, (-1, 2)).repeat_interleave(GROUP, -2)
    return (p[..., 0] * (1 + codes / 16) + p[..., 1]).to(dtype)


def rotate32(x, cos, sin):
    """Rotate-half of the first cos.shape[-1] elements in elementary fp32 operations, rounded to x's type."""
    dt, rot = x.dtype, cos.shape[-1]
    x, cos, sin = x.float(), cos.float(), sin.float()
    head, rest = x[..., :rot], x[..., rot:]
    half = torch.cat((-head[..., rot // 2:], head[..., :rot // 2]), -1)
    return torch.cat((head * cos + half * sin, rest), -1).to(dt)


def pages(n, page_rows, gen, cuts=3, device="cuda"):
    """A sequence of n tokens over shuffled pages whose runs begin and end inside pages, as splices leave it. Returns
    (tiles int32 [T, 4], (page, row) of each token int64 [n, 2], pages in the pool)."""
    runs, left, page = [], n, 0
    while left > 0:
        a = int(torch.randint(0, page_rows, (1,), generator=gen)) if len(runs) < cuts else 0
        m = min(left, int(torch.randint(1, page_rows - a + 1, (1,), generator=gen)) if len(runs) < cuts else page_rows)
        runs.append([page, a, m])
        left -= m
        page += 1
    total = page + 2
    order = torch.randperm(total, generator=gen).tolist()
    tab, where, pos = [], [], 0
    for p, a, m in runs:
        for o in range(0, m, 32):
            k = min(32, m - o)
            tab.append((order[p], a + o, k, pos))
            where += [(order[p], a + o + i) for i in range(k)]
            pos += k
    return (torch.tensor(tab, dtype=torch.int32).reshape(-1, 4).to(device),
            torch.tensor(where, dtype=torch.int64).reshape(-1, 2).to(device), total)
