"""Timed cases of the 4-bit serving operators: a KV cache and weights held in 4 bits with group scales.

Each operator in its plain form (elementary torch operations in fp32, rounded once) and as the call a
user makes:

  store   normalise (optional) and rotate a step's queries and keys, write keys and values as 4-bit
          rows into the slots of a paged cache, and read rows back as 16-bit values: the new ones, or
          the whole sequence as a prefill chunk does      threadcut_b200.int4.append_rope_int4, gather_int4
  prune   write a span of rows, rotate its keys in place by the length of the span that was cut before
          it, and read it back                            write_int4, rotate_keys_int4, gather_int4
  attend  one query token of each sequence over a 4-bit cache, contiguous with lengths, or in pages
                                                          decode_attention_int4
  gemv    a few tokens times a 4-bit weight matrix        gemv_int4

The number format. A group of neighbouring elements (32 of a cache row, 32, 64 or 128 of a weight row)
has a scale S and an offset z of the 16-bit type T, and a code of 0..15 an element that stands for
S (1 + code / 16) + z. A cache row of d elements is d / 2 bytes of codes (element e in byte e / 2, the
even one in the low half), then d / 32 pairs (S, z); its values are rounded to T. Weights lie in tiles of
16 rows and 64 columns of 512 bytes, their pairs (S, z) as [row tile][group][row % 8][row / 8].

Sizes are those of this repository's workloads (32 query and 8 KV heads of 128, caches of 1,536 to
98,304 tokens, 64 ragged sequences of 1,024 to 16,384, projections of hidden size 2,560), and odd ones.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"
EPS = 1e-6
THETA = 1.0e6
GROUP = 32  # elements of a cache row that share a scale


def listed():
    return [
        # one decode step: 32 + 8 + 8 heads of one token, with q/k norm
        dict(name="store_step", op="store", dtype="bf16", table="same", hq=32, hkv=8, d=128, rot=128, t=1, n0=0, norm=True,
             page_rows=64),
        # an odd chunk of a model that rotates half of each 64-element head, fp32 tables
        dict(name="store_partial_rot", op="store", dtype="fp16", table="fp32", hq=16, hkv=4, d=64, rot=32, t=517, n0=333,
             norm=False, page_rows=96),
        # a whole prompt written at once and read back for its prefill
        dict(name="store_prompt", op="store", dtype="bf16", table="same", hq=32, hkv=8, d=128, rot=128, t=16384, n0=0,
             norm=False, page_rows=64),
        # a chunk behind the longest context, all of which its prefill reads
        dict(name="store_chunk", op="store", dtype="bf16", table="same", hq=32, hkv=8, d=128, rot=128, t=512, n0=97792,
             norm=False, page_rows=64),
        # a short span moved by an odd gap
        dict(name="prune_odd", op="prune", dtype="fp16", hkv=4, d=64, c=701, gap=333, page_rows=96),
        # the suffix that follows the cut of a long context
        dict(name="prune_suffix", op="prune", dtype="bf16", hkv=8, d=128, c=49152, gap=32768, page_rows=64),
        # one short sequence in pages: latency
        dict(name="attend_step", op="attend", dtype="bf16", b=1, hkv=8, g=4, d=128, n=1536, lo=1536, page_rows=64),
        # the longest context in pages
        dict(name="attend_context", op="attend", dtype="bf16", b=1, hkv=8, g=4, d=128, n=98304, lo=98304, page_rows=64),
        # the 64 ragged sequences, contiguous
        dict(name="attend_batch", op="attend", dtype="fp16", b=64, hkv=8, g=4, d=128, n=16384, lo=1024, page_rows=0),
        # one token through the attention output projection: latency
        dict(name="gemv_out", op="gemv", dtype="bf16", m=1, n=2560, k=4096, group=64),
        # one token through the gate and up projections
        dict(name="gemv_gate_up", op="gemv", dtype="bf16", m=1, n=19456, k=2560, group=64),
        # a few sequences' tokens through the vocabulary projection
        dict(name="gemv_vocabulary", op="gemv", dtype="fp16", m=7, n=151936, k=2560, group=128),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "prune", "attend", "attend", "gemv", "gemv"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    rows = rng.choice([32, 64, 100])
    if op == "store":
        # short chunks of models with q/k norm, chunks and prompts of the others
        norm = rng.random() < 0.4
        return dict(op=op, dtype=dtype, table=rng.choice(["same", "fp32"]), hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=d,
                    rot=rng.choice([32, 64]), t=_log(rng, 1, 100 if norm else 12000), n0=_log(rng, 1, 20000), norm=norm,
                    page_rows=rows)
    if op == "prune":
        return dict(op=op, dtype=dtype, hkv=hkv, d=d, c=_log(rng, 1, 20000), gap=_log(rng, 1, 60000), page_rows=rows)
    if op == "attend":
        paged = rng.random() < 0.5
        n = _log(rng, 1, 60000 if paged else 20000)
        return dict(op=op, dtype=dtype, b=1 if paged else _log(rng, 1, 24), hkv=hkv, g=rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]),
                    d=d, n=n, lo=n if paged else rng.randint(0, n), page_rows=rows if paged else 0)
    return dict(op=op, dtype=dtype, m=_log(rng, 1, 32), n=_log(rng, 1, 40000), k=_log(rng, 16, 12000),
                group=rng.choice([32, 64, 128]))


def _runs(n, rows, gen):
    """A sequence of n tokens in pages of `rows` rows, as pruning leaves it: it begins inside its first page, and near
    its middle a page ends early and the next run begins inside its own. Returns [(page, first row, rows)], pages."""
    first, cut, skip = (int(x) for x in torch.randint(0, rows, (3,), generator=gen, device=DEV).tolist())
    sizes, left, middle = [], n, n // 2
    while left > 0:
        start = first if not sizes else 0
        size = min(rows - start, left)
        if middle is not None and n - left >= middle:
            size, middle = min(size, cut + 1), None
            sizes.append((start, size))
            left -= size
            if left > 0:
                sizes.append((skip, min(rows - skip, left)))
                left -= sizes[-1][1]
            continue
        sizes.append((start, size))
        left -= size
    pages = len(sizes) + 2
    order = torch.randperm(pages, generator=gen, device=DEV).tolist()
    return [(order[i], s, m) for i, (s, m) in enumerate(sizes)], pages


def _tiles(runs):
    """int32 [T, 4]: page, first row, rows (32 at most) and position of the first row."""
    runs = np.asarray(runs, np.int64).reshape(-1, 3)
    count = (runs[:, 2] + 31) // 32
    at = np.repeat(np.arange(len(runs)), count)
    off = (np.arange(len(at)) - np.repeat(np.cumsum(count) - count, count)) * 32
    size = np.minimum(32, runs[at, 2] - off)
    tab = np.stack((runs[at, 0], runs[at, 1] + off, size, np.cumsum(size) - size), axis=1)
    return torch.from_numpy(tab.astype(np.int32)).to(DEV)


def _places(tiles, n):
    """Page and row of tokens 0..n-1."""
    pos = torch.arange(n, device=DEV)
    at = torch.searchsorted(tiles[:, 3].long().contiguous(), pos, right=True) - 1
    return tiles[at, 0].long(), tiles[at, 1].long() + pos - tiles[at, 3].long()


def _random_rows(shape, d, dt, gen):
    """Cache rows of roughly normal data: bell-shaped codes under a group's own scale and offset."""
    codes = torch.randn(*shape, d, generator=gen, device=DEV, dtype=torch.float16).mul_(3.6).add_(7.5).round_().clamp_(0, 15)
    codes = codes.to(torch.uint8)
    lo = -2.1 + 0.3 * torch.randn(*shape, d // GROUP, generator=gen, device=DEV)
    step = 0.28 * (0.7 + 0.6 * torch.rand(*shape, d // GROUP, generator=gen, device=DEV))
    scale = (16 * step).to(dt)
    return _pack(codes, scale, (lo - scale.float()).to(dt))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dt)

    op = case["op"]
    if op == "gemv":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        tiles, blocks, groups = -(-n // 16), -(-k // 64), -(-k // group)
        # weights of an initialised projection, standard deviation 0.02; what lies behind n and k is zero
        codes = torch.randn(n, k, generator=gen, device=DEV, dtype=torch.float16).mul_(3.6).add_(7.5).round_().clamp_(0, 15)
        full = torch.zeros(16 * tiles, 64 * blocks, device=DEV, dtype=torch.uint8)
        full[:n, :k] = codes.to(torch.uint8)
        scale = torch.zeros(16 * tiles, groups, device=DEV, dtype=dt)
        offset = torch.zeros_like(scale)
        step = 0.0056 * (0.7 + 0.6 * torch.rand(n, groups, generator=gen, device=DEV))
        scale[:n] = (16 * step).to(dt)
        offset[:n] = (-0.042 + 0.006 * torch.randn(n, groups, generator=gen, device=DEV) - scale[:n].float()).to(dt)
        return dict(op=op, x=normal(m, k), n=n, k=k, group=group, codes=_lay_codes(full), params=_lay_params(scale, offset))
    hkv, d = case["hkv"], case["d"]
    if op == "attend":
        b, g, n = case["b"], case["g"], case["n"]
        s = dict(op=op, scale=d ** -0.5, d=d, dtype=dt, tiles=None, lengths=None)
        if case["page_rows"]:
            runs, pages = _runs(n, case["page_rows"], gen)
            s["tiles"] = _tiles(runs)
            s["q"], shape = normal(hkv, g, d), (pages, hkv, case["page_rows"])
        else:
            lens = torch.randint(case["lo"], n + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
            lens[0] = n
            s["q"], s["lengths"], shape = normal(b, hkv, g, d), lens, (b, hkv, n + 40)
        s["k"], s["v"] = _random_rows(shape, d, dt, gen), _random_rows(shape, d, dt, gen)
        if not case["page_rows"]:
            # buffers with room to grow, as a cache keeps them
            s["k"], s["v"] = s["k"][:, :, :n], s["v"][:, :, :n]
        return s
    if op == "prune":
        c = case["c"]
        runs, pages = _runs(c, case["page_rows"], gen)
        tiles = _tiles(runs)
        page, row = _places(tiles, c)
        pool = [torch.zeros(pages, hkv, case["page_rows"], d // 2 + d // 8, device=DEV, dtype=torch.uint8) for _ in range(2)]
        return dict(op=op, k=normal(hkv, c, d), v=normal(hkv, c, d), k_pool=pool[0], v_pool=pool[1], tiles=tiles, n=c, d=d,
                    dtype=dt, slots=torch.stack((page, row), 1).to(torch.int32).contiguous(), delta=-case["gap"],
                    inv_freq=THETA ** (-torch.arange(0, d, 2).float() / d))
    hq, t, n0 = case["hq"], case["t"], case["n0"]
    # the fused projection's output, one row a token; q, k and v are views of it
    qkv = normal(t, hq + 2 * hkv, d).transpose(0, 1)
    runs, pages = _runs(n0 + t, case["page_rows"], gen)
    tiles = _tiles(runs)
    page, row = _places(tiles, n0 + t)
    slots = torch.stack((page[n0:], row[n0:]), 1).to(torch.int32).contiguous()
    shape = (pages, hkv, case["page_rows"])
    at = torch.arange(n0, n0 + t, device=DEV).double()
    inv = THETA ** (-torch.arange(0, case["rot"], 2, device=DEV).double() / case["rot"])
    angle = torch.cat((at[:, None] * inv, at[:, None] * inv), dim=1)
    tab = dt if case["table"] == "same" else torch.float32
    weight = [(1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).to(dt) for _ in range(2)]
    return dict(op=op, q=qkv[:hq], k=qkv[hq:hq + hkv], v=qkv[hq + hkv:], cos=angle.cos().to(tab), sin=angle.sin().to(tab),
                slots=slots, k_pool=_random_rows(shape, d, dt, gen), v_pool=_random_rows(shape, d, dt, gen), tiles=tiles,
                n=n0 + t, d=d, dtype=dt, q_norm=weight[0] if case["norm"] else None,
                k_norm=weight[1] if case["norm"] else None)


# ------------------------------------------------------------------ plain forms
def _pack(codes, scale, offset):
    """Rows of bytes from codes [..., d] and the groups' (S, z) [..., d / 32]."""
    params = torch.stack((scale, offset), -1).flatten(-2).view(torch.uint8)
    return torch.cat((codes[..., 0::2] | (codes[..., 1::2] << 4), params), dim=-1)


def _quantised(x):
    """x [..., d] as rows of bytes."""
    g = x.unflatten(-1, (-1, GROUP)).float()
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 0.9375).to(x.dtype)
    offset = (lo - scale.float()).to(x.dtype)
    s, z = scale.double().unsqueeze(-1), offset.double().unsqueeze(-1)
    # the nearest level, ties to the even one: in 64 bits, as many elements lie on a border
    codes = ((g.double() - z) / s * 16 - 16).round().clamp(0, 15).masked_fill(s == 0, 0)
    return _pack(codes.to(torch.uint8).flatten(-2), scale, offset)


def _values(rows, d, dt):
    """The values of rows of bytes, in fp32 after their rounding to the cache's type."""
    codes = torch.stack((rows[..., :d // 2] & 15, rows[..., :d // 2] >> 4), -1).flatten(-2)
    params = rows[..., d // 2:].contiguous().view(dt).unflatten(-1, (-1, 1, 2)).float()
    x = params[..., 0] * (1 + codes.unflatten(-1, (-1, GROUP)).float() / 16) + params[..., 1]
    return x.to(dt).float().flatten(-2)


def _norm_rotate(x, weight, cos, sin):
    """x [h, t, d]: RMSNorm over d (with a weight), then the rotate-half rotation of the first elements."""
    dt, x, cos, sin = x.dtype, x.float(), cos.float(), sin.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    rot = cos.shape[-1]
    head, rest = x[..., :rot], x[..., rot:]
    half = torch.cat((-head[..., rot // 2:], head[..., :rot // 2]), dim=-1)
    return torch.cat((head * cos + half * sin, rest), dim=-1).to(dt)


def _write(s, k, v):
    page, row = s["slots"][:, 0].long(), s["slots"][:, 1].long()
    s["k_pool"][page, :, row] = _quantised(k).transpose(0, 1)
    s["v_pool"][page, :, row] = _quantised(v).transpose(0, 1)


def _read(s):
    page, row = _places(s["tiles"], s["n"])
    return [_values(s[p][page, :, row], s["d"], s["dtype"]).transpose(0, 1).contiguous().to(s["dtype"])
            for p in ("k_pool", "v_pool")]


def _store(s):
    q = _norm_rotate(s["q"], s["q_norm"], s["cos"], s["sin"])
    _write(s, _norm_rotate(s["k"], s["k_norm"], s["cos"], s["sin"]), s["v"])
    return [q] + _read(s)


def _prune(s):
    _write(s, s["k"], s["v"])
    page, row = _places(s["tiles"], s["n"])
    keys = _values(s["k_pool"][page, :, row], s["d"], s["dtype"])
    angle = s["delta"] * s["inv_freq"]  # fp32, on the host
    cos, sin = (torch.cat((x, x)).to(DEV) for x in (angle.cos(), angle.sin()))
    half = torch.cat((-keys[..., s["d"] // 2:], keys[..., :s["d"] // 2]), dim=-1)
    s["k_pool"][page, :, row] = _quantised((keys * cos + half * sin).to(s["dtype"]))
    return _read(s)


def _softmax(x):
    """Softmax over the last axis of scores masked with -inf; a row with nothing visible gives zeros."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _attend(s):
    q, k, v = s["q"].float(), s["k"], s["v"]
    if s["tiles"] is not None:
        n = int(s["tiles"][-1, 2:].sum())
        page, row = _places(s["tiles"], n)
        k, v = (x[page, :, row].transpose(0, 1) for x in (k, v))
    x = (q @ _values(k, s["d"], s["dtype"]).transpose(-1, -2)) * s["scale"]
    if s["lengths"] is not None:
        seen = torch.arange(x.shape[-1], device=DEV) < s["lengths"][:, None]
        x = x.masked_fill(~seen[:, None, None], -math.inf)
    return (_softmax(x) @ _values(v, s["d"], s["dtype"])).to(s["q"].dtype)


SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]  # of a word's 8 codes, in the order of their columns


def _lay_codes(codes):
    """Codes [16 R, 64 C] as tiles [R, C, 512]: lane 4 r + c's 16 bytes are the words of (row r, columns 8 c..),
    (row r + 8, the same), (row r, columns 32 + 8 c..), (row r + 8, the same)."""
    rows, cols = codes.shape
    x = codes.view(rows // 16, 2, 8, cols // 64, 2, 4, 8).permute(0, 3, 2, 5, 4, 1, 6)
    # bytes of a word, lowest first: columns (0, 2), (4, 6), (1, 3), (5, 7)
    low, high = x[..., [0, 4, 1, 5]], x[..., [2, 6, 3, 7]]
    return (low | (high << 4)).reshape(rows // 16, cols // 64, 512)


def _lay_params(scale, offset):
    """(S, z) [16 R, groups] as [R, groups, 8, 2, 2]."""
    rows, groups = scale.shape
    return torch.stack((scale, offset), -1).view(rows // 16, 2, 8, groups, 2).permute(0, 3, 2, 1, 4).contiguous()


def _gemv(s):
    tiles, blocks, _ = s["codes"].shape
    words = s["codes"].view(torch.int32).view(tiles, blocks, 8, 4, 2, 2)
    shifts = torch.tensor(SHIFTS, device=DEV, dtype=torch.int32)
    codes = ((words[..., None] >> shifts) & 15).permute(0, 5, 2, 1, 4, 3, 6).reshape(16 * tiles, 64 * blocks)
    params = s["params"].float().permute(0, 3, 2, 1, 4).reshape(16 * tiles, -1, 2)
    scale, offset = (params[..., i].repeat_interleave(s["group"], 1)[:s["n"], :s["k"]] for i in (0, 1))
    weight = scale * (1 + codes[:s["n"], :s["k"]].float() / 16) + offset
    return (s["x"].float() @ weight.t()).to(s["x"].dtype)


def run(state):
    s, op = state, state["op"]
    if own:
        from threadcut_b200 import int4
    if op == "store":
        if not own:
            return _store(s)
        q = int4.append_rope_int4(s["k"], s["v"], s["cos"], s["sin"], s["k_pool"], s["v_pool"], s["slots"], q=s["q"],
                                  q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return q, *int4.gather_int4(s["k_pool"], s["v_pool"], s["tiles"], s["n"], s["dtype"])
    if op == "prune":
        if not own:
            return _prune(s)
        int4.write_int4(s["k"], s["v"], s["k_pool"], s["v_pool"], s["slots"])
        int4.rotate_keys_int4([s["k_pool"]], s["tiles"], s["delta"], s["inv_freq"], s["dtype"])
        return int4.gather_int4(s["k_pool"], s["v_pool"], s["tiles"], s["n"], s["dtype"])
    if op == "attend":
        if not own:
            return _attend(s)
        return int4.decode_attention_int4(s["q"], s["k"], s["v"], s["scale"], s["lengths"], tiles=s["tiles"])
    if not own:
        return _gemv(s)
    return int4.gemv_int4(s["x"], int4.Int4Weight(s["codes"], s["params"], s["n"], s["k"], s["group"]))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "gemv":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 4 * n * -(-k // case["group"]) + 2 * m * (n + k), "flops": 2 * m * n * k}
    hkv, d = case["hkv"], case["d"]
    row = 5 * d // 8
    if op == "attend":
        b, g = case["b"], case["g"]
        # the lengths are spread evenly over lo..n, the first of them n
        rows = case["n"] + (b - 1) * (case["lo"] + case["n"]) / 2
        return {"bytes": 2 * rows * hkv * row + 4 * b * hkv * g * d + 4 * b, "flops": 4 * rows * hkv * g * d}
    if op == "prune":
        c = case["c"]
        # rows written once (the keys' after their rotation), and read back as 16-bit values
        return {"bytes": 2 * hkv * c * (2 * d + row + 2 * d), "flops": 2 * hkv * c * d * 10}
    hq, t, n, rot = case["hq"], case["t"], case["n0"] + case["t"], case["rot"]
    tab = 4 if case["table"] == "fp32" else 2
    new = (2 * hq + 2 * hkv) * t * d * 2 + 2 * hkv * t * row + 2 * t * rot * tab + 8 * t + (4 * d if case["norm"] else 0)
    old = 2 * hkv * case["n0"] * row
    return {"bytes": new + old + 2 * hkv * n * d * 2,
            "flops": (hq + hkv) * t * (3 * rot + (4 * d if case["norm"] else 0)) + 2 * hkv * (t * 8 + n * 2) * d}


# ------------------------------------------------------------------ the definitions in 64 bits
def _levels64(x, dt):
    """What x (float64 values of type dt) reads back as, in float64."""
    out = torch.empty_like(x)
    for a in range(0, x.shape[-1], GROUP):
        g = x[..., a:a + GROUP]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        scale = ((high - low) * (16 / 15)).to(dt).double()
        zero = (low - scale).to(dt).double()
        level = torch.where(scale > 0, torch.round(16 * ((g - zero) / torch.where(scale > 0, scale, 1.0) - 1)), 0.0)
        out[..., a:a + GROUP] = (scale + scale * torch.clamp(level, 0, 15) / 16 + zero).to(dt).double()
    return out


def _bytes64(rows, d, dt):
    """Values of rows of bytes, in float64."""
    out = torch.empty(*rows.shape[:-1], d, dtype=torch.float64, device=rows.device)
    for a in range(d // GROUP):
        p = rows[..., d // 2 + 4 * a:d // 2 + 4 * a + 4].contiguous().view(dt).double()
        byte = rows[..., GROUP // 2 * a:GROUP // 2 * (a + 1)].double()
        high = torch.floor(byte / 16)
        for e, level in ((0, byte - 16 * high), (1, high)):
            out[..., GROUP * a + e:GROUP * (a + 1):2] = (p[..., :1] * (16 + level) / 16 + p[..., 1:]).to(dt).double()
    return out


def _sequence(tiles, pool):
    return torch.cat([pool[p, :, r:r + m] for p, r, m, _ in tiles.tolist()], dim=1)


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "gemv":
        # the tiles again, lane by lane
        n, k, group, dt = case["n"], case["k"], case["group"], s["x"].dtype
        tiles, blocks, _ = s["codes"].shape
        byte = s["codes"].view(tiles, blocks, 32, 4, 4)
        w = torch.zeros(tiles, 16, blocks, 64, dtype=torch.float64, device=DEV)
        for lane in range(32):
            r, c = lane // 4, lane % 4
            for word in range(4):
                for e in range(8):
                    bit = 4 * (e // 2) + 16 * (e % 2)
                    code = (byte[:, :, lane, word, bit // 8] >> (bit % 8)) & 15
                    w[:, r + 8 * (word % 2), :, 32 * (word // 2) + 8 * c + e] = code.double()
        w = w.view(16 * tiles, 64 * blocks)[:n, :k]
        y = torch.zeros(case["m"], n, dtype=torch.float64, device=DEV)
        p = s["params"].double()
        for i in range(p.shape[1]):
            x = s["x"][:, i * group:(i + 1) * group].double()
            rows = p[:, i].transpose(1, 2).reshape(16 * tiles, 2)[:n]
            part = w[:, i * group:(i + 1) * group] @ x.t()
            y += ((part / 16 + x.sum(1)) * rows[:, :1] + x.sum(1) * rows[:, 1:]).t()
        return y
    hkv, d, dt = case["hkv"], case["d"], s["dtype"]
    if op == "attend":
        b, g = case["b"], case["g"]
        out = torch.zeros(b, hkv, g, d, dtype=torch.float64, device=DEV)
        for i in range(b):
            if s["tiles"] is not None:
                rows = [_sequence(s["tiles"], x) for x in (s["k"], s["v"])]
            else:
                rows = [x[i, :, :int(s["lengths"][i])] for x in (s["k"], s["v"])]
            if rows[0].shape[1] == 0:
                continue
            q = s["q"].view(b, hkv, g, d)[i].double()
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, _bytes64(rows[0], d, dt)) * s["scale"], dim=2)
            out[i] = torch.einsum("hgn,hnd->hgd", p, _bytes64(rows[1], d, dt))
        return out.view(s["q"].shape)
    if op == "prune":
        keys = _levels64(s["k"].double(), dt)
        angle = (s["delta"] * s["inv_freq"]).double().to(DEV)  # the angle itself is a 32-bit number
        a, c = keys[..., :d // 2], keys[..., d // 2:]
        keys = torch.cat((a * angle.cos() - c * angle.sin(), c * angle.cos() + a * angle.sin()), -1).to(dt).double()
        return _levels64(keys, dt), _levels64(s["v"].double(), dt)
    cos, sin, rot = s["cos"].double(), s["sin"].double(), case["rot"]

    def turn(x, w):
        x = x.double().clone()
        if w is not None:
            x = w.double() * x / torch.sqrt((x * x).sum(2, keepdim=True) / d + EPS)
        a, c = x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone()
        x[..., :rot // 2] = a * cos[:, :rot // 2] - c * sin[:, :rot // 2]
        x[..., rot // 2:rot] = c * cos[:, rot // 2:] + a * sin[:, rot // 2:]
        return x

    n0 = case["n0"]
    new = [_levels64(turn(s["k"], s["k_norm"]).to(dt).double(), dt), _levels64(s["v"].double(), dt)]
    old = [_bytes64(_sequence(s["tiles"], s[x])[:, :n0], d, dt) for x in ("k_pool", "v_pool")]
    return turn(s["q"], s["q_norm"]), torch.cat((old[0], new[0]), 1), torch.cat((old[1], new[1]), 1)
