"""Timed cases of the serving operators over a shared, windowed or paged KV cache.

Three operators of the decode and prefill loop of a coding agent's long context, each in its plain
form (elementary torch operations in fp32, rounded once) and as the call a user makes:

  append   normalise (optional) and rotate a step's queries and keys, write keys and values into
           the slots of a paged cache                      threadcut_b200.paged.append_rope
  window   attention with a sliding window whose first `sinks` tokens stay visible: one query token
           per sequence                                    threadcut_b200.flash_decode.decode_attention_window
           and a chunk of queries over the cache           threadcut_b200.prefill.prefill_attention_window
  shared   one query token of each of `b` continuations of one cached prefix, each with its own
           suffix                                          threadcut_b200.flash_decode.decode_attention_shared

The head counts (32 query and 8 KV heads of 128), the 1,536-, 16,384- and 98,304-token caches and the
64 ragged sequences of 1,024 to 16,384 tokens are those of this repository's workloads.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"
EPS = 1e-6
THETA = 1.0e6


def listed():
    return [
        # one decode step: 32 + 8 + 8 heads of one token, with q/k norm
        dict(name="append_step", op="append", dtype="bf16", table="same", hq=32, hkv=8, d=128, rot=128, t=1, norm=True,
             page_rows=64),
        # an odd chunk of a model that rotates half of each 64-element head, fp32 tables
        dict(name="append_partial_rot", op="append", dtype="fp16", table="fp32", hq=16, hkv=4, d=64, rot=32, t=517,
             norm=False, page_rows=96),
        # a whole prompt written at once
        dict(name="append_prompt", op="append", dtype="bf16", table="same", hq=32, hkv=8, d=128, rot=128, t=16384,
             norm=True, page_rows=64),
        # one token of one long sequence: latency
        dict(name="window_step", op="window_decode", dtype="bf16", b=1, hkv=8, g=4, d=128, n=98304, lo=98304,
             window=4096, sinks=4),
        # a small odd batch, 64-element heads, unaligned lengths, some shorter than the window
        dict(name="window_odd", op="window_decode", dtype="fp16", b=7, hkv=4, g=7, d=64, n=3001, lo=1, window=333,
             sinks=5),
        # the 64 ragged sequences
        dict(name="window_batch", op="window_decode", dtype="bf16", b=64, hkv=8, g=4, d=128, n=16384, lo=1024,
             window=2048, sinks=16),
        # a prompt chunk over a long cache
        dict(name="window_chunk", op="window_prefill", dtype="bf16", b=1, hkv=8, g=4, d=128, lq=512, lk=98304,
             window=4096, sinks=4),
        # two odd chunks of a model with 64-element heads
        dict(name="window_chunk_odd", op="window_prefill", dtype="fp16", b=2, hkv=4, g=2, d=64, lq=777, lk=5001,
             window=500, sinks=33),
        # a whole prompt from nothing
        dict(name="window_prompt", op="window_prefill", dtype="bf16", b=1, hkv=8, g=4, d=128, lq=8192, lk=8192,
             window=2048, sinks=0),
        # two samples of a short request
        dict(name="shared_pair", op="shared", dtype="bf16", b=2, hkv=8, g=4, d=128, n=1536, m=40, lo=1),
        # eight sub-agents over one repository context
        dict(name="shared_agents", op="shared", dtype="bf16", b=8, hkv=8, g=4, d=128, n=16384, m=700, lo=100),
        # 64 continuations of the longest context
        dict(name="shared_wide", op="shared", dtype="bf16", b=64, hkv=8, g=4, d=128, n=98304, m=1024, lo=64),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "window_decode", "window_prefill", "shared"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "append":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), table=rng.choice(["same", "fp32"]),
                    hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=rng.choice([64, 128, 256]), rot=rng.choice([32, 64]),
                    t=_log(rng, 1, 12000), norm=rng.random() < 0.5, page_rows=rng.choice([32, 64, 100]))
    if op == "window_decode":
        n = _log(rng, 1, 40000)
        return dict(op=op, dtype=dtype, b=_log(rng, 1, 24), hkv=hkv, g=g, d=d, n=n, lo=rng.randint(0, n),
                    window=_log(rng, 1, 5000), sinks=rng.choice([0, 1, 4, 33, 128]))
    if op == "window_prefill":
        lq = _log(rng, 1, 2500)
        return dict(op=op, dtype=dtype, b=rng.choice([1, 1, 2]), hkv=hkv, g=g, d=d, lq=lq,
                    lk=lq + _log(rng, 1, 40000), window=_log(rng, 1, 5000), sinks=rng.choice([0, 1, 4, 33, 128]))
    n = _log(rng, 1, 60000)
    m = _log(rng, 1, 1500)
    return dict(op=op, dtype=dtype, b=_log(rng, 1, 48), hkv=hkv, g=g, d=d, n=n, m=m, lo=rng.randint(0, m))


def _lengths(case, most, gen):
    lens = torch.randint(case["lo"], most + 1, (case["b"],), generator=gen, device=DEV, dtype=torch.int32)
    lens[0] = most
    return lens


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dt)

    op = case["op"]
    if op == "append":
        hq, hkv, d, t, rows = case["hq"], case["hkv"], case["d"], case["t"], case["page_rows"]
        # the fused projection's output, one row a token; q, k and v are views of it
        qkv = normal(t, hq + 2 * hkv, d).transpose(0, 1)
        # the tokens' slots: the rest of a partly filled page, then pages in the order the pool gave them
        first = int(torch.randint(0, rows, (1,), generator=gen, device=DEV))
        pages = -(-(rows - 1 + t) // rows)
        order = torch.randperm(pages + 2, generator=gen, device=DEV)[:pages]
        at = first + torch.arange(t, device=DEV)
        slots = torch.stack((order[at // rows], at % rows), dim=1).to(torch.int32).contiguous()
        pos = torch.randint(0, 100000, (1,), generator=gen, device=DEV).double() + torch.arange(t, device=DEV).double()
        inv = THETA ** (-torch.arange(0, case["rot"], 2, device=DEV).double() / case["rot"])
        angle = torch.cat((pos[:, None] * inv, pos[:, None] * inv), dim=1)
        tab = dt if case["table"] == "same" else torch.float32
        weight = [(1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).to(dt) for _ in range(2)]
        return dict(op=op, q=qkv[:hq], k=qkv[hq:hq + hkv], v=qkv[hq + hkv:], cos=angle.cos().to(tab),
                    sin=angle.sin().to(tab), slots=slots, k_pool=normal(pages + 2, hkv, rows, d),
                    v_pool=normal(pages + 2, hkv, rows, d), q_norm=weight[0] if case["norm"] else None,
                    k_norm=weight[1] if case["norm"] else None)
    b, hkv, g, d = case["b"], case["hkv"], case["g"], case["d"]
    scale = d ** -0.5
    if op == "window_decode":
        n = case["n"]
        # buffers with room to grow, as a cache keeps them
        return dict(op=op, q=normal(b, hkv, g, d), k=normal(b, hkv, n + 40, d)[:, :, :n],
                    v=normal(b, hkv, n + 40, d)[:, :, :n], lengths=_lengths(case, n, gen), scale=scale,
                    window=case["window"], sinks=case["sinks"])
    if op == "window_prefill":
        lq, lk = case["lq"], case["lk"]
        return dict(op=op, q=normal(b, lq, hkv * g, d).transpose(1, 2), k=normal(b, hkv, lk + 40, d)[:, :, :lk],
                    v=normal(b, hkv, lk + 40, d)[:, :, :lk], scale=scale, window=case["window"], sinks=case["sinks"])
    n, m = case["n"], case["m"]
    return dict(op=op, q=normal(b, hkv, g, d), kp=normal(hkv, n + 40, d)[:, :n], vp=normal(hkv, n + 40, d)[:, :n],
                k=normal(b, hkv, m, d), v=normal(b, hkv, m, d), lengths=_lengths(case, m, gen), scale=scale)


# ------------------------------------------------------------------ plain forms
def _norm_rotate(x, weight, cos, sin):
    """x [h, t, d]: RMSNorm over d (with a weight), then the rotate-half rotation of the first elements."""
    dt, x, cos, sin = x.dtype, x.float(), cos.float(), sin.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    rot = cos.shape[-1]
    head, rest = x[..., :rot], x[..., rot:]
    half = torch.cat((-head[..., rot // 2:], head[..., :rot // 2]), dim=-1)
    return torch.cat((head * cos + half * sin, rest), dim=-1).to(dt)


def _append(s):
    page, row = s["slots"][:, 0].long(), s["slots"][:, 1].long()
    s["k_pool"][page, :, row] = _norm_rotate(s["k"], s["k_norm"], s["cos"], s["sin"]).transpose(0, 1)
    s["v_pool"][page, :, row] = s["v"].transpose(0, 1)
    return _norm_rotate(s["q"], s["q_norm"], s["cos"], s["sin"])


def _softmax(x):
    """Softmax over the last axis of scores masked with -inf; a row with nothing visible gives zeros."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _window_decode(s):
    b, hkv, n, d = s["k"].shape
    # the rows a query sees: the sinks, then the window's, without those counted twice
    size, sinks = min(s["window"], n), min(s["sinks"], n)
    lens = s["lengths"].long()[:, None]
    back = lens - size + torch.arange(size, device=DEV)
    front = torch.arange(sinks, device=DEV).expand(b, -1)
    rows = torch.cat((front, back), dim=1)
    seen = torch.cat((front < (lens - size).clamp(min=0), back >= 0), dim=1)
    at = rows.clamp(min=0)[:, None, :, None].expand(-1, hkv, -1, d)
    k, v = s["k"].gather(2, at).float(), s["v"].gather(2, at).float()
    x = (s["q"].float() @ k.transpose(2, 3)) * s["scale"]
    p = _softmax(x.masked_fill(~seen[:, None, None], -math.inf))
    return (p @ v).to(s["q"].dtype)


def _window_prefill(s):
    b, hq, lq, d = s["q"].shape
    hkv, lk = s["k"].shape[1:3]
    # keys that some query sees: the sinks and everything after the first query's window begins
    first = max(0, lk - lq - s["window"] + 1)
    sinks = min(s["sinks"], first)
    rows = torch.cat((torch.arange(sinks, device=DEV), torch.arange(first, lk, device=DEV)))
    at = (lk - lq + torch.arange(lq, device=DEV))[:, None]
    seen = (rows <= at) & ((rows < s["sinks"]) | (rows > at - s["window"]))
    k, v = s["k"][:, :, rows].float()[:, :, None], s["v"][:, :, rows].float()[:, :, None]
    q = s["q"].float().reshape(b, hkv, hq // hkv, lq, d)
    p = _softmax(((q @ k.transpose(3, 4)) * s["scale"]).masked_fill(~seen, -math.inf))
    return (p @ v).reshape(b, hq, lq, d).transpose(1, 2).contiguous().to(s["q"].dtype)


def _shared(s):
    b, hkv, g, d = s["q"].shape
    q = s["q"].float()
    rows = q.transpose(0, 1).reshape(hkv, b * g, d)
    x0 = (rows @ s["kp"].float().transpose(1, 2)).reshape(hkv, b, g, -1).transpose(0, 1) * s["scale"]
    x1 = (q @ s["k"].float().transpose(2, 3)) * s["scale"]
    m = x1.shape[-1]
    seen = torch.arange(m, device=DEV) < s["lengths"][:, None]
    p = _softmax(torch.cat((x0, x1.masked_fill(~seen[:, None, None], -math.inf)), dim=-1))
    n = x0.shape[-1]
    o = p[..., :n].transpose(0, 1).reshape(hkv, b * g, n) @ s["vp"].float()
    o = o.reshape(hkv, b, g, d).transpose(0, 1) + p[..., n:] @ s["v"].float()
    return o.to(s["q"].dtype)


def run(state):
    s, op = state, state["op"]
    if op == "append":
        if own:
            from threadcut_b200.paged import append_rope
            q = append_rope(s["k"], s["v"], s["cos"], s["sin"], s["k_pool"], s["v_pool"], s["slots"], q=s["q"],
                            q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        else:
            q = _append(s)
        return q, s["k_pool"], s["v_pool"]
    if op == "window_decode":
        if own:
            from threadcut_b200.flash_decode import decode_attention_window
            return decode_attention_window(s["q"], s["k"], s["v"], s["scale"], s["window"], s["sinks"], s["lengths"])
        return _window_decode(s)
    if op == "window_prefill":
        if own:
            from threadcut_b200.prefill import prefill_attention_window
            return prefill_attention_window(s["q"], s["k"], s["v"], s["scale"], s["window"], s["sinks"])
        return _window_prefill(s)
    if own:
        from threadcut_b200.flash_decode import decode_attention_shared
        return decode_attention_shared(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["scale"], s["lengths"])
    return _shared(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "append":
        heads, t, d, rot = case["hq"] + 2 * case["hkv"], case["t"], case["d"], case["rot"]
        tab = 4 if case["table"] == "fp32" else es
        turned = (case["hq"] + case["hkv"]) * t
        return {"bytes": 2 * heads * t * d * es + 2 * t * rot * tab + 8 * t + (2 * d * es if case["norm"] else 0),
                "flops": turned * (3 * rot + (4 * d if case["norm"] else 0))}
    b, hkv, g, d = case["b"], case["hkv"], case["g"], case["d"]
    if case["op"] == "window_decode":
        # the lengths are spread evenly over lo..n, the first of them n
        size = case["window"] + case["sinks"]
        lens = [case["n"]] + [case["lo"] + (case["n"] - case["lo"]) * (i + 0.5) / max(1, b - 1) for i in range(b - 1)]
        rows = sum(min(x, size) for x in lens)
        return {"bytes": 2 * rows * hkv * d * es + 2 * b * hkv * g * d * es + 4 * b, "flops": 4 * rows * hkv * g * d}
    if case["op"] == "window_prefill":
        lq, lk, w, sinks = case["lq"], case["lk"], case["window"], case["sinks"]
        pairs = sum(min(p + 1, w) + min(sinks, max(0, p + 1 - w)) for p in range(lk - lq, lk))
        first = max(0, lk - lq - w + 1)
        rows = lk - first + min(sinks, first)
        return {"bytes": 2 * b * hkv * rows * d * es + 2 * b * lq * hkv * g * d * es, "flops": 4 * b * pairs * hkv * g * d}
    n, m = case["n"], case["m"]
    tails = m + (b - 1) * (case["lo"] + m) / 2
    return {"bytes": 2 * (n + tails) * hkv * d * es + 2 * b * hkv * g * d * es + 4 * b,
            "flops": 4 * (b * n + tails) * hkv * g * d}


# ------------------------------------------------------------------ the definitions in 64 bits
def _attend64(q, k, v, scale):
    """One query head's rows q [r, d] over the keys it sees k, v [n, d]."""
    if k.shape[0] == 0:
        return torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    return torch.softmax(torch.einsum("rd,nd->rn", q, k) * scale, dim=1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        cos, sin = s["cos"].double(), s["sin"].double()
        rot, d = case["rot"], case["d"]

        def turn(x, w):
            x = x.double().clone()
            if w is not None:
                x = w.double() * x / torch.sqrt((x * x).sum(2, keepdim=True) / d + EPS)
            a, c = x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone()
            x[..., :rot // 2] = a * cos[:, :rot // 2] - c * sin[:, :rot // 2]
            x[..., rot // 2:rot] = c * cos[:, rot // 2:] + a * sin[:, rot // 2:]
            return x

        pools = [s["k_pool"].double(), s["v_pool"].double()]
        page, row = s["slots"].long().unbind(1)
        for pool, x in zip(pools, (turn(s["k"], s["k_norm"]), s["v"].double())):
            for h in range(case["hkv"]):
                pool[page, h, row] = x[h]
        return turn(s["q"], s["q_norm"]), pools[0], pools[1]
    b, hkv, g, d = case["b"], case["hkv"], case["g"], case["d"]
    if case["op"] == "window_decode":
        out = torch.zeros(b, hkv, g, d, dtype=torch.float64, device=DEV)
        for i, n in enumerate(s["lengths"].tolist()):
            see = [j for j in range(n) if j < s["sinks"] or j >= n - s["window"]]
            for h in range(hkv):
                out[i, h] = _attend64(s["q"][i, h].double(), s["k"][i, h][see].double(), s["v"][i, h][see].double(),
                                      s["scale"])
        return out
    if case["op"] == "window_prefill":
        lq, lk = case["lq"], case["lk"]
        out = torch.zeros(b, lq, hkv * g, d, dtype=torch.float64, device=DEV)
        gap = (lk - lq + torch.arange(lq, device=DEV))[:, None] - torch.arange(lk, device=DEV)[None]
        hidden = (gap < 0) | ((gap >= s["window"]) & (torch.arange(lk, device=DEV) >= s["sinks"])[None])
        for i in range(b):
            for hq in range(hkv * g):
                k, v = s["k"][i, hq // g].double(), s["v"][i, hq // g].double()
                x = (s["q"][i, hq].double() @ k.T) * s["scale"]
                x[hidden] = -math.inf
                out[i, :, hq] = torch.softmax(x, dim=1) @ v
        return out
    out = torch.zeros(b, hkv, g, d, dtype=torch.float64, device=DEV)
    for h in range(hkv):
        kp, vp = s["kp"][h].double(), s["vp"][h].double()
        for i, m in enumerate(s["lengths"].tolist()):
            out[i, h] = _attend64(s["q"][i, h].double(), torch.cat((kp, s["k"][i, h, :m].double())),
                                  torch.cat((vp, s["v"][i, h, :m].double())), s["scale"])
    return out
