"""4-bit cache rows: written (with norm and rotation), read back and rotated in place, against plain torch and float64."""
import pytest
import torch

import int4_ref as ref
from threadcut_b200 import int4
from threadcut_b200.kv import shift_keys

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(*shape, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def pools(pages, hkv, rows, d, fill=0xA5):
    return [torch.full((pages, hkv, rows, ref.row_bytes(d)), fill, dtype=torch.uint8, device=DEV) for _ in range(2)]


def slots_of(where):
    return where.to(torch.int32).contiguous()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,t,rows", [(1, 1, 32), (3, 33, 40), (8, 130, 64)])
def test_write_and_read_back(dtype, d, hkv, t, rows):
    gen = torch.Generator().manual_seed(d + t)
    tiles, where, total = ref.pages(t, rows, gen)
    k, v = randn(hkv, t, d, dtype=dtype, seed=1), randn(hkv, t, d, dtype=dtype, seed=2, scale=30.0)
    kp, vp = pools(total, hkv, rows, d)
    before = kp.clone(), vp.clone()
    int4.write_int4(k, v, kp, vp, slots_of(where))
    for pool, old, x in ((kp, before[0], k), (vp, before[1], v)):
        want = old.clone()
        want[where[:, 0], :, where[:, 1]] = ref.rows_of(x).transpose(0, 1)
        assert torch.equal(pool, want)  # the rows to the byte, and no other byte
    gk, gv = int4.gather_int4(kp, vp, tiles, t, dtype)
    assert gk.is_contiguous() and gk.dtype == dtype and gk.shape == (hkv, t, d)
    assert torch.equal(gk, ref.values_of(ref.rows_of(k), d, dtype))
    assert torch.equal(gv, ref.values_of(ref.rows_of(v), d, dtype))
    # half a level, and the roundings of z and of the value: (1/2) S/16 + 2 half-steps of the largest of |z|, |x| + 2 S
    codes, s, z = ref.quantise64(k)
    half = torch.finfo(dtype).eps / 2
    most = s.double() / 32 + 2 * half * (z.double().abs() + 2 * s.double())
    assert ((gk.double() - k.double()).abs() <= most.repeat_interleave(32, -1)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,rot,table", [(64, 64, "same"), (64, 32, "f32"), (128, 128, "same"), (128, 128, "f32"),
                                         (128, 6, "same"), (256, 64, "f32"), (256, 256, "same")])
@pytest.mark.parametrize("hq,hkv,t", [(4, 1, 1), (5, 3, 7), (32, 8, 65)])
def test_rotation_is_that_of_elementary_operations(dtype, d, rot, table, hq, hkv, t):
    q, k, v = (randn(h, t, d, dtype=dtype, seed=i) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    angle = randn(t, rot, dtype=F32, seed=4) * 3
    tab = dtype if table == "same" else F32
    cos, sin = angle.cos().to(tab), angle.sin().to(tab)
    _, where, total = ref.pages(t, 32, torch.Generator().manual_seed(t))
    kp, vp = pools(total, hkv, 32, d)
    out = int4.append_rope_int4(k, v, cos, sin, kp, vp, slots_of(where), q=q)
    assert torch.equal(out, ref.rotate32(q, cos, sin))
    assert torch.equal(kp[where[:, 0], :, where[:, 1]].transpose(0, 1), ref.rows_of(ref.rotate32(k, cos, sin)))
    assert torch.equal(vp[where[:, 0], :, where[:, 1]].transpose(0, 1), ref.rows_of(v))
    # batched views, and one launch without queries
    kp2, vp2 = pools(total, hkv, 32, d)
    out2 = int4.append_rope_int4(k[None], v[None], cos[None], sin[None], kp2, vp2, slots_of(where), q=q[None])
    assert torch.equal(out2[0], out) and torch.equal(kp2, kp) and torch.equal(vp2, vp)
    kp3, vp3 = pools(total, hkv, 32, d)
    assert int4.append_rope_int4(k, v, cos, sin, kp3, vp3, slots_of(where)) is None
    assert torch.equal(kp3, kp) and torch.equal(vp3, vp)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,rot,t", [(128, 128, 1), (64, 32, 40), (256, 256, 9), (128, 10, 5)])
def test_norm_and_rotation_within_half_a_level(dtype, d, rot, t):
    hq, hkv, eps = 6, 2, 1e-6
    q, k, v = (randn(h, t, d, dtype=dtype, seed=i, scale=2.0) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    wq, wk = (1 + 0.1 * randn(d, dtype=dtype, seed=i) for i in (5, 6))
    angle = randn(t, rot, dtype=F32, seed=4) * 3
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    tiles, where, total = ref.pages(t, 32, torch.Generator().manual_seed(t))
    kp, vp = pools(total, hkv, 32, d)
    out = int4.append_rope_int4(k, v, cos, sin, kp, vp, slots_of(where), q=q, q_norm=wq, k_norm=wk, eps=eps)

    def exact(x, w):
        x = x.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
        head, rest = x[..., :rot], x[..., rot:]
        half = torch.cat((-head[..., rot // 2:], head[..., :rot // 2]), -1)
        return torch.cat((head * cos.double() + half * sin.double(), rest), -1), x.abs().amax(-1, keepdim=True)

    # fp32 on the way (d + 16 roundings of the two products), then one to T (fp16: steps of 2^-24 at least)
    eh = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == HF else 0.0
    want, size = exact(q, wq)
    slack = (d + 16) * 2.0 ** -24 * 2 * size
    assert ((out.double() - want).abs() <= slack + eh * want.abs() * 1.001 + tiny).all()
    gk, _ = int4.gather_int4(kp, vp, tiles, t, dtype)
    want, size = exact(k, wk)
    # the written key is off by that; then half a level of its group and the roundings of z and of the value, with the
    # group's range taken from the exact keys and their own error
    g = want.unflatten(-1, (-1, 32))
    err = ((d + 16) * 2.0 ** -24 * 2 * size + eh * size * 1.001 + tiny).amax(-1, keepdim=True)
    width = (g.amax(-1) - g.amin(-1) + 2 * err) / 0.9375 * (1 + eh) + 2 * tiny
    most = err + width / 32 + 2 * eh * (g.abs().amax(-1) + err + 3 * width) + 2 * tiny
    assert ((gk.double() - want).abs() <= most.repeat_interleave(32, -1)).all()


@pytest.mark.parametrize("view", ["fused", "odd_start", "gaps", "transposed"])
def test_strides_and_starts(view):
    hq, hkv, t, d = 4, 2, 11, 128
    if view == "fused":
        x = randn(t, hq + 2 * hkv, d, dtype=BF).transpose(0, 1)
        q, k, v = x[:hq], x[hq:hq + hkv], x[hq + hkv:]
    elif view == "odd_start":  # rows off 16-byte boundaries
        x = randn(hq + 2 * hkv, t, d + 3, dtype=BF)[..., 1:d + 1]
        q, k, v = x[:hq], x[hq:hq + hkv], x[hq + hkv:]
    elif view == "gaps":  # a last dimension that is not contiguous
        x = randn(hq + 2 * hkv, t, 2 * d, dtype=BF)[..., ::2]
        q, k, v = x[:hq], x[hq:hq + hkv], x[hq + hkv:]
    else:
        q, k, v = (randn(t, h, d, dtype=BF, seed=h + i).transpose(0, 1) for i, h in enumerate((hq, hkv, hkv)))
    angle = randn(t, d + 5, dtype=F32, seed=4)[:, 3:d + 3]
    cos, sin = angle.cos(), angle.sin()
    _, where, total = ref.pages(t, 32, torch.Generator().manual_seed(1))
    # pools that are views of a larger buffer
    big = [torch.zeros(total, hkv + 1, 34, ref.row_bytes(d), dtype=torch.uint8, device=DEV) for _ in range(2)]
    kp, vp = (b[:, :hkv, 1:33] for b in big)
    out = int4.append_rope_int4(k, v, cos, sin, kp, vp, slots_of(where), q=q)
    assert torch.equal(out, ref.rotate32(q, cos, sin))
    assert torch.equal(kp[where[:, 0], :, where[:, 1]].transpose(0, 1), ref.rows_of(ref.rotate32(k.contiguous(), cos, sin)))
    assert torch.equal(vp[where[:, 0], :, where[:, 1]].transpose(0, 1), ref.rows_of(v.contiguous()))
    assert not big[0][:, hkv].any() and not big[0][:, :, 0].any() and not big[0][:, :, 33].any()


def test_slots_outside_the_pool_are_skipped():
    kp, vp = pools(3, 2, 32, 64)
    before = kp.clone()
    k = randn(2, 5, 64, dtype=BF)
    slots = torch.tensor([[0, 32], [3, 0], [-1, 4], [1, -1], [2, 31]], dtype=torch.int32, device=DEV)
    int4.write_int4(k, k, kp, vp, slots)
    want = before.clone()
    want[2, :, 31] = ref.rows_of(k[:, 4])
    assert torch.equal(kp, want) and torch.equal(vp, want)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_groups_at_the_edges_of_the_type(dtype):
    d, big = 64, (1e38 if dtype == BF else 20000.0)
    tiny = torch.finfo(dtype).smallest_normal
    rows = torch.zeros(8, d, dtype=torch.float64)
    rows[1] = 3.25                                        # one value throughout: itself
    rows[2, ::2], rows[2, 1::2] = big, -big               # the widest range that is promised
    rows[3] = torch.linspace(-1, 1, d, dtype=torch.float64) * tiny
    rows[4] = 100 + torch.linspace(0, 1, d, dtype=torch.float64)
    rows[5, 7] = float("nan")                             # spoils its own group only
    rows[6, 40], rows[7, 3] = float("inf"), -float("inf")
    rows[5, 32:], rows[6, :32], rows[7, 32:] = 2.0, 2.0, 2.0
    x = rows.to(dtype).to(DEV)[None]
    kp, vp = pools(1, 1, 32, d)
    slots = torch.stack((torch.zeros(8), torch.arange(8)), 1).to(torch.int32).to(DEV)
    int4.write_int4(x, x, kp, vp, slots)
    got = int4.gather_int4(kp, vp, torch.tensor([[0, 0, 8, 0]], dtype=torch.int32, device=DEV), 8, dtype)[0][0]
    assert torch.equal(got[:5], ref.values_of(ref.rows_of(x[0, :5]), d, dtype))
    assert torch.equal(got[0], x[0, 0]) and torch.equal(got[1], x[0, 1])
    for i, (bad, good) in ((5, (slice(0, 32), slice(32, 64))), (6, (slice(32, 64), slice(0, 32))),
                           (7, (slice(0, 32), slice(32, 64)))):
        assert torch.isnan(got[i, bad]).all() and (got[i, good] == 2).all()
    if dtype == HF:  # beyond the promise: NaN, never a finite number far off
        far = torch.full((1, 1, d), -60000.0, dtype=dtype, device=DEV)
        far[..., ::2] = -50000.0
        int4.write_int4(far, far, kp, vp, slots[:1])
        assert torch.isnan(int4.gather_int4(kp, vp, torch.tensor([[0, 0, 1, 0]], dtype=torch.int32, device=DEV), 1,
                                            dtype)[0]).all()


def test_read_back_skips_what_lies_outside():
    d, dtype = 128, BF
    kp, vp = (ref.rows_of(randn(3, 2, 32, d, dtype=dtype, seed=s)) for s in (1, 2))
    tiles = torch.tensor([[0, 30, 5, 2],      # two rows of the page, three behind it
                          [3, 0, 32, 5], [-1, 0, 32, 37],  # no such page
                          [1, 4, 3, 68],      # positions 68, 69; 70 is behind the outputs
                          [2, -2, 4, 10],     # rows -2, -1 are outside
                          [2, 8, 0, 20], [2, 8, -5, 20], [1, 0, 2, -1]], dtype=torch.int32, device=DEV)
    k, v = int4.gather_int4(kp, vp, tiles, 70, dtype)
    for got, pool in ((k, kp), (v, vp)):
        val = ref.values_of(pool, d, dtype)
        assert torch.equal(got[:, 2:4], val[0, :, 30:32])
        assert torch.equal(got[:, 68:70], val[1, :, 4:6])
        assert torch.equal(got[:, 12:14], val[2, :, 0:2])
        assert torch.equal(got[:, 0], val[1, :, 1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hkv,c,rows,layers", [(64, 3, 1, 32, 1), (128, 8, 200, 64, 3), (256, 2, 77, 40, 2),
                                                 (128, 1, 33, 100, 1)])
def test_keys_rotate_where_they_lie(dtype, d, hkv, c, rows, layers):
    tiles, where, total = ref.pages(c, rows, torch.Generator().manual_seed(c))
    kps = [ref.rows_of(randn(total, hkv, rows, d, dtype=dtype, seed=l)) for l in range(layers)]
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2).float() / d))
    before = [p.clone() for p in kps]
    int4.rotate_keys_int4(kps, tiles, -333, inv, dtype)
    for pool, old in zip(kps, before):
        keys = ref.values_of(old[where[:, 0], :, where[:, 1]], d, dtype).transpose(0, 1).contiguous()
        want = old.clone()
        want[where[:, 0], :, where[:, 1]] = ref.rows_of(shift_keys(keys, -333, inv)).transpose(0, 1)
        assert torch.equal(pool, want)


def test_rotation_skips_what_lies_outside():
    d = 64
    pool = ref.rows_of(randn(2, 1, 32, d, dtype=BF))
    before = pool.clone()
    tiles = torch.tensor([[2, 0, 32], [-1, 0, 32], [0, 32, 4], [1, 0, 0], [1, 0, -3]], dtype=torch.int32, device=DEV)
    inv = 1.0 / (1e4 ** (torch.arange(0, d, 2).float() / d))
    int4.rotate_keys_int4([pool], tiles, 5, inv, BF)
    assert torch.equal(pool, before)
    int4.rotate_keys_int4([pool], tiles[:0], 5, inv, BF)
    assert torch.equal(pool, before)


def test_nothing_to_do():
    kp, vp = pools(1, 2, 32, 64)
    before = kp.clone()
    e = torch.empty(2, 0, 64, dtype=BF, device=DEV)
    int4.write_int4(e, e, kp, vp, torch.empty(0, 2, dtype=torch.int32, device=DEV))
    q = int4.append_rope_int4(e, e, e[0], e[0], kp, vp, torch.empty(0, 2, dtype=torch.int32, device=DEV), q=e)
    assert q.shape == e.shape and torch.equal(kp, before)
    k, v = int4.gather_int4(kp, vp, torch.empty(0, 4, dtype=torch.int32, device=DEV), 0, BF)
    assert k.shape == (2, 0, 64) == v.shape


def test_another_stream_and_a_graph():
    hkv, t, d = 2, 40, 128
    tiles, where, total = ref.pages(t, 64, torch.Generator().manual_seed(3))
    kp, vp = pools(total, hkv, 64, d)
    k, v = randn(hkv, t, d, dtype=BF, seed=1), randn(hkv, t, d, dtype=BF, seed=2)
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2).float() / d))
    slots = slots_of(where)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        int4.write_int4(k, v, kp, vp, slots)
        first = int4.gather_int4(kp, vp, tiles, t, BF)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        int4.write_int4(k, v, kp, vp, slots)
        int4.rotate_keys_int4([kp], tiles, -9, inv, BF)
        out = int4.gather_int4(kp, vp, tiles, t, BF)
    for seed in (5, 6):
        k.copy_(randn(hkv, t, d, dtype=BF, seed=seed))
        graph.replay()
        want = ref.values_of(ref.rows_of(shift_keys(ref.values_of(ref.rows_of(k), d, BF), -9, inv)), d, BF)
        assert torch.equal(out[0], want) and torch.equal(out[1], first[1])
