"""Paged append with the rotation (paged.append_rope, PagedKV.append, tc_paged_append_rope) on a B200
against the formula in float64.

Tolerance: the kernel works in fp32 and rounds once. Half a step of the output type relative to the
value, plus the fp32 part: the sum of squares of d <= 512 elements is 16 sequential adds and a 5-step
butterfly (relative error <= 21 * 2^-24, halved by the square root), rsqrt 2 steps, two products, and
the rotation's two products and a sum: under 32 * 2^-24 of |z_i cos| + |z_j sin|. fp16 results below
its normal range are off by at most 2^-25.
"""
import numpy as np
import pytest
import torch

from threadcut_b200 import _lib
from threadcut_b200.flash_decode import decode_attention
from threadcut_b200.paged import PagedKV, append_rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


def f64(t):
    return t.detach().double().cpu().numpy()


def turn_ref(x, w, cos, sin, eps):
    """(result, scale of the fp32 error) of normalise + rotate for x [h, t, d], in float64."""
    x, cos, sin = f64(x), f64(cos), f64(sin)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * f64(w)
    rot = cos.shape[-1]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    c0, c1, s0, s1 = cos[:, :rot // 2], cos[:, rot // 2:], sin[:, :rot // 2], sin[:, rot // 2:]
    out = np.concatenate((a * c0 - b * s0, b * c1 + a * s1, x[..., rot:]), -1)
    size = np.concatenate((abs(a * c0) + abs(b * s0), abs(b * c1) + abs(a * s1), abs(x[..., rot:])), -1)
    return out, size


def assert_close(got, ref, size, dtype):
    tol = torch.finfo(dtype).eps / 2 * np.abs(ref) + 32 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == F16 else 0.0)
    err = np.abs(f64(got) - ref)
    assert (err <= tol).all(), f"max error {err.max()}, worst excess {(err - tol).max()}"


def make(t, hq, hkv, d, rot, dtype, table, norm, page_rows, layout, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    if layout == "fused":      # views of one projection output, a row a token
        qkv = normal(t, hq + 2 * hkv, d).transpose(0, 1)
        q, k, v = qkv[:hq], qkv[hq:hq + hkv], qkv[hq + hkv:]
    elif layout == "heads":    # contiguous [h, t, d]
        q, k, v = normal(hq, t, d), normal(hkv, t, d), normal(hkv, t, d)
    elif layout == "odd":      # rows that start off any 16-byte boundary
        q, k, v = normal(hq, t, d + 3)[..., 1:d + 1], normal(hkv, t, d + 1)[..., 1:], normal(hkv, t, d + 5)[..., :d]
    else:                      # last dimension not contiguous
        q, k, v = (normal(h, d, t).transpose(1, 2) for h in (hq, hkv, hkv))
    first = 17 % page_rows
    pages = -(-(first + t) // page_rows)
    order = torch.randperm(pages + 2, generator=g, device=DEV)[:pages]
    at = first + torch.arange(t, device=DEV)
    slots = torch.stack((order[at // page_rows], at % page_rows), 1).to(torch.int32).contiguous()
    pos = 1000 + torch.arange(t, device=DEV).double()
    ang = pos[:, None] * 1e4 ** (-torch.arange(0, rot, 2, device=DEV).double() / rot)
    ang = torch.cat((ang, ang + 0.25), 1)  # the halves differ: the formula takes each table entry as it is
    w = [(1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2)]
    return dict(q=q, k=k, v=v, cos=ang.cos().to(table), sin=ang.sin().to(table), slots=slots,
                k_pool=normal(pages + 2, hkv, page_rows, d), v_pool=normal(pages + 2, hkv, page_rows, d), w=w)


def check_case(c, dtype, eps=1e-6, with_q=True):
    kp0, vp0 = c["k_pool"].clone(), c["v_pool"].clone()
    out = append_rope(c["k"], c["v"], c["cos"], c["sin"], c["k_pool"], c["v_pool"], c["slots"],
                      q=c["q"] if with_q else None, q_norm=c["w"][0], k_norm=c["w"][1], eps=eps)
    page, row = c["slots"].long().unbind(1)
    if with_q:
        assert out.shape == c["q"].shape and out.dtype == dtype
        assert_close(out, *turn_ref(c["q"], c["w"][0], c["cos"], c["sin"], eps), dtype)
    else:
        assert out is None
    got = c["k_pool"][page, :, row].transpose(0, 1)
    assert_close(got, *turn_ref(c["k"], c["w"][1], c["cos"], c["sin"], eps), dtype)
    assert torch.equal(c["v_pool"][page, :, row].transpose(0, 1), c["v"])
    # every other row of the pools is as it was
    kp0[page, :, row], vp0[page, :, row] = c["k_pool"][page, :, row], c["v_pool"][page, :, row]
    assert torch.equal(kp0, c["k_pool"]) and torch.equal(vp0, c["v_pool"])


@pytest.mark.parametrize("dtype,table", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("layout", ["fused", "heads", "odd", "strided"])
@pytest.mark.parametrize("t", [1, 3, 65])
def test_types_and_layouts(dtype, table, layout, t):
    check_case(make(t, 32, 8, 128, 128, dtype, table, True, 64, layout), dtype)


@pytest.mark.parametrize("d,rot", [(2, 2), (6, 4), (64, 64), (64, 32), (80, 80), (96, 48), (128, 64), (128, 2), (256, 256),
                                   (256, 64), (512, 512), (512, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm", [False, True])
def test_head_sizes_and_partial_rotation(d, rot, dtype, norm):
    check_case(make(33, 6, 3, d, rot, dtype, dtype, norm, 32, "fused", seed=d + rot), dtype)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (5, 5), (40, 8), (128, 2)])
@pytest.mark.parametrize("t", [1, 2, 200])
def test_head_counts(hq, hkv, t):
    check_case(make(t, hq, hkv, 64, 64, F16, F16, True, 100, "fused", seed=hq), F16)


@pytest.mark.parametrize("d", [64, 66])
def test_without_queries(d):
    check_case(make(41, 4, 2, d, d, BF16, BF16, True, 64, "heads"), BF16, with_q=False)


def test_only_one_norm_weight():
    c = make(9, 4, 2, 64, 64, F32, F32, True, 64, "fused")
    c["w"][0] = None
    check_case(c, F32)
    c = make(9, 4, 2, 64, 64, F32, F32, True, 64, "fused")
    c["w"][1] = None
    check_case(c, F32)


def test_a_long_prompt():
    check_case(make(9001, 32, 8, 128, 128, BF16, BF16, True, 64, "fused"), BF16)


def test_zero_rows_and_a_zero_vector():
    c = make(5, 4, 2, 128, 128, BF16, BF16, True, 64, "fused")
    c["k"][:, 2].zero_()  # norm of a zero row: eps keeps it finite
    check_case(c, BF16)
    kp, vp = c["k_pool"].clone(), c["v_pool"].clone()
    e = torch.empty(2, 0, 128, device=DEV, dtype=BF16)
    tab = torch.empty(0, 128, device=DEV, dtype=BF16)
    out = append_rope(e, e, tab, tab, c["k_pool"], c["v_pool"], torch.empty(0, 2, device=DEV, dtype=torch.int32),
                      q=torch.empty(4, 0, 128, device=DEV, dtype=BF16))
    assert tuple(out.shape) == (4, 0, 128)
    assert torch.equal(kp, c["k_pool"]) and torch.equal(vp, c["v_pool"])


@pytest.mark.parametrize("d", [128, 30])
def test_a_slot_outside_the_pool_is_skipped(d):
    c = make(6, 4, 2, d, d, BF16, BF16, False, 64, "heads")
    pages, rows = c["k_pool"].shape[0], c["k_pool"].shape[2]
    page, row = c["slots"].long().unbind(1)
    c["slots"] = c["slots"].clone()
    c["slots"][1] = torch.tensor([-1, 0], dtype=torch.int32)
    c["slots"][2] = torch.tensor([pages, 0], dtype=torch.int32)
    c["slots"][3] = torch.tensor([0, rows], dtype=torch.int32)
    c["slots"][4] = torch.tensor([0, -5], dtype=torch.int32)
    kp, vp = c["k_pool"].clone(), c["v_pool"].clone()
    q = append_rope(c["k"], c["v"], c["cos"], c["sin"], c["k_pool"], c["v_pool"], c["slots"], q=c["q"])
    assert_close(q, *turn_ref(c["q"], None, c["cos"], c["sin"], 0), BF16)  # queries have no slot
    keep = [0, 5]
    kp[page[keep], :, row[keep]] = c["k_pool"][page[keep], :, row[keep]]
    vp[page[keep], :, row[keep]] = c["v"][:, keep].transpose(0, 1)
    assert torch.equal(kp, c["k_pool"]) and torch.equal(vp, c["v_pool"])


@pytest.mark.parametrize("d", [128, 36])
def test_queries_in_place_through_the_c_entry(d):
    c = make(70, 8, 2, d, d, BF16, BF16, True, 64, "heads")
    ref = turn_ref(c["q"], c["w"][0], c["cos"], c["sin"], 1e-6)
    q, k, v, kp = c["q"], c["k"], c["v"], c["k_pool"]
    st = _lib.lib().tc_paged_append_rope(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(), kp.data_ptr(), c["v_pool"].data_ptr(), 8, 2, d, 70,
        *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *q.stride()[:2], c["w"][0].data_ptr(), c["w"][1].data_ptr(),
        1e-6, c["cos"].data_ptr(), c["sin"].data_ptr(), d, d, d, 2, kp.shape[2], kp.shape[0], *kp.stride()[:3],
        c["slots"].data_ptr(), 2, _lib.stream_ptr(q.device))
    assert st == 0
    assert_close(q, *ref, BF16)


def test_batched_shapes_and_transformers_tables():
    """The [1, heads, t, d] projections and [1, t, rot] position embeddings of a transformers layer."""
    c = make(20, 8, 2, 64, 64, BF16, BF16, False, 64, "fused")
    q = append_rope(c["k"][None], c["v"][None], c["cos"][None], c["sin"][None], c["k_pool"], c["v_pool"], c["slots"],
                    q=c["q"][None])
    assert q.shape == (1, 8, 20, 64)
    assert_close(q[0], *turn_ref(c["q"], None, c["cos"], c["sin"], 0), BF16)


def test_another_stream_and_a_replayed_graph():
    c = make(50, 8, 2, 128, 128, BF16, BF16, True, 64, "fused")
    args = (c["k"], c["v"], c["cos"], c["sin"])
    pools = [torch.zeros_like(c["k_pool"]) for _ in range(4)]
    kw = dict(q=c["q"], q_norm=c["w"][0], k_norm=c["w"][1])
    want = append_rope(*args, pools[0], pools[1], c["slots"], **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = append_rope(*args, pools[2], pools[3], c["slots"], **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    graph = torch.cuda.CUDAGraph()
    pools[2].zero_()
    with torch.cuda.graph(graph):
        out = append_rope(*args, pools[2], pools[3], c["slots"], **kw)
    c["q"].mul_(2), c["k"].mul_(2), c["v"].mul_(2)
    want = append_rope(*args, pools[0], pools[1], c["slots"], **kw)
    for _ in range(2):
        graph.replay()
        assert torch.equal(out, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_a_prompt_and_steps_through_paged_kv():
    """reserve + append + decode over a prompt and a few steps, against attention over the same rows."""
    hq, hkv, d = 8, 2, 128
    kv = PagedKV(2, hkv, d, max_tokens=400, device=DEV)
    ks, vs = [], []
    for step, t in enumerate((150, 1, 1, 30, 1)):
        c = make(t, hq, hkv, d, d, BF16, BF16, True, 64, "fused", seed=step)
        kv.reserve(t)
        for layer in range(2):
            q = kv.append(layer, c["k"], c["v"], c["cos"], c["sin"], q=c["q"], q_norm=c["w"][0], k_norm=c["w"][1])
        spare = torch.empty(1, hkv, t, d, device=DEV, dtype=BF16)
        own_slots = torch.stack((torch.zeros(t), torch.arange(t)), 1).to(DEV, torch.int32)
        append_rope(c["k"], c["v"], c["cos"], c["sin"], spare, torch.empty_like(spare), own_slots, k_norm=c["w"][1])
        ks.append(spare[0])
        vs.append(c["v"])
        k, v = torch.cat(ks, 1), torch.cat(vs, 1)
        for layer in range(2):
            gk, gv = kv.gather(layer)
            assert torch.equal(gk, k) and torch.equal(gv, v)
            qq = q[:, -1].reshape(hkv, hq // hkv, d)
            assert torch.equal(kv.decode(layer, qq, d ** -0.5), decode_attention(qq, k, v, d ** -0.5))
