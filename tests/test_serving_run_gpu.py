"""The serving operators together, as an agent's engine runs them, on a B200: a prompt appended and
prefilled under a sliding window, decode steps, a splice, another chunk, and then several continuations of
the one paged context, each appending into its own suffix and decoding over prefix and suffix; every
attention against float64 over the rows the cache holds (tolerances of attn_bounds)."""
import pytest
import torch

from attn_bounds import P_SINGLE, P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib
from threadcut_b200.match import Split
from threadcut_b200.paged import PagedKV, append_rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


class Model:
    """Random projections of one attention layer and its rotary tables."""

    def __init__(self, hq, hkv, d, dtype, seed):
        self.hq, self.hkv, self.d, self.dtype = hq, hkv, d, dtype
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.inv = 1e4 ** (-torch.arange(0, d, 2, device=DEV).double() / d)
        self.norms = [(1 + 0.1 * self.rand(d)).to(dtype) for _ in range(2)]

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEV)

    def qkv(self, t):
        x = self.rand(t, self.hq + 2 * self.hkv, self.d).to(self.dtype).transpose(0, 1)
        return x[:self.hq], x[self.hq:self.hq + self.hkv], x[self.hq + self.hkv:]

    def tables(self, positions):
        a = positions.double()[:, None] * self.inv
        a = torch.cat((a, a), 1)
        return a.cos().to(self.dtype), a.sin().to(self.dtype)


def window_seen(lq, lk, window, sinks):
    at = (lk - lq + torch.arange(lq, device=DEV))[:, None]
    j = torch.arange(lk, device=DEV)
    return (j <= at) & ((j < sinks) | (j > at - window))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (10 ** 9, 0)])
def test_prompt_steps_splice_and_continuations(dtype, d, window, sinks):
    hq, hkv, g, layers = 8, 2, 4, 2
    scale = d ** -0.5
    m = Model(hq, hkv, d, dtype, 3)
    kv = PagedKV(layers, hkv, d, max_tokens=1200, dtype=dtype, device=DEV)

    def chunk(t):
        cos, sin = m.tables(kv.n + torch.arange(t, device=DEV))
        kv.reserve(t)
        for layer in range(layers):
            q, k, v = m.qkv(t)
            qr = kv.append(layer, k, v, cos, sin, q=q, q_norm=m.norms[0], k_norm=m.norms[1], eps=EPS)
            ks, vs = kv.gather(layer)
            assert torch.equal(vs[:, -t:], v)
            kk, vv = ks.repeat_interleave(g, 0), vs.repeat_interleave(g, 0)
            seen = window_seen(t, kv.n, window, sinks)
            if t == 1:
                out = kv.decode(layer, qr.reshape(hkv, g, d), scale, window=window, sinks=sinks).reshape(hq, 1, d)
                bits = P_SPLIT[dtype]
            else:
                out = kv.prefill(layer, qr[None], scale, window=window, sinks=sinks)[0].transpose(0, 1)
                bits = P_SINGLE[dtype]
            assert_within(out, *attend64(qr, kk, vv, scale, seen, bits))

    chunk(500)
    for _ in range(3):
        chunk(1)
    kv.splice(Split(120, 300, 203), m.inv.float())
    chunk(77)
    chunk(1)

    # five continuations: their suffixes are a pool of one page each
    b, cap = 5, 40
    sk, sv = (torch.full((layers, b, hkv, cap, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    lens = torch.tensor([0, 3, 0, 7, 1], device=DEV, dtype=torch.int32)
    for i, n in enumerate(lens.tolist()):  # some start with rows of their own
        sk[:, i, :, :n] = m.rand(layers, hkv, n, d).to(dtype)
        sv[:, i, :, :n] = m.rand(layers, hkv, n, d).to(dtype)
    prefix = [kv.gather(layer) for layer in range(layers)]
    for _ in range(4):
        cos, sin = m.tables(kv.n + lens)
        slots = torch.stack((torch.arange(b, device=DEV, dtype=torch.int32), lens), 1)
        lens += 1
        for layer in range(layers):
            q, k, v = m.qkv(b)
            qr = append_rope(k, v, cos, sin, sk[layer], sv[layer], slots, q=q, q_norm=m.norms[0], k_norm=m.norms[1],
                             eps=EPS)
            qr = qr.transpose(0, 1).reshape(b, hkv, g, d)
            out = kv.decode_shared(layer, qr, sk[layer], sv[layer], scale, lens)
            kk = torch.cat((prefix[layer][0].expand(b, -1, -1, -1), sk[layer]), 2)
            vv = torch.cat((prefix[layer][1].expand(b, -1, -1, -1), sv[layer]), 2)
            seen = torch.arange(kv.n + cap, device=DEV) < kv.n + lens[:, None]
            ref, tol = zip(*(attend64(qr[i], kk[i][:, :kv.n + n], vv[i][:, :kv.n + n], scale)
                             for i, n in enumerate(lens.tolist())))
            assert int(seen.sum()) == sum(kv.n + n for n in lens.tolist())
            assert_within(out, torch.stack(ref), torch.stack(tol))
    for layer in range(layers):  # nothing but the appended rows was written
        for i, n in enumerate(lens.tolist()):
            assert torch.isfinite(sk[layer, i, :, :n]).all() and torch.isnan(sk[layer, i, :, n:]).all()
        assert all(torch.equal(a, c) for a, c in zip(kv.gather(layer), prefix[layer]))


def test_a_captured_step_of_the_continuations():
    """append_rope + decode_shared of a step captured once; slots, lengths and projections change in place
    between replays."""
    hq, hkv, g, d, b, cap, dtype = 8, 2, 4, 128, 3, 30, torch.bfloat16
    m = Model(hq, hkv, d, dtype, 4)
    kv = PagedKV(1, hkv, d, max_tokens=400, dtype=dtype, device=DEV)
    kv.reserve(333)
    kv.write(0, *(m.rand(hkv, 333, d).to(dtype) for _ in range(2)))
    sk, sv, sk2, sv2 = (torch.zeros(b, hkv, cap, d, device=DEV, dtype=dtype) for _ in range(4))
    x = m.rand(b, hq + 2 * hkv, d).to(dtype)
    lens = torch.zeros(b, device=DEV, dtype=torch.int32)
    slots = torch.zeros(b, 2, device=DEV, dtype=torch.int32)
    cos, sin = m.tables(torch.arange(b, device=DEV))

    def step(k_buf, v_buf):
        h = x.transpose(0, 1)
        q = append_rope(h[hq:hq + hkv], h[hq + hkv:], cos, sin, k_buf, v_buf, slots, q=h[:hq])
        return kv.decode_shared(0, q.transpose(0, 1).reshape(b, hkv, g, d), k_buf, v_buf, 0.1, lens)

    def advance(i):
        x.copy_(m.rand(*x.shape).to(dtype))
        slots.copy_(torch.stack((torch.arange(b, device=DEV, dtype=torch.int32), lens), 1))
        for t, new in zip((cos, sin), m.tables(333 + lens)):
            t.copy_(new)
        lens.add_(1)

    advance(0)
    step(sk, sv)  # warm-up: tables and workspaces exist
    lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sk, sv)
    sk.zero_(), sv.zero_()
    for i in range(5):
        advance(i)
        graph.replay()
        want = step(sk2, sv2)
        assert torch.equal(out, want) and torch.equal(sk, sk2) and torch.equal(sv, sv2)
