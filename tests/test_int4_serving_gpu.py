"""The 4-bit operators together, as they are used: a paged cache of 4-bit rows (PagedKVInt4) through a prompt, decode steps and
splices, behind the attention plugin and behind the fused decode step with 4-bit projections."""
import pytest
import torch
from transformers import AutoModelForCausalLM, Qwen3Config
from transformers.cache_utils import DynamicCache

import int4_ref as ref
from attn_bounds import P_SINGLE, P_SPLIT, assert_within, attend64
from threadcut_b200 import _lib, int4, tp
from threadcut_b200 import attention as tc_attention
from threadcut_b200 import kv as tc_kv
from threadcut_b200.match import Split
from threadcut_b200.paged import PagedKV, PagedKVInt4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
EPS = 1e-6


@pytest.fixture(autouse=True, scope="module")
def _no_device_errors():
    _lib.device_errors(clear=True)
    yield
    assert _lib.device_errors(clear=True) == 0


class Projections:
    """Random projections of one attention layer and its rotary tables."""

    def __init__(self, hq, hkv, d, dtype, seed):
        self.hq, self.hkv, self.d, self.dtype = hq, hkv, d, dtype
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.inv = 1e4 ** (-torch.arange(0, d, 2, device=DEV).double() / d)

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEV)

    def qkv(self, t):
        x = self.rand(t, self.hq + 2 * self.hkv, self.d).to(self.dtype).transpose(0, 1)
        return x[:self.hq], x[self.hq:self.hq + self.hkv], x[self.hq + self.hkv:]

    def tables(self, positions):
        a = positions.double()[:, None] * self.inv
        a = torch.cat((a, a), 1)
        return a.cos().to(self.dtype), a.sin().to(self.dtype)


def stored(x):
    """What rows written from x read back as."""
    return ref.values_of(ref.rows_of(x), x.shape[-1], x.dtype)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (BF, 64)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (70, 0), (None, 0)])
def test_prompt_steps_and_splices(dtype, d, window, sinks):
    hq, hkv, g, layers = 8, 2, 4, 2
    if window is None and d != 128:
        window = 10 ** 9  # the prefill without a window takes heads of 128
    scale = d ** -0.5
    m = Projections(hq, hkv, d, dtype, 3)
    kv = PagedKVInt4(layers, hkv, d, max_tokens=1000, dtype=dtype, device=DEV)
    assert kv.k[0].dtype == torch.uint8 and kv.k[0].shape[-1] == kv.row_bytes == 5 * d // 8
    rows = [[torch.empty(hkv, 0, d, dtype=dtype, device=DEV) for _ in range(2)] for _ in range(layers)]

    def chunk(t, fused=True):
        cos, sin = m.tables(kv.n + torch.arange(t, device=DEV))
        kv.reserve(t)
        for layer in range(layers):
            q, k, v = m.qkv(t)
            kr, qr = ref.rotate32(k, cos, sin), ref.rotate32(q, cos, sin)
            if fused:
                assert torch.equal(kv.append(layer, k, v, cos, sin, q=q, eps=EPS), qr)
            elif t > 1:
                kv.write(layer, kr, v)
            want = rows[layer] = [torch.cat((a, stored(x)), 1) for a, x in zip(rows[layer], (kr, v))]
            if fused or t > 1:
                assert all(torch.equal(a, b) for a, b in zip(kv.gather(layer), want))
            at = (kv.n - t + torch.arange(t, device=DEV))[:, None]
            j = torch.arange(kv.n, device=DEV)
            seen = j <= at
            if window is not None:
                seen &= (j < sinks) | (j > at - window)
            kk, vv = (x.repeat_interleave(g, 0) for x in want)
            if t == 1:
                new = {} if fused else dict(k_new=kr[:, 0], v_new=v[:, 0])
                out = kv.decode(layer, qr.reshape(hkv, g, d), scale, window=window, sinks=sinks, **new).reshape(hq, 1, d)
                bits = P_SPLIT[dtype]
            else:
                out = kv.prefill(layer, qr[None], scale, window=window, sinks=sinks)[0].transpose(0, 1)
                bits = P_SINGLE[dtype]
            assert_within(out, *attend64(qr, kk, vv, scale, seen, bits))
            assert all(torch.equal(a, b) for a, b in zip(kv.gather(layer), want))

    def splice(a, c0, n):
        kv.splice(Split(a, c0, n - c0), m.inv.float())
        for layer in range(layers):
            k, v = rows[layer]
            c = k[:, c0:].contiguous()
            if a < c0 and c.shape[1]:
                c = stored(tc_kv.shift_keys(c, a - c0, m.inv.float()))
            rows[layer] = [torch.cat((k[:, :a], c), 1), torch.cat((v[:, :a], v[:, c0:]), 1)]
            assert all(torch.equal(x, y) for x, y in zip(kv.gather(layer), rows[layer]))

    chunk(1)
    chunk(299)
    chunk(1)
    chunk(1, fused=False)
    splice(120, 203, 302)
    chunk(77, fused=False)
    chunk(1)
    splice(7, 8, kv.n)
    chunk(1)
    splice(64, 64, kv.n)      # nothing in between
    splice(33, kv.n, kv.n)    # nothing behind
    chunk(1)
    assert all(torch.equal(a, b[:, 5:]) for a, b in zip(kv.gather(1, 5), rows[1]))
    kv.compact()
    assert kv.n == rows[0][0].shape[1]
    assert all(torch.equal(a, b) for layer in range(layers) for a, b in zip(kv.gather(layer), rows[layer]))
    chunk(1)
    kv.truncate(20)
    rows = [[x[:, :20] for x in r] for r in rows]
    chunk(2)
    kv.truncate(0)
    q = torch.ones(hkv, g, d, dtype=dtype, device=DEV)
    assert kv.gather(0)[0].shape == (hkv, 0, d) and not kv.decode(0, q, scale).any()


def test_a_whole_layer_captured():
    """One decode step of a layer with 4-bit cache and projections, captured once: its inputs, slots and tables change in place,
    and every replay gives the eager step's bits."""
    hidden, inter, hq, hkv, d, pages = 512, 1100, 8, 2, 64, 6
    gen = torch.Generator(device=DEV).manual_seed(5)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(BF)

    wqkv, wo, wgu, wd = (int4.quantize_weight(rand(n, k, scale=k ** -0.5), 64) for n, k in (
        ((hq + 2 * hkv) * d, hidden), (hidden, hq * d), (2 * inter, hidden), (hidden, inter)))
    x = rand(1, hidden)
    pools = [ref.rows_of(rand(pages, hkv, 64, d)) for _ in range(2)]
    tiles = torch.tensor([[p, r, 32] for p in range(pages) for r in (0, 32)], dtype=torch.int32, device=DEV)
    slot = torch.tensor([[2, 7]], dtype=torch.int32, device=DEV)
    cos, sin = rand(1, d), rand(1, d)

    def step(k_pool, v_pool):
        qkv = int4.gemv_int4(x, wqkv).view(hq + 2 * hkv, 1, d)
        q = int4.append_rope_int4(qkv[hq:hq + hkv], qkv[hq + hkv:], cos, sin, k_pool, v_pool, slot, q=qkv[:hq])
        o = int4.decode_attention_int4(q.reshape(hkv, hq // hkv, d), k_pool, v_pool, 0.125, tiles=tiles)
        h = x + int4.gemv_int4(o.view(1, -1), wo)
        return h + int4.gemv_int4(int4.gemv_int4(h, wgu), wd, swiglu=True)

    graphed, eager = ([p.clone() for p in pools] for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*graphed)
    s.synchronize()
    for p, q in zip(graphed, pools):
        p.copy_(q)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:  # two of them, that share the stream's workspace
        with torch.cuda.graph(graph, stream=s):
            outs.append(step(*graphed))
    for i in range(4):
        x.copy_(rand(1, hidden))
        cos.copy_(rand(1, d))
        slot.copy_(torch.tensor([[i, 9 * i]], dtype=torch.int32))
        want = step(*eager)
        graphs[i % 2].replay()
        assert torch.isfinite(want).all() and torch.equal(outs[i % 2], want)
        assert all(torch.equal(a, b) for a, b in zip(graphed, eager))


def tiny(dtype=BF, **kwargs):
    torch.manual_seed(0)
    cfg = Qwen3Config(**dict(dict(vocab_size=520, hidden_size=256, intermediate_size=544, num_hidden_layers=2,
                                  num_attention_heads=8, num_key_value_heads=2, head_dim=128, max_position_embeddings=8192),
                             **kwargs))
    return AutoModelForCausalLM.from_config(cfg, dtype=dtype, attn_implementation=tc_attention.NAME).to(DEV).eval()


def near(got, want):
    """Logits of two roundings of one computation. A token passes some 10 roundings a layer to at most 2^-8, so two layers
    move a logit by about sqrt(20) 2^-9 of the logits' own size: 1 %, and 5e-5 of a correlation. Where the one computation sees
    c of n rows before they are quantised, those move its attention by some 0.08 sqrt(2 c / n) of its size, 0.08 being half a
    level's root mean square for normal elements: 4 % for 36 of 340, 8e-4 of a correlation at the very most."""
    got, want = got.float().flatten(), want.float().flatten()
    assert torch.corrcoef(torch.stack([got, want]))[0, 1].item() > 0.999
    assert want[got.argmax()] >= want.max() - 0.1 * want.std()


@pytest.mark.parametrize("d", [128, 64])
def test_cache_behind_the_plugin(d):
    """A model over a 4-bit cache against the same model over a contiguous cache that holds the values of its rows, for the
    steps, for a chunk, and after a splice."""
    model = tiny(head_dim=d)
    cfg = model.config
    inv = model.model.rotary_emb.inv_freq
    ids = torch.randint(0, 520, (1, 400), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = tc_kv.new_cache(cfg, paged=True, max_tokens=600, bits=4)

    def call(a, b):
        """ids[a:b] over the cache, and over a copy of what it holds."""
        plain = DynamicCache(config=cfg)
        for layer, full in zip(plain.layers, cache.layers):
            layer.update(*full.materialize())
        got = model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True).logits[0, -1]
        near(got, model(input_ids=ids[:, a:b], past_key_values=plain, use_cache=True).logits[0, -1])

    with torch.no_grad():
        model(input_ids=ids[:, :300], past_key_values=cache, use_cache=True)
        store = cache.layers[0].state.kv
        assert isinstance(store, PagedKVInt4) and cache.get_seq_length() == 300
        assert tc_kv.cache_bytes(cache) == 2 * 300 * 2 * (5 * d // 8) * 2
        for i in range(300, 304):
            call(i, i + 1)
        call(304, 340)
        held = [store.gather(layer) for layer in range(2)]
        tc_kv.splice(cache, Split(100, 140, 200), inv)
        for layer, (k, v) in enumerate(held):
            ks, vs = store.gather(layer)
            assert torch.equal(vs, torch.cat((v[:, :100], v[:, 140:]), 1)) and torch.equal(ks[:, :100], k[:, :100])
            assert torch.equal(ks[:, 100:], stored(tc_kv.shift_keys(k[:, 140:].contiguous(), -40, inv)))
        assert cache.get_seq_length() == 300
        call(340, 341)
        cache.crop(290)
        call(341, 342)
        assert cache.get_seq_length() == 291


def test_a_full_pool_is_packed_again():
    model = tiny()
    cache = tc_kv.new_cache(model.config, paged=True, max_tokens=64, page_rows=32, bits=4)
    k = torch.randn(1, 2, 40, 128, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    inv = model.model.rotary_emb.inv_freq
    want = k[0, :, :0]
    for _ in range(90):  # 66 pages, one or two newly used a turn and as many left with a few rows
        for layer in cache.layers:
            layer.update(k, k)
        want = torch.cat((want, stored(k[0])), 1)
        n = cache.get_seq_length()
        tc_kv.splice(cache, Split(n - 38, n - 3, 3), inv)
        want = torch.cat((want[:, :n - 38], want[:, n - 3:]), 1)
    assert cache.get_seq_length() == want.shape[1] == 450
    assert torch.equal(cache.layers[1].state.kv.gather(1)[1], want)


def test_use_paged_cache_selects_the_rows():
    cfg = tiny().config
    k = torch.ones(1, 2, 3, 128, dtype=BF, device=DEV)
    try:
        for bits, kind in ((4, PagedKVInt4), (16, PagedKV)):
            tc_kv.use_paged_cache(max_tokens=100, bits=bits)
            cache = tc_kv.new_cache(cfg)
            cache.layers[0].update(k, k)
            assert type(cache.layers[0].state.kv) is kind
            assert type(tc_kv.new_cache(cfg, paged=False).layers[0]) is tc_kv.GrowingLayer
    finally:
        tc_kv.use_paged_cache(False)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("paged", [True, False])
def test_fused_step_with_4_bit_weights(dtype, paged):
    """accelerate(weight_bits=4) over a 4-bit cache (or the contiguous one) against the model in fp32 whose projections are what
    the 4-bit weights stand for, over a copy of what the cache holds."""
    model = tiny(dtype)
    exact = tiny(torch.float32)
    exact.set_attn_implementation("sdpa")
    ids = torch.randint(0, 520, (1, 306), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = tc_kv.new_cache(model.config, paged=paged, max_tokens=400, bits=4 if paged else None)
    with torch.no_grad():
        for a, b in zip(exact.parameters(), model.parameters()):
            a.copy_(b)
        for w in [m.weight for layer in exact.model.layers for m in layer.modules() if isinstance(m, torch.nn.Linear)] + [
                exact.lm_head.weight]:
            w.copy_(int4.dequantize_weight(int4.quantize_weight(w.to(dtype))))
        model(input_ids=ids[:, :300], past_key_values=cache, use_cache=True)
        dec = tp.accelerate(model, weight_bits=4)
        try:
            assert dec.weight_bits == 4 and not dec.use_peer_sums
            def refuse(*_):
                raise AssertionError("the model's own forward was called")

            for i in range(300, 306):
                n = cache.get_seq_length()
                plain = DynamicCache(config=exact.config)
                for layer, full in zip(plain.layers, cache.layers):
                    k, v = full.materialize() if paged else (full.keys, full.values)
                    layer.update(k.float(), v.float())
                x = ids[:, i:i + 1]
                hook = model.model.register_forward_pre_hook(refuse)
                got = model(input_ids=x, past_key_values=cache, use_cache=True)
                hook.remove()
                assert cache.get_seq_length() == n + 1 and got.past_key_values is cache
                near(got.logits[0, -1], exact(input_ids=x, past_key_values=plain, use_cache=True).logits[0, -1])
                if i == 302:
                    tc_kv.splice(cache, Split(100, 110, n + 1 - 110), model.model.rotary_emb.inv_freq)
            chunk = model(input_ids=ids[:, :5], past_key_values=cache, use_cache=True)  # the model's own forward
            assert chunk.logits.shape[1] == 5 and cache.get_seq_length() == 301
        finally:
            tp.restore(model)


def test_accelerate_leaves_16_bit_pages_to_the_model():
    model = tiny()
    cache = tc_kv.new_cache(model.config, paged=True, max_tokens=100)
    ids = torch.arange(40, device=DEV)[None]
    with torch.no_grad():
        model(input_ids=ids[:, :30], past_key_values=cache, use_cache=True)
        dec = tp.accelerate(model)
        try:
            assert not tp._fusable(cache, dec)
        finally:
            tp.restore(model)


def test_refusals_of_the_cache():
    kv = PagedKVInt4(1, 2, 128, max_tokens=100, device=DEV)
    k = torch.ones(2, 3, 128, dtype=BF, device=DEV)
    q = torch.ones(2, 4, 128, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="reserve"):
        kv.write(0, k, k)
    kv.reserve(3)
    for bad in (k[:, :2], k.half(), k[..., :64], k[:1]):
        with pytest.raises(ValueError):
            kv.write(0, bad, bad)
    with pytest.raises(ValueError):
        kv.append(0, k, k[:, :, :64], k[0], k[0])
    kv.write(0, k, k)
    for call in (lambda: kv.decode(0, q.half(), 1.0), lambda: kv.decode(0, q[:1], 1.0), lambda: kv.decode(0, q, 1.0, sinks=2),
                 lambda: kv.decode(0, q, 1.0, window=0), lambda: kv.decode(0, q, 1.0, k_new=k[:, 0]),
                 lambda: kv.decode(0, q, 1.0, k_new=k[:, 0], v_new=k[:, 0]),  # no slot of a single row
                 lambda: kv.decode(0, q.repeat(1, 5, 1), 1.0), lambda: kv.decode(0, q, float("nan")),
                 lambda: kv.decode_shared(0, q[None], k[None], k[None], 1.0),
                 lambda: kv.prefill(0, torch.ones(1, 8, 4, 128, dtype=BF, device=DEV), 1.0),
                 lambda: kv.prefill(0, torch.ones(1, 8, 3, 128, dtype=BF, device=DEV), 1.0, sinks=1),
                 lambda: kv.prefill(0, torch.ones(1, 8, 3, 128, dtype=BF, device=DEV), 1.0, window=0),
                 lambda: kv.splice(Split(2, 2, 2), torch.ones(64))):
        with pytest.raises(ValueError):
            call()


def test_refusals_with_tensors_on_the_device():
    d = 128
    pool = torch.zeros(4, 2, 64, 80, dtype=torch.uint8, device=DEV)
    k = torch.ones(2, 3, d, dtype=BF, device=DEV)
    q = torch.ones(2, 4, d, dtype=BF, device=DEV)
    cos = torch.ones(3, d, dtype=BF, device=DEV)
    slots = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    tiles = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    w = int4.quantize_weight(torch.ones(32, d, dtype=BF, device=DEV))

    def append(k=k, v=k, cos=cos, sin=cos, kp=pool, vp=pool, slots=slots, **kw):
        return lambda: int4.append_rope_int4(k, v, cos, sin, kp, vp, slots, **kw)

    def gather(kp=pool, vp=pool, tiles=tiles, n=4, dtype=BF):
        return lambda: int4.gather_int4(kp, vp, tiles, n, dtype)

    def rotate(pools=(pool,), tiles=tiles, inv=torch.ones(64), dtype=BF):
        return lambda: int4.rotate_keys_int4(pools, tiles, 3, inv, dtype)

    def decode(q=q, k=pool, v=pool, scale=1.0, lengths=None, tiles=tiles, splits=None):
        return lambda: int4.decode_attention_int4(q, k, v, scale, lengths, tiles=tiles, splits=splits)

    def gemv(x=q[0], w=w, **kw):
        return lambda: int4.gemv_int4(x, w, **kw)

    off = torch.zeros(4 * 2 * 64 * 80 + 16, dtype=torch.uint8, device=DEV)[8:-8].view(pool.shape)
    wide = torch.zeros(4, 2, 64, 84, dtype=torch.uint8, device=DEV)[..., :80]
    for call in (
            append(k=k.float(), v=k.float()), append(v=k.half()), append(v=k[:1]), append(q=k.half()), append(q=k[:, :2]),
            append(cos=cos.half(), sin=cos.half()), append(sin=cos[:, :64]), append(cos=cos[:2], sin=cos[:2]),
            append(cos=cos[:, :3], sin=cos[:, :3]), append(cos=torch.ones(3, 256, device=DEV), sin=torch.ones(3, 256, device=DEV)),
            append(kp=pool.int()), append(kp=pool[:, :1]), append(vp=pool[:, :, :32]), append(kp=off, vp=off),
            append(kp=wide, vp=wide), append(slots=slots.long()), append(slots=slots[:2]), append(slots=slots.t().repeat(1, 2)),
            append(q_norm=cos[0, :64]), append(k_norm=cos[0].float()), append(eps=-1.0), append(eps=float("nan")),
            append(k=k[None].repeat(2, 1, 1, 1), v=k[None].repeat(2, 1, 1, 1)), append(k=k[..., :96], v=k[..., :96]),
            lambda: int4.write_int4(k, k, pool, pool, slots[:1]),
            gather(tiles=tiles[:, :3].contiguous()), gather(tiles=tiles.long()), gather(n=-1), gather(dtype=torch.float32),
            gather(kp=pool[..., :48], vp=pool[..., :48]), gather(kp=off, vp=off), gather(vp=pool[:2]),
            rotate(inv=torch.ones(32)), rotate(tiles=tiles[:, :2].contiguous()), rotate(dtype=torch.float32),
            rotate(pools=(pool, pool[:2])), rotate(pools=(off,)), rotate(tiles=tiles.t()),
            decode(q=q.float()), decode(k=pool.int(), v=pool.int()), decode(scale=float("inf")), decode(splits=-1),
            decode(splits=70000), decode(q=q.repeat(1, 5, 1)), decode(q=q[..., :96]), decode(q=q[:1]), decode(k=off, v=off),
            decode(tiles=tiles.long()), decode(tiles=tiles[:, :2].contiguous()), decode(lengths=tiles[0, :1]),
            decode(tiles=None, q=q[None].repeat(3, 1, 1, 1)), decode(tiles=None, q=q[None].repeat(4, 1, 1, 1), lengths=tiles[0, :3]),
            gemv(x=q[0].half()), gemv(x=q[0].float()), gemv(x=q[0, :, :100]), gemv(swiglu=True), gemv(w=w._replace(n=33)),
            gemv(w=w._replace(k=130)), gemv(w=w._replace(group=48)), gemv(w=w._replace(codes=w.codes.int())),
            gemv(w=w._replace(params=w.params.half())), gemv(w=w._replace(codes=w.codes[..., ::2].repeat(1, 1, 2)[..., :511]))):
        with pytest.raises((ValueError, TypeError)):
            call()
    assert not pool.any()


def test_many_layers_rotate_in_turns():
    pools = [ref.rows_of(torch.randn(1, 1, 32, 64, device=DEV).to(BF)) for _ in range(131)]
    want = [p.clone() for p in pools]
    tiles = torch.tensor([[0, 3, 20]], dtype=torch.int32, device=DEV)
    inv = 1.0 / (1e4 ** (torch.arange(0, 64, 2).float() / 64))
    int4.rotate_keys_int4(pools, tiles, -5, inv, BF)
    for p in want:
        int4.rotate_keys_int4([p], tiles, -5, inv, BF)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
