"""The decoder with 4-bit weights on one rank and on two `gloo` ranks, on CPU: slicing, quantising, the sums over ranks and the
gathered logits are the product code, the launches of the step are torch restatements (the projections with what the 4-bit weights
stand for). Expected: the model in fp32 with those values as its weights."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from transformers import AutoModelForCausalLM, Qwen3Config

import test_tp_cpu as plain
from threadcut_b200 import int4, tp

N = 20


def models():
    torch.manual_seed(0)
    # every rank's slice of the columns is whole groups of 64, so that its weights are those of the whole matrix
    cfg = Qwen3Config(vocab_size=512, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=16, max_position_embeddings=4096)
    model, exact = (AutoModelForCausalLM.from_config(cfg, dtype=t, attn_implementation="eager").eval()
                    for t in (torch.bfloat16, torch.float32))
    with torch.no_grad():
        for a, b in zip(exact.parameters(), model.parameters()):
            a.copy_(b)
        for m in exact.modules():
            if isinstance(m, torch.nn.Linear):
                m.weight.copy_(int4.dequantize_weight(int4.quantize_weight(m.weight.to(torch.bfloat16))))
    return model, exact


def run(rank, world):
    model, exact = models()
    ids = torch.randint(0, 512, (1, N + 1), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = exact(input_ids=ids).logits[0, -1]
        held = exact(input_ids=ids[:, :N], use_cache=True).past_key_values
        dec = tp.TPDecoder(model, "cpu", world=world, rank=rank, group=None, weight_bits=4)
        assert not dec.use_peer_sums and all(isinstance(w, int4.Int4Weight) for layer in dec.layers_w
                                             for w in (layer.wqkv, layer.wo, layer.wgu, layer.wd))
        assert (dec.lm_head.n, dec.layers_w[0].wo.k, dec.layers_w[0].wd.k) == (512 // world, 128 // world, 256 // world)
        for i, layer in enumerate(held.layers):
            dec.load(i, layer.keys.to(torch.bfloat16), layer.values.to(torch.bfloat16))
        logits = dec.logits(ids[0, N:], N).float()
        dec.crop(N)
        token = int(dec.step(ids[0, N:], N))
    # a token passes some 10 roundings a layer to at most 2^-8, each rank's sums one more: two layers move a logit by about
    # sqrt(24) 2^-9 of the logits' own size, 1 %, and 5e-5 of a correlation; the cache's rounding is of that kind too
    corr = torch.corrcoef(torch.stack([logits, want]))[0, 1].item()
    return corr, token == int(logits.argmax()), bool(want[logits.argmax()] >= want.max() - 0.1 * want.std())


def stand_ins(target):
    plain._cpu_ops(target)
    target(tp, "_gemv", lambda x, w: (x.float() @ int4.dequantize_weight(w).t()).to(x.dtype))
    target(tp, "_gemv_swiglu", lambda gu, w: (torch.nn.functional.silu(gu[:, :w.k].float()).to(gu.dtype) * gu[:, w.k:]).float()
           .matmul(int4.dequantize_weight(w).t()).to(gu.dtype))


def worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        stand_ins(setattr)
        q.put((rank, run(rank, world)))
    finally:
        dist.destroy_process_group()


def check(result):
    corr, same, near = result
    assert corr > 0.999 and same and near, result


def test_one_rank(monkeypatch):
    stand_ins(monkeypatch.setattr)
    check(run(0, 1))


@pytest.mark.parametrize("world", [2])
def test_gloo_ranks(world):
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), plain._free_port()
    procs = [ctx.Process(target=worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=120)
    assert all(p.exitcode == 0 for p in procs), [p.exitcode for p in procs]
    for _, result in sorted(q.get(timeout=5) for _ in range(world)):
        check(result)
