"""The attention plugin's reading of masks, on the CPU: which masks count as the causal one or as a window, also for
tensors made under torch.inference_mode(), which have no version counter."""
from types import SimpleNamespace

import pytest
import torch

from threadcut_b200 import attention as A
from threadcut_b200.prefill import causal_offset_mask


@pytest.fixture(autouse=True)
def _fresh(monkeypatch):
    monkeypatch.setattr(A, "_mask_seen", {})
    monkeypatch.setattr(A, "_window_seen", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def window_mask(lq, lk, w):
    at = (lk - lq + torch.arange(lq))[:, None]
    j = torch.arange(lk)
    return ((j <= at) & (j > at - w))[None, None]


def window_of(mask, lq, lk, w):
    """_window_of for a query that looks like one on the GPU."""
    query = SimpleNamespace(shape=(1, 8, lq, 128), is_cuda=True, dtype=torch.bfloat16, requires_grad=False)
    key = torch.empty(1, 2, lk, 128)
    return A._window_of(query, key, key, mask, lq, lk, 0.1, dict(sliding_window=w))


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("lq,lk,w", [(1, 30, 7), (5, 30, 7), (30, 30, 40)])
def test_a_window_is_known_in_either_mode(mode, lq, lk, w):
    with mode():
        mask = window_mask(lq, lk, w)
        for _ in range(2):
            assert window_of(mask, lq, lk, w) == w
        assert window_of(mask, lq, lk, 3) is None  # another window than the mask's
        mask[0, 0, 0, 0 if w < lk else 1] ^= True  # changed in place: compared anew
        assert window_of(mask, lq, lk, w) is None


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("lq,lk", [(1, 30), (5, 30), (30, 30)])
def test_the_causal_mask_is_known_in_either_mode(mode, lq, lk):
    with mode():
        mask = causal_offset_mask(lq, lk, "cpu")[None, None].clone()
        for _ in range(2):
            assert A._is_causal_offset(mask, lq, lk)
        mask[0, 0, 0, 0] ^= True
        assert not A._is_causal_offset(mask, lq, lk)
        assert not A._is_causal_offset(mask[:, :, :, 1:], lq, lk)


def test_a_mask_of_one_mode_used_in_the_other():
    normal = window_mask(5, 30, 7)
    with torch.inference_mode():
        made_there = window_mask(5, 30, 7)
        assert window_of(normal, 5, 30, 7) == 7
    assert window_of(made_there, 5, 30, 7) == 7
    assert window_of(normal, 5, 30, 7) == 7


def test_values_of_another_head_size_are_no_window():
    """The windowed kernels take keys and values of one shape; SDPA does not need that."""
    query = SimpleNamespace(shape=(1, 8, 5, 128), is_cuda=True, dtype=torch.bfloat16, requires_grad=False)
    key, value, same = (torch.empty(1, 2, 30, d) for d in (128, 64, 128))
    mask, kw = window_mask(5, 30, 7), dict(sliding_window=7)
    assert A._window_of(query, key, same, mask, 5, 30, 0.1, kw) == 7
    assert A._window_of(query, key, value, mask, 5, 30, 0.1, kw) is None


def test_broadcast_keys_are_no_window():
    """The windowed prefill runs them on its plain kernel, which SDPA beats."""
    query = SimpleNamespace(shape=(1, 8, 5, 128), is_cuda=True, dtype=torch.bfloat16, requires_grad=False)
    mask, kw = window_mask(5, 30, 7), dict(sliding_window=7)
    own, shared = torch.empty(1, 2, 30, 128), torch.empty(1, 1, 30, 128).expand(1, 2, 30, 128)
    assert A._window_of(query, own, own, mask, 5, 30, 0.1, kw) == 7
    assert A._window_of(query, own.as_strided(own.shape, (0,) + own.stride()[1:]), own, mask, 5, 30, 0.1, kw) == 7
    for k, v in ((shared, own), (own, shared)):
        assert A._window_of(query, k, v, mask, 5, 30, 0.1, kw) is None


@pytest.mark.parametrize("d,pad", [(64, 1), (64, 8), (128, 3), (20, 1)])
def test_sdpa_gets_rows_on_their_boundaries(monkeypatch, d, pad):
    """Views that start between two 16-byte boundaries are copied, others and rows of an odd length go as they are."""
    seen = []
    real = torch.nn.functional.scaled_dot_product_attention
    monkeypatch.setattr(A.F, "scaled_dot_product_attention", lambda *a, **k: (seen.extend(a), real(*a, **k))[1])
    torch.manual_seed(0)
    full = [torch.randn(1, h, n, d + pad, dtype=torch.bfloat16) for h, n in ((8, 5), (2, 30), (2, 30))]
    x = [t[..., pad:] for t in full]
    mask = window_mask(5, 30, 7)
    out, _ = A.attention(None, *x, mask, scaling=0.1)
    want = real(*(t.contiguous() for t in x), attn_mask=mask, scale=0.1, enable_gqa=True)
    assert torch.equal(out, want.transpose(1, 2))
    for given, used in zip(x, seen):
        if d * 2 % 16 == 0:
            assert used.data_ptr() % 16 == 0 and all(s * 2 % 16 == 0 for s in used.stride()[:-1])
        if d * 2 % 16 or pad == 8:
            assert used.data_ptr() == given.data_ptr()
    leaf = x[1].detach().requires_grad_()  # the copy carries gradients
    A.attention(None, x[0], leaf, x[2], mask, scaling=0.1)[0].float().sum().backward()
    assert leaf.grad is not None and leaf.grad.abs().sum() > 0
