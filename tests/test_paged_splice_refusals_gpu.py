"""A splice that is refused leaves a paged cache as it was."""
import pytest
import torch

from threadcut_b200.match import Split
from threadcut_b200.paged import PagedKV, PagedKVInt4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("store", [PagedKV, PagedKVInt4])
def test_frequencies_of_another_head_size(store):
    d = 128
    kv = store(2, 2, d, max_tokens=200, device=DEV)
    kv.reserve(150)
    for layer in range(2):
        kv.write(layer, *(torch.randn(2, 150, d, device=DEV).to(torch.bfloat16) for _ in range(2)))
    held = [kv.gather(layer) for layer in range(2)]
    for bad in (torch.ones(32), torch.ones(128), torch.ones(0)):
        with pytest.raises(ValueError, match="inv_freq"):
            kv.splice(Split(20, 50, 100), bad)
        assert kv.n == 150
    assert all(torch.equal(a, b) for layer in range(2) for a, b in zip(kv.gather(layer), held[layer]))
    kv.splice(Split(20, 50, 100), torch.ones(64))
    assert kv.n == 120
    kv.splice(Split(20, 20, 100), torch.ones(3))  # nothing in between: nothing is rotated
    assert kv.n == 120
    kv.splice(Split(20, 120, 0), torch.ones(3))   # nothing behind
    assert kv.n == 20
