"""The workspace of a shared-prefix decode, without a GPU: a short prefix leaves the suffixes their slices."""
import pytest

from threadcut_b200 import _lib

HKV, G, D = 8, 4, 128


def parts(batch, n, m):
    """Slices of the prefix and of each suffix together: a slice holds d sums and two statistics a row, in fp32."""
    rows = batch * HKV * G
    size = _lib.lib().tc_decode_attention_shared_workspace_size(batch, HKV, G, D, n, m, 2)
    return round(size / (rows * 4 * (D + 2)))


@pytest.mark.parametrize("batch", [40, 48, 64, 100, 256])
@pytest.mark.parametrize("m", [64, 130, 1500, 4096, 20000])
def test_a_short_prefix_does_not_cut_long_suffixes_small(batch, m):
    """batch * HKV suffixes fill the GPU by themselves: a suffix is at most 3 slices, or slices of 16 key tiles (of 64)
    and more; the prefix of at most 3 tiles at most 3."""
    tiles = -(-m // 64)
    for n in (1, 64, 65, 130, 192):
        assert parts(batch, n, m) <= -(-n // 64) + max(3, tiles // 16)


def test_every_source_has_a_slice():
    for batch in (1, 8, 64):
        assert parts(batch, 0, 0) == 0
        for n, m in ((0, 1), (1, 0)):
            assert parts(batch, n, m) == 1
        for n, m in ((1, 1), (64, 5000), (5000, 64), (100000, 1), (1, 100000)):
            assert parts(batch, n, m) >= 2
