"""A block of 32 values that holds NaN, by the formula: it makes its own 32 dimensions NaN in the heads and tokens that
see its key, and nothing else. That holds wherever the key lies, in a step that all rows of a tile see or at the edge
of the mask."""
import numpy as np
import pytest

from tests.test_gpu_kv4_attention import Batch
from tests.test_gpu_kv4_kernels import wide

pytestmark = pytest.mark.gpu
PLACE = [0, 4, 1, 5, 2, 6, 3, 7, 8, 12, 9, 13, 10, 14, 11, 15]  # of a token's scale among a block's sixteen


def spoil(b, r, j, head, block):
    """The cache with a NaN for the value scale of one block of request r's key j."""
    cache = b.cache.copy()
    at = 17 * b.D + 32 * block + 2 * PLACE.index(j % 16)
    cache[b.table[r, j // b.page], head, j % b.page // 16, at: at + 2] = 0xFF
    return cache


@pytest.mark.parametrize("wide_table", [False, True])
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_only_its_own_dimensions(hip, D, new, window, wide_table):
    print(f"[attend] D={D} new={new} window={window} wide={wide_table}", flush=True)
    L, G = 230, 7
    b = Batch([L, 90], [new, min(new, 90)], 2 * G, 2, D, 16, seed=D + new)
    table = wide(b) if wide_table else None
    clean = b.run(window=window, table=table)
    assert np.isfinite(clean).all()
    for j, block in ((3, 0), (70, 1), (100, D // 32 - 1), (L - 24, 1), (L - new // 2 - 1, 0), (L - 1, D // 32 - 1)):
        got = b.run(window=window, table=table, cache=spoil(b, 0, j, 1, block))
        want = clean.copy()
        for i in range(new):
            p = L - new + i
            if j <= p and (not window or j > p - window):
                want[i, G:, 32 * block: 32 * block + 32] = np.nan
        assert np.array_equal(got, want, equal_nan=True), (j, block, np.argwhere((got != want) & ~(np.isnan(got) & np.isnan(want)))[:5])


@pytest.mark.parametrize("wide_table", [False, True])
def test_two_blocks_of_two_keys(hip, wide_table):
    """Keys of one step, each with another block: a row has what it sees."""
    b = Batch([200], [20], 14, 2, 128, 16, seed=5)
    table = wide(b) if wide_table else None
    want = b.run(table=table)
    cache = spoil(b, 0, 185, 0, 1)
    b.cache = cache
    cache = spoil(b, 0, 195, 0, 3)
    got = b.run(table=table, cache=cache)
    want[5:, :7, 32:64] = np.nan
    want[15:, :7, 96:] = np.nan
    assert np.array_equal(got, want, equal_nan=True)
