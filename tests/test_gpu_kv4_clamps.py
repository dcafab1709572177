"""What the entry makes of wrong tables and lengths: a page id past the cache is its last page, a negative one its
first, a length past the table row the row's end. Each is compared, bit by bit, with the call that says so; every byte
of these caches is a written one, so that no NaN hides a difference."""
import numpy as np
import pytest

from tests.test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu


def full(new, positions, seed):
    """A batch whose pages are all full, in tables of so many positions that name them again and again: with 40 new
    tokens and 32,768 positions the prefill kernel's, else the split kernel's."""
    b = Batch([96, 160], new, 14, 2, 64, 16, seed=seed, spare=0)
    table = np.random.default_rng(seed).integers(0, b.pages, (2, positions // 16)).astype(np.int32)
    b.table = table
    return b


@pytest.mark.parametrize("new,positions", [([1, 1], 512), ([1, 5], 32768), ([40, 40], 512), ([40, 40], 32768)])
def test_page_ids(hip, new, positions):
    print(f"[attend] ids new={new} positions={positions}", flush=True)
    b = full(new, positions, 41)
    b.lens = np.array([positions // 2 - 3, 400], np.int32)
    clean = b.run()
    assert np.isfinite(clean).all()
    for wrong, right in ((b.pages, b.pages - 1), (b.pages + 1, b.pages - 1), (1 << 30, b.pages - 1), (2**31 - 1, b.pages - 1), (-1, 0), (-5, 0), (-2**31, 0)):
        tables = [b.table.copy() for _ in range(2)]
        for t, page in zip(tables, (wrong, right)):
            t[0, [0, 3, positions // 32 - 1]] = page
            t[1, [1, 24]] = page  # 24: where the second request ends
        got, want = (b.run(table=t) for t in tables)
        assert np.isfinite(want).all() and np.array_equal(got, want), (wrong, right)


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("new,positions", [([1, 1], 512), ([1, 5], 32768), ([40, 40], 512), ([40, 40], 32768)])
def test_lengths(hip, new, positions, window):
    print(f"[attend] lengths new={new} positions={positions} window={window}", flush=True)
    b = full(new, positions, 42)
    b.lens = np.array([positions, positions], np.int32)
    want = b.run(window=window)
    assert np.isfinite(want).all()
    for more in (1, 15, 16, 64, 100000, 2**31 - 1 - positions):
        b.lens = np.array([positions + more, positions], np.int32)
        assert np.array_equal(b.run(window=window), want), more
