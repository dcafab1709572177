"""First tokens that fall from one request to the next name more tokens than the call has: no request of such a call is
taken, its outputs stay as they were, and those past the last request are zeros as ever."""
import numpy as np
import pytest

from tests.test_gpu_kv4_attention import Batch
from tests.test_gpu_kv4_kernels import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("positions", [0, 1 << 15, 1 << 20])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("R,new", [(3, 1), (3, 30), (64, 2), (65, 1), (600, 1), (200, 12)])
def test_falling_starts(hip, R, new, D, positions):
    print(f"[attend] falling starts R={R} new={new} D={D} positions={positions}", flush=True)
    b = Batch([40 + r % 7 for r in range(R)], [new] * R, 14, 2, D, 16, seed=R)
    table = wide(b, positions) if positions else None
    b.check(table=table, pad=3)
    rows = R * new
    for at, to in ((1, rows), (R - 1, 0), (R // 2, -5), (R // 2, 2**31 - 1)):
        right = b.start.copy()
        b.start[at] = to
        got = b.run(table=table, pad=3)
        b.start = right
        assert np.all(got[:rows] == 99) and np.all(got[rows:] == 0), (at, to)
