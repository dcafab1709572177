"""Windows near 2^31, the largest that the entry takes: they hide nothing, also from requests with more query tokens
than keys, whose first positions lie below 0."""
import pytest

from tests.test_gpu_kv4_attention import Batch
from tests.test_gpu_kv4_kernels import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide_table", [False, True])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 2**31 - 60])
@pytest.mark.parametrize("H,Hk,D", [(28, 4, 128), (9, 3, 64), (6, 2, 256)])
def test_more_tokens_than_keys(hip, H, Hk, D, window, wide_table):
    print(f"[attend] window={window} heads={H}/{Hk} D={D} wide={wide_table}", flush=True)
    b = Batch([100, 0, 300, 5], [150, 3, 500, 1], H, Hk, D, 16, seed=31)
    b.check(window=window, table=wide(b) if wide_table else None)
    b = Batch([70], [73], H, Hk, D, 16, seed=32)
    b.check(window=window, table=wide(b) if wide_table else None)
