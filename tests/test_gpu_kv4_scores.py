"""Scores of any size. Dimension 0 of a key has one of sixteen levels (its codes) and a query reads only that dimension, so
scores are exact products and lie far apart: the keys of the highest level share the weights evenly.

From scores of 2^25 on, the 14 that is added to a weight's exponent is rounded to as much as 16, and a weight of 2^16
passes f16; as two terms cut toward zero it is still itself."""
import numpy as np
import pytest

from tests.test_gpu_kv4_attention import Batch
from tests.test_gpu_kv4_kernels import relay, wide

pytestmark = pytest.mark.gpu


def levels(L, Hk, D, rng):
    """Keys whose dimension 0 is -8..7 (as codes), and values of their own for each level."""
    level = rng.integers(0, 16, L)
    level[:16] = rng.permutation(16)  # each of them somewhere
    k = np.zeros((L, Hk, D), np.float32)
    k[:, :, 1] = -8  # the block's extreme: its scale is the same for all keys
    k[:, :, 0] = (level - 8)[:, None]
    v = np.zeros((L, Hk, D), np.float32)
    for d in range(D):
        v[:, :, d] = np.where(level % 16 == d % 16, rng.choice([-8.0, 4.0, 6.0], L), 0)[:, None]
        if d % 32 == 0:
            v[:, :, d] = np.where(level == 0, -8.0, 0)[:, None]
    return k, v


@pytest.mark.parametrize("wide_table", [False, True])
@pytest.mark.parametrize("gap", [3e3, 1e6, 3e6, 1.1e7, 4e7, 1e9, 1e15])
@pytest.mark.parametrize("D,new", [(64, 1), (128, 3), (256, 1), (128, 40)])
def test_scores_of_any_size(hip, D, new, gap, wide_table):
    """Scores far apart and far from 0: the keys of the highest share the weights evenly."""
    print(f"[attend] D={D} new={new} gap={gap} wide={wide_table}", flush=True)
    rng = np.random.default_rng(8)
    b = Batch([333, 64], [new, min(new, 64)], 14, 2, D, 16, seed=1)
    relay(b, [levels(int(n), 2, D, rng) for n in b.lens])
    q = np.zeros_like(b.q)
    q[:, :, 0] = rng.choice([-1.0, 1.0], q.shape[:2])
    b.check(q=q, scale=gap, table=wide(b) if wide_table else None)
