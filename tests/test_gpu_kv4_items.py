"""Single tokens of as many items (requests times key heads) as workgroups of eight waves have places, and of a few
more and less, with tables of a few steps and of many."""
import numpy as np
import pytest

from tests.test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longest", [60, 250, 700])
@pytest.mark.parametrize("items", [248, 264, 376, 392, 504, 512, 520])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_waves(hip, D, items, longest):
    print(f"[attend] D={D} items={items} longest={longest}", flush=True)
    lens = np.random.default_rng(items).integers(0, longest + 1, items // 8)
    lens[3] = longest
    Batch(lens, np.ones(len(lens), int), 16, 8, D, 16, seed=items).check()
