"""How exact the log probabilities' sums are.

Tolerance of ordinary rows: an output is rounded once, 2^-24 of itself (6e-8); log S takes over the relative error of
S, at most some 5e-7 where terms are off by the rounding of their exponents (|x - m| log2 e 2^-24, 2e-7 where most of S
lies) and sums of a few hundred terms by a few 2^-24."""
import numpy as np
import pytest

from fak_amd import fakhip
from tests import kv4_cases as kc
from tests.gpu_util import Dev

pytestmark = pytest.mark.gpu


def run(x, tokens, top):
    rows, n = x.shape
    with Dev.from_host(x) as dx, Dev.from_host(tokens.astype(np.int32)) as dt, Dev(rows * 4) as dl, Dev(rows * 4) as de, \
            Dev(rows * top * 4) as dtl, Dev(rows * top * 4) as dti:
        fakhip.call("fhip_logprobs_f32", dx.ptr, dt.ptr, dl.ptr, de.ptr, dtl.ptr, dti.ptr, rows, n, n, top)
        return dl.to_host(np.float32), de.to_host(np.float32), dtl.to_host(np.float32).reshape(rows, top)


@pytest.mark.parametrize("rows,n", [(96, 49152), (300, 1000), (40, 152064)])
def test_ordinary_rows(hip, rows, n):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    x[np.arange(rows), rng.integers(0, n, rows)] += 12
    tokens = rng.integers(0, n, rows)
    got, want = run(x, tokens, 5), kc.logprobs(x, tokens, 5)[:3]
    for name, g, w in zip(("log probability", "entropy", "alternatives"), got, want):
        off = np.abs(g - w) / (6e-8 * np.abs(w) + 5e-7)
        print(f"[logprobs] {rows} rows of {n}: {name} {off.max():.2f} of the tolerance", flush=True)
        assert off.max() <= 1, name


@pytest.mark.parametrize("rows,n,apart", [(64, 1 << 20, 1 << 20), (64, 1 << 20, 2048), (2, (1 << 24) - 3, 1 << 24)])
def test_many_small_terms_beside_the_largest(hip, rows, n, apart):
    """All logits but some are 17.4 below the largest: one of their terms is less than half a last bit of a sum that holds
    the largest's 1, all of a lane's together are not. The sums of two kinds of terms are known exactly."""
    x = np.full((rows, n), -17.4, np.float32)
    tops = np.arange(5, n, apart)
    x[:, tops] = 0
    few, rest, d = len(tops), n - len(tops), float(np.float32(-17.4))
    S = few + rest * np.exp(d)
    logp, entropy, top = run(x, np.full(rows, 5), 1)
    print(f"[logprobs] {rows} rows of {n}: {np.abs(logp + np.log(S)).max():.2e}", flush=True)
    assert np.abs(logp + np.log(S)).max() <= 2e-6 and np.abs(top + np.log(S)).max() <= 2e-6
    assert np.abs(entropy - (np.log(S) - rest * d * np.exp(d) / S)).max() <= 2e-6 * (1 + entropy.max())
