"""The serving example against a plain model of it: log probabilities of prompts in one batch, in chunks behind what the
cache holds, and token by token.

Tolerance: each product is within 1e-3 of its outputs' RMS at these sizes; errors of that size, put into the plain
model's products, move a log probability by up to 0.02 (a key or value now and then goes to the next of its sixteen
codes). 0.06 is three times that. The second test, without a GPU, shows what wrong attention does: with uniform
weights, another mask or another window the same log probabilities move by at least 0.2."""
import numpy as np
import pytest

from tests.serving_model import Model

SIZE = dict(hidden=512, heads=8, heads_kv=2, dim=64, layers=2, vocab=512, page=16)
TOL = 0.06
LENGTHS = (40, 1, 23)


def prompts():
    rng = np.random.default_rng(3)
    return [list(rng.integers(0, 512, n)) for n in LENGTHS]


def of_given(model):
    """The log probabilities that a batch of the prompts returns."""
    return [model.log_probabilities(p)[np.arange(len(p) - 1), p[1:]] for p in prompts()]


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("chunks", [[40], [17, 4, 19], [1] * 5 + [2] * 17 + [1], [1] * 40])
def test_log_probabilities(hip, window, chunks):
    from fak_amd.serving_step import Server
    given = prompts()
    want = [Model(window=window, **SIZE).log_probabilities(p) for p in given]
    s = Server(3, 64, window=window, **SIZE)
    worst = [0.0]
    try:
        at = 0
        for n in chunks:
            part = [p[at:at + n] for p in given]
            for r, o in enumerate(s.step(part)):
                if o is None:
                    continue
                last = at + len(part[r]) - 1
                expect = want[r][np.arange(at, last), part[r][1:]]
                worst += list(np.abs(o[1] - expect))
                p = want[r][last]
                worst.append(abs(o[2] + (np.exp(p) * p).sum()))
                assert p[o[0]] >= p.max() - TOL  # the most likely, or as good as it
            at += n
        print(f"[serve] window={window} chunks of {chunks[0]}: {max(worst):.4f}", flush=True)
        assert max(worst) <= TOL
    finally:
        s.close()


class Uniform(Model):
    def attention(self, q, k, v):
        return super().attention(q * 0, k, v)


class FirstKeyOnly(Model):
    def sight(self, i, n):
        return slice(0, 1)


class NextKeyToo(Model):
    def sight(self, i, n):
        return slice(super().sight(i, n).start, min(n, i + 2))


class NotItself(Model):
    def sight(self, i, n):
        return slice(super().sight(i, n).start, max(i, 1))


class AnotherWindow(Model):
    def sight(self, i, n):
        return slice(max(0, i - 5 if self.window else i - 10), i + 1)


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("wrong", [Uniform, FirstKeyOnly, NextKeyToo, NotItself, AnotherWindow])
def test_wrong_attention_would_show(wrong, window):
    right, other = (of_given(m(window=window, **SIZE)) for m in (Model, wrong))
    assert max(np.abs(a - b).max() for a, b in zip(right, other) if len(a)) >= 0.2


@pytest.mark.parametrize("window", [0, 5])
def test_errors_of_products_do_not(window):
    right, other = (of_given(Model(window=window, noise=e, **SIZE)) for e in (0.0, 1e-3))
    assert max(np.abs(a - b).max() for a, b in zip(right, other) if len(a)) <= 0.02
