"""The serving example's model in plain numpy, a request at a time and in 64 bits but for what the cache holds: the
oracle of what Server.step answers."""
from __future__ import annotations

import numpy as np

import oracle
from fak_amd import synth
from tests import kv4_cases as kc


def rms(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)


def turned(x):
    """Rotary positions: dimensions i and i + half of token t turned by t 10000^(-i / half)."""
    T, _, D = x.shape
    f = np.exp(-np.log(10000.0) * np.arange(D // 2) / (D // 2))
    z = (x[..., : D // 2] + 1j * x[..., D // 2:]) * np.exp(1j * np.arange(T)[:, None, None] * f)
    return np.concatenate([z.real, z.imag], -1)


def stored(x):
    """What the 4-bit cache holds of x."""
    return kc.values(*kc.quantize(x.astype(np.float32)))


class Model:
    def __init__(self, hidden, heads, heads_kv, dim, layers, vocab, window, seed=1, noise=0.0, **_):
        def weight(out, in_, s):
            return oracle.q4k_dequant(synth.q4k_weights(out, in_, s), out, in_).astype(np.float64).T

        shapes = [(heads * dim, hidden), (heads_kv * dim, hidden), (heads_kv * dim, hidden), (hidden, heads * dim)]
        self.layers = [[weight(o, i, seed + 7 * n + j) for j, (o, i) in enumerate(shapes)] for n in range(layers)]
        self.head = weight(vocab, hidden, seed + 1000)
        self.H, self.HK, self.D, self.hidden, self.window, self.noise = heads, heads_kv, dim, hidden, window, noise

    def sight(self, i, n):
        """Keys that token i of n sees."""
        return slice(max(0, i + 1 - self.window) if self.window else 0, i + 1)

    def product(self, x, w):
        y = x @ w
        if self.noise:  # errors of a product, of so much of its outputs' RMS
            y = y + self.noise * np.sqrt((y * y).mean()) * np.random.default_rng(y.size).standard_normal(y.shape)
        return y

    def attention(self, q, k, v):
        T, G = len(q), self.H // self.HK
        o = np.zeros((T, self.H, self.D))
        for i in range(T):
            see = self.sight(i, T)
            for h in range(self.H):
                s = k[see, h // G] @ q[i, h] * self.D ** -0.5
                e = np.exp(s - s.max())
                o[i, h] = e @ v[see, h // G] / e.sum()
        return o

    def log_probabilities(self, tokens):
        """Of every next token, after each of a request's tokens: [tokens, vocab]."""
        x = np.stack([np.random.default_rng(int(t)).standard_normal(self.hidden).astype(np.float32) for t in tokens]).astype(np.float64)
        T = len(x)
        for wq, wk, wv, wo in self.layers:
            y = rms(x)
            q, k = (turned(rms(self.product(y, w).reshape(T, n, self.D))) for w, n in ((wq, self.H), (wk, self.HK)))
            v = self.product(y, wv).reshape(T, self.HK, self.D)
            x = x + rms(self.product(self.attention(q, stored(k), stored(v)).reshape(T, -1), wo))
        z = self.product(rms(x) * 0.01, self.head)
        return z - z.max(-1, keepdims=True) - np.log(np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True))
