"""The serving entries around the matmuls as a decode loop uses them: a small random Q4_K transformer (attention
blocks only) that answers a batch of prompts of unequal lengths.

    python -m fak_amd.serving_step --requests 4 --prompt 40 --steps 8 [--layers 2 --page 64 --window 0]

One step on the device: fhip_kv_slots_i32 for the batch, and for each layer the q/k/v products, fhip_kv4_append_f32,
fhip_kv4_attention_f32 and the output product; then the logits' product and fhip_logprobs_f32, whose first
alternative is the next token. Norms, rotary positions and residuals are the host's (the library has none). Weights
and embeddings are random: the answers mean nothing, the log probabilities and their times are real.
"""
from __future__ import annotations

import argparse
import contextlib
import ctypes as C
import time

import numpy as np

from . import fakhip, synth


class Buffer:
    """Device memory of one array, the default pool's."""

    def __init__(self, nbytes: int, host: np.ndarray = None):
        self.ptr = fakhip.alloc_call("fhip_malloc", max(nbytes, 16))
        if host is not None:
            try:
                self.put(host)
            except Exception:
                self.free()
                raise

    def put(self, a: np.ndarray) -> None:
        a = np.ascontiguousarray(a)
        fakhip.call("fhip_h2d", self.ptr, a.ctypes.data, a.nbytes)

    def get(self, shape, dtype=np.float32) -> np.ndarray:
        a = np.empty(shape, dtype)
        fakhip.call("fhip_d2h", a.ctypes.data, self.ptr, a.nbytes)
        return a

    def free(self) -> None:
        fakhip.load().fhip_free(self.ptr)


def ints(a) -> Buffer:
    a = np.asarray(a, np.int32)
    return Buffer(a.nbytes, a)


def unit_rows(x: np.ndarray) -> np.ndarray:
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + 1e-6)


def rotate(x: np.ndarray, pos: np.ndarray) -> np.ndarray:
    """Rotary positions of [tokens, heads, dim]; a token without a position (-1) stays."""
    half = x.shape[-1] // 2
    angle = np.maximum(pos, 0)[:, None, None] * (10000.0 ** (-np.arange(half) / half))[None, None]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1).astype(np.float32)


class Server:
    """Requests that share one page pool. `step` takes each request's new tokens."""

    def __init__(self, requests, positions, hidden=3584, heads=28, heads_kv=4, dim=128, layers=2, vocab=8192, page=64, window=0, top=5, seed=1):
        self.R, self.hidden, self.H, self.HK, self.D = requests, hidden, heads, heads_kv, dim
        self.vocab, self.page, self.window, self.top = vocab, page, window, top
        self.cols = -(-positions // page)
        self.pages = requests * self.cols
        self.held = []
        try:
            self.fill(layers, seed)
        except Exception:
            self.close()
            raise

    def fill(self, layers, seed) -> None:
        """Weights, caches and the pages' bookkeeping."""
        size = fakhip.load().fhip_kv4_cache_bytes(self.pages, self.page, self.HK, self.D)
        self.layers = []
        for i in range(layers):
            w = [self.weight(out, in_, seed + 7 * i + j)
                 for j, (out, in_) in enumerate([(self.H * self.D, self.hidden), (self.HK * self.D, self.hidden), (self.HK * self.D, self.hidden),
                                                 (self.hidden, self.H * self.D)])]
            self.layers.append((w, self.hold(Buffer(size))))
        self.head = self.weight(self.vocab, self.hidden, seed + 1000)
        self.free_list = self.hold(ints(np.random.default_rng(seed).permutation(self.pages)))
        self.table = self.hold(ints(np.full((self.R, self.cols), -1)))
        self.lens, self.lens_next = self.hold(ints(np.zeros(self.R))), self.hold(ints(np.zeros(self.R)))
        self.taken, self.taken_next = self.hold(ints([0, 0])), self.hold(ints([0, 0]))
        self.start = self.hold(ints(np.zeros(self.R + 1)))

    def hold(self, b: Buffer) -> Buffer:
        self.held.append(b)
        return b

    def weight(self, out, in_, seed):
        raw = synth.q4k_weights(out, in_, seed)
        b = Buffer.__new__(Buffer)
        b.ptr = fakhip.alloc_call("fhip_q4k_upload", raw.ctypes.data, out, in_)
        return self.hold(b).ptr

    def close(self) -> None:
        for b in self.held:
            b.free()

    def step(self, tokens):
        """tokens[r]: the request's new token ids (none: it waits). Returns for each request with any the next
        id, and the given tokens' log probabilities where the batch knows them: token i + 1 of a request after
        its token i; and the entropy after its last. A step that finds no room for a request raises and leaves
        lengths and pages as they were."""
        if not any(len(t) for t in tokens):
            return [None] * self.R
        with contextlib.ExitStack() as stack:
            return self.run(tokens, stack)

    def run(self, tokens, stack):
        """A step whose buffers are the stack's."""
        def own(b: Buffer) -> Buffer:
            stack.callback(b.free)
            return b

        flat = np.concatenate([np.asarray(t, np.int64) for t in tokens])
        T, R, H, HK, D = len(flat), self.R, self.H, self.HK, self.D
        counts = [len(t) for t in tokens]
        fresh, slots, pos = own(ints(counts)), own(ints(np.zeros(T))), own(ints(np.zeros(T)))
        q, k, v, o, x_dev, y_dev, logits, logp_dev, entropy_dev, tl_dev, ti_dev = (
            own(Buffer(T * n * 4)) for n in (H * D, HK * D, HK * D, H * D, self.hidden, self.hidden, self.vocab, 1, 1, self.top, self.top))
        given = own(ints(np.concatenate([np.append(np.asarray(t[1:], np.int32), np.int32(-1)) if len(t) else np.zeros(0, np.int32) for t in tokens])))
        fakhip.call("fhip_kv_slots_i32", self.lens.ptr, fresh.ptr, self.free_list.ptr, self.taken.ptr, self.table.ptr, slots.ptr, pos.ptr,
                    self.start.ptr, self.lens_next.ptr, self.taken_next.ptr, R, T, self.cols, self.pages, self.page)
        where = pos.get(T, np.int32)
        if self.taken_next.get(2, np.int32)[1]:  # nothing is written yet, and the pages named in the table are named anew
            raise RuntimeError("requests past the pages or the table")
        self.lens, self.lens_next = self.lens_next, self.lens
        self.taken, self.taken_next = self.taken_next, self.taken
        x = np.stack([np.random.default_rng(int(t)).standard_normal(self.hidden).astype(np.float32) for t in flat])
        for (wq, wk, wv, wo), cache in self.layers:
            x_dev.put(unit_rows(x))
            w = (C.c_void_p * 3)(wq, wk, wv)
            y = (C.c_void_p * 3)(q.ptr, k.ptr, v.ptr)
            fakhip.call("fhip_q4k_matmul_group_f32", w, y, (C.c_int * 3)(H * D, HK * D, HK * D), 3, x_dev.ptr, self.hidden, T)
            q.put(rotate(unit_rows(q.get((T, H, D))), where))
            k.put(rotate(unit_rows(k.get((T, HK, D))), where))
            fakhip.call("fhip_kv4_append_f32", cache.ptr, k.ptr, v.ptr, slots.ptr, T, HK, D, self.pages, self.page, HK * D, HK * D)
            fakhip.call("fhip_kv4_attention_f32", cache.ptr, q.ptr, o.ptr, self.start.ptr, self.lens.ptr, self.table.ptr, R, T, max(counts),
                        H, HK, D, self.pages, self.page, self.cols, H * D, self.window, D ** -0.5)
            fakhip.call("fhip_q4k_matmul_f32", wo, o.ptr, y_dev.ptr, self.hidden, H * D, T)
            x = x + unit_rows(y_dev.get((T, self.hidden)))
        x_dev.put(unit_rows(x) * np.float32(0.01))
        fakhip.call("fhip_q4k_matmul_f32", self.head, x_dev.ptr, logits.ptr, self.vocab, self.hidden, T)
        fakhip.call("fhip_logprobs_f32", logits.ptr, given.ptr, logp_dev.ptr, entropy_dev.ptr, tl_dev.ptr, ti_dev.ptr, T, self.vocab, self.vocab, self.top)
        logp, entropy, ti = logp_dev.get(T), entropy_dev.get(T), ti_dev.get((T, self.top), np.int32)
        out, at = [], 0
        for n in counts:
            out.append((int(ti[at + n - 1, 0]), logp[at:at + n - 1], float(entropy[at + n - 1])) if n else None)
            at += n
        return out


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=40, help="tokens of the longest prompt")
    ap.add_argument("--steps", type=int, default=8, help="tokens answered for each request")
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--seed", type=int, default=1)
    a = ap.parse_args(argv)
    fakhip.init()
    rng = np.random.default_rng(a.seed)
    s = Server(a.requests, a.prompt + a.steps, layers=a.layers, page=a.page, window=a.window, seed=a.seed)
    try:
        tokens = [list(rng.integers(0, s.vocab, rng.integers(1, a.prompt + 1))) for _ in range(a.requests)]
        for i in range(a.steps):
            t0 = time.perf_counter()
            out = s.step(tokens)
            took = time.perf_counter() - t0
            known = np.concatenate([lp for _, lp, _ in out])
            print(f"step {i}: {sum(map(len, tokens))} tokens, {1e3 * took:.1f} ms with the host's part; next {[n for n, _, _ in out]}, "
                  f"entropy {np.mean([e for _, _, e in out]):.3f}" + (f", prompts' log probability {known.mean():.3f} a token" if len(known) else ""))
            tokens = [[n] for n, _, _ in out]
    finally:
        s.close()


if __name__ == "__main__":
    main()
