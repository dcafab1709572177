"""The serving example's own bookkeeping, without a GPU: a stand-in for the library keeps the allocations, moves bytes,
forms the slots by the plain rules and computes nothing else."""
import ctypes as C

import numpy as np
import pytest

from fak_amd import serving_step
from tests import kv4_cases as kc


class Library:
    def __init__(self, monkeypatch):
        self.live, self.calls, self.fail_at = {}, [], None
        for name in ("alloc_call", "call", "load"):
            monkeypatch.setattr(serving_step.fakhip, name, getattr(self, name))

    def load(self):
        return self

    def fhip_kv4_cache_bytes(self, pages, page, heads_kv, dim):
        return pages * heads_kv * page // 16 * 18 * dim

    def fhip_free(self, ptr):
        del self.live[ptr]  # an unknown pointer, or one freed before, is an error

    def alloc_call(self, fn, *args):
        if self.fail_at is not None:
            self.fail_at -= 1
            if self.fail_at < 0:
                raise MemoryError(fn)
        block = C.create_string_buffer(args[0] if fn == "fhip_malloc" else 16)
        self.live[C.addressof(block)] = block
        return C.addressof(block)

    def ints(self, ptr, n):
        return np.frombuffer((C.c_int32 * n).from_address(ptr), np.int32) if n else np.zeros(0, np.int32)

    def call(self, fn, *a):
        self.calls.append(fn)
        if fn in ("fhip_h2d", "fhip_d2h"):
            C.memmove(a[0], a[1], a[2])
        elif fn == "fhip_kv_slots_i32":
            R, T, cols, free_pages, page = a[10:]
            lens, new, free, taken = (self.ints(p, n) for p, n in zip(a[:4], (R, R, free_pages, 1)))
            out = kc.slots(lens, new, free, int(taken[0]), self.ints(a[4], R * cols).reshape(R, cols), T, page)
            for p, x in zip((a[5], a[6], a[7], a[8], a[9], a[4]), out):
                self.ints(p, x.size)[:] = x.ravel()


@pytest.fixture
def library(monkeypatch):
    return Library(monkeypatch)


def server(**kw):
    return serving_step.Server(3, 64, **{**dict(hidden=256, heads=4, heads_kv=2, dim=64, layers=1, vocab=256, page=16), **kw})


def held(s, lib):
    return lib.ints(s.lens.ptr, s.R).tolist(), int(lib.ints(s.taken.ptr, 1)[0])


def test_a_step_frees_what_it_took(library):
    s = server()
    before = set(library.live)
    for tokens in ([[1, 2, 3], [4], [5, 6]], [[7], [8], [9]], [[], [1], []]):
        s.step(tokens)
        assert set(library.live) == before
    assert held(s, library)[0] == [4, 3, 3]
    s.close()
    assert not library.live


@pytest.mark.parametrize("n", range(15))
def test_a_failed_allocation_leaves_nothing_behind(library, n):
    s = server()
    before = set(library.live)
    library.fail_at = n
    with pytest.raises(MemoryError):
        s.step([[1, 2], [3], []])
    library.fail_at = None
    assert set(library.live) == before and held(s, library) == ([0, 0, 0], 0)


def test_a_server_that_cannot_be_built_leaves_nothing_behind(library):
    s = server()
    n = len(library.live)
    s.close()
    for i in range(n):
        library.fail_at = i
        with pytest.raises(MemoryError):
            server()
        assert not library.live


def test_all_requests_wait(library):
    s = server()
    s.step([[1, 2], [3], []])
    state, before = held(s, library), set(library.live)
    assert s.step([[], [], []]) == [None] * 3
    assert held(s, library) == state and set(library.live) == before
    assert s.step([[4], [], [5]])[1] is None and held(s, library)[0] == [3, 1, 1]


def test_a_refused_step_changes_nothing(library):
    """A request past its table's row: the others' lengths and pages stay too, as no key was written."""
    s = server()
    s.step([[1] * 20, [2], [3]])
    state, before = held(s, library), set(library.live)
    library.calls.clear()
    with pytest.raises(RuntimeError):
        s.step([[4], [5] * 64, [6]])
    assert held(s, library) == state and set(library.live) == before
    assert "fhip_kv4_append_f32" not in library.calls
    s.step([[4], [5], [6]])
    assert held(s, library) == ([21, 2, 2], 4)
