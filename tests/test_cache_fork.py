"""Shared pages of the KV cache on the CPU (KVCacheState.cpp through
tests/kv_fork_shim.cpp): forks share full pages and get a page of their own for
the partly filled one, a page is freed by its last owner, a sequence takes a
page of its own before it appends into a shared one, and a sequence's pages are
replaced all or nothing."""

import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "aicompiler-test_b200", "csrc")


@pytest.fixture(scope="module")
def kv(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("kvfork") / "libkvfork.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-I", os.path.join(ROOT, "tests"),
                    os.path.join(ROOT, "tests", "kv_fork_shim.cpp"), os.path.join(CSRC, "KVCacheState.cpp"),
                    "-o", out], check=True, capture_output=True)
    lib = ctypes.CDLL(out)
    p, z, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
    ip, zp = ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t)
    for name, res, args in [
            ("kv_last_error", ctypes.c_char_p, []), ("kv_pool_new", p, [z, z]), ("kv_pool_free", None, [p]),
            ("kv_pool_stats", None, [p, zp]), ("kv_pool_allocate", i, [p]), ("kv_pool_release", i, [p, i]),
            ("kv_pool_is_allocated", i, [p, i]), ("kv_pool_fail_next", None, [p, z]), ("kv_pool_retain", i, [p, i]),
            ("kv_pool_owners", z, [p, i]), ("kv_state_new", p, [p, z, i, i]), ("kv_state_free", None, [p]),
            ("kv_state_stage", i, [p, z]), ("kv_state_rollback", i, [p, z]), ("kv_state_reset", i, [p]),
            ("kv_state_commit", i, [p, z]), ("kv_state_length", z, [p]), ("kv_state_pages", z, [p, ip, z]),
            ("kv_state_row", z, [p, ip, z]), ("kv_sink_fail_next", None, [p, i]), ("kv_sink_count", z, [p]),
            ("kv_sink_row", z, [p, z, ip, z]), ("kv_state_fork", i, [p, p, ip]), ("kv_state_unshare", i, [p, ip]),
            ("kv_state_replace", i, [p, z, ip, z, z])]:
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
    return lib


class World:
    def __init__(self, kv, pages=10, size=4, capacity=16, states=3, sink=True):
        self.kv = kv
        self.pool = kv.kv_pool_new(size, pages)
        self.states = [kv.kv_state_new(self.pool, capacity, s, int(sink)) for s in range(states)]

    def grow(self, s, length):
        assert self.kv.kv_state_stage(self.states[s], length) == 0
        assert self.kv.kv_state_commit(self.states[s], length) == 0

    def pages(self, s):
        out = (ctypes.c_int * 64)()
        return list(out[:self.kv.kv_state_pages(self.states[s], out, 64)])

    def used(self):
        out = (ctypes.c_size_t * 6)()
        self.kv.kv_pool_stats(self.pool, out)
        return out[1]

    def owners(self, page):
        return self.kv.kv_pool_owners(self.pool, page)

    def fork(self, source, s):
        out = (ctypes.c_int * 8)()
        n = self.kv.kv_state_fork(self.states[s], self.states[source], out)
        return n if n < 0 else [(out[2 * i], out[2 * i + 1]) for i in range(n)]

    def unshare(self, s):
        out = (ctypes.c_int * 8)()
        n = self.kv.kv_state_unshare(self.states[s], out)
        return n if n < 0 else [(out[2 * i], out[2 * i + 1]) for i in range(n)]

    def sent(self, s):
        out = (ctypes.c_int * 64)()
        last = self.kv.kv_sink_count(self.states[s]) - 1
        return [x for x in out[:self.kv.kv_sink_row(self.states[s], last, out, 64)] if x >= 0]

    def close(self):
        for s in self.states:
            self.kv.kv_state_free(s)
        assert self.used() == 0
        self.kv.kv_pool_free(self.pool)


def test_forks_share_full_pages_and_own_their_last(kv):
    w = World(kv)
    w.grow(0, 10)  # two full pages and half of a third
    a = w.pages(0)
    assert w.fork(0, 1) == [(a[2], w.pages(1)[2])]
    assert w.fork(0, 2) == [(a[2], w.pages(2)[2])]
    for s in (1, 2):
        assert w.pages(s)[:2] == a[:2] and w.pages(s)[2] not in a and w.sent(s) == w.pages(s)
        assert kv.kv_state_length(w.states[s]) == 10
    assert [w.owners(p) for p in a] == [3, 3, 1] and w.used() == 5
    assert kv.kv_state_reset(w.states[0]) == 0
    assert [w.owners(p) for p in a] == [2, 2, 0] and w.used() == 4
    w.close()


def test_a_fork_of_whole_pages_copies_nothing(kv):
    w = World(kv)
    w.grow(0, 8)
    assert w.fork(0, 1) == [] and w.used() == 2
    assert w.unshare(1) == []  # the next position starts a page
    w.grow(1, 9)
    assert w.pages(1)[:2] == w.pages(0) and w.used() == 3
    w.close()


def test_appending_into_a_shared_page_takes_an_own_one(kv):
    w = World(kv)
    w.grow(0, 8)
    w.fork(0, 1)
    shared = w.pages(0)
    assert kv.kv_state_rollback(w.states[1], 6) == 0  # into the second shared page
    got = w.unshare(1)
    assert got == [(shared[1], w.pages(1)[1])] and w.pages(1)[0] == shared[0] and w.pages(1)[1] != shared[1]
    assert w.owners(shared[1]) == 1 and w.sent(1) == w.pages(1) and w.unshare(1) == []
    assert kv.kv_state_rollback(w.states[0], 6) == 0
    assert w.unshare(0) == []  # nobody else has it any more
    w.close()


def test_forks_fail_whole(kv):
    w = World(kv, pages=4)
    w.grow(0, 10)
    used = w.used()
    kv.kv_pool_fail_next(w.pool, 1)
    assert w.fork(0, 1) == -1 and b"exhausted" in kv.kv_last_error()
    assert w.used() == used and w.pages(1) == [] and [w.owners(p) for p in w.pages(0)] == [1, 1, 1]
    kv.kv_sink_fail_next(w.states[1], 1)
    assert w.fork(0, 1) == -1
    assert w.used() == used and w.pages(1) == [] and [w.owners(p) for p in w.pages(0)] == [1, 1, 1]
    assert w.fork(1, 2) == -1  # nothing to fork from
    assert len(w.fork(0, 1)) == 1
    assert w.fork(0, 1) == -1 and b"empty" in kv.kv_last_error()
    w.close()


def test_taking_an_own_page_fails_whole(kv):
    w = World(kv)
    w.grow(0, 8)
    w.fork(0, 1)
    kv.kv_state_rollback(w.states[1], 6)
    before = w.pages(1)
    kv.kv_pool_fail_next(w.pool, 1)
    assert w.unshare(1) == -1 and w.pages(1) == before
    kv.kv_sink_fail_next(w.states[1], 1)
    assert w.unshare(1) == -1 and w.pages(1) == before and w.used() == 2 and w.owners(before[1]) == 2
    w.close()


def test_pages_are_replaced_whole(kv):
    w = World(kv)
    w.grow(0, 14)
    old = w.pages(0)
    new = [kv.kv_pool_allocate(w.pool)]
    arr = (ctypes.c_int * 1)(*new)
    kv.kv_sink_fail_next(w.states[0], 1)
    assert kv.kv_state_replace(w.states[0], 1, arr, 1, 7) == -1
    assert w.pages(0) == old and kv.kv_state_length(w.states[0]) == 14
    assert kv.kv_state_replace(w.states[0], 1, arr, 1, 9) == -1  # does not hold nine
    assert kv.kv_state_replace(w.states[0], 1, arr, 1, 7) == 0
    assert w.pages(0) == [old[0], new[0]] and w.sent(0) == w.pages(0) and w.used() == 2
    assert kv.kv_state_length(w.states[0]) == 7
    w.close()


def test_pages_count_their_owners(kv):
    w = World(kv)
    page = kv.kv_pool_allocate(w.pool)
    assert kv.kv_pool_retain(w.pool, page) == 0 and w.owners(page) == 2
    assert kv.kv_pool_release(w.pool, page) == 0 and kv.kv_pool_is_allocated(w.pool, page) == 1
    assert kv.kv_pool_release(w.pool, page) == 0 and kv.kv_pool_is_allocated(w.pool, page) == 0
    assert kv.kv_pool_release(w.pool, page) == -1 and kv.kv_pool_retain(w.pool, page) == -1
    assert kv.kv_pool_retain(w.pool, 99) == -1 and w.owners(-1) == 0
    w.close()
