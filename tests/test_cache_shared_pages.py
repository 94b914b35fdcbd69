"""What several sequences share stays as it is, whatever lengths are set by hand: the KV
cache state on the CPU (through tests/kv_fork_shim.cpp and tests/kv_shared_shim.cpp)."""

import ctypes
import os
import subprocess

import pytest

from test_cache_fork import CSRC, ROOT, World, kv  # noqa: F401


@pytest.fixture(scope="module")
def filled(kv, tmp_path_factory):  # noqa: F811
    """The kv library with the calls of kv_shared_shim.cpp."""
    out = str(tmp_path_factory.mktemp("kvshared") / "libkvshared.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-I", os.path.join(ROOT, "tests"),
                    os.path.join(ROOT, "tests", "kv_shared_shim.cpp"), os.path.join(CSRC, "KVCacheState.cpp"),
                    "-o", out], check=True, capture_output=True)
    lib = ctypes.CDLL(out)
    for name in ("kv_last_error", "kv_pool_new", "kv_pool_free", "kv_pool_stats", "kv_pool_allocate", "kv_pool_fail_next",
                 "kv_pool_owners", "kv_state_new", "kv_state_free", "kv_state_stage", "kv_state_rollback",
                 "kv_state_commit", "kv_state_length", "kv_state_pages", "kv_sink_fail_next", "kv_sink_count",
                 "kv_sink_row", "kv_state_fork", "kv_state_unshare"):
        f = getattr(lib, name)
        f.restype, f.argtypes = getattr(kv, name).restype, getattr(kv, name).argtypes
    ip = ctypes.POINTER(ctypes.c_int)
    lib.kv_state_unshare_filled.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ip, ip, ctypes.c_size_t]
    return lib


def test_a_lowered_length_takes_own_pages_for_all_that_is_appended(kv):  # noqa: F811
    w = World(kv, pages=12)
    w.grow(0, 16)
    assert w.fork(0, 1) == []
    shared = w.pages(0)
    assert kv.kv_state_commit(w.states[1], 5) == 0  # keeps the pages behind
    copies = w.unshare(1)
    assert kv.kv_state_stage(w.states[1], 14) == 0
    mine = w.pages(1)
    assert copies == list(zip(shared[1:], mine[1:])) and mine[0] == shared[0]
    assert not set(mine[1:]) & set(shared) and w.sent(1) == mine
    assert [w.owners(p) for p in shared] == [2, 1, 1, 1] and [w.owners(p) for p in mine[1:]] == [1, 1, 1]
    assert w.unshare(1) == []
    assert kv.kv_state_commit(w.states[0], 5) == 0
    assert w.unshare(0) == []  # nobody else has the rest any more
    w.close()


def test_several_own_pages_are_taken_whole_or_not_at_all(kv):  # noqa: F811
    w = World(kv, pages=6)
    w.grow(0, 16)
    w.fork(0, 1)
    kv.kv_state_commit(w.states[1], 5)
    before = w.pages(1)
    assert w.unshare(1) == -1 and b"exhausted" in kv.kv_last_error()  # three wanted, two free
    assert w.pages(1) == before and w.used() == 4 and [w.owners(p) for p in before] == [2] * 4
    kv.kv_state_commit(w.states[1], 9)
    kv.kv_sink_fail_next(w.states[1], 1)
    assert w.unshare(1) == -1
    assert w.pages(1) == before and w.sent(1) == before and w.used() == 4 and [w.owners(p) for p in before] == [2] * 4
    assert len(w.unshare(1)) == 2 and w.used() == 6
    w.close()


def test_committed_positions_without_pages_cannot_be_forked(kv):  # noqa: F811
    w = World(kv)
    assert kv.kv_state_stage(w.states[0], 4) == 0
    for length in (10, 5, 16):  # more than the one page that is there
        assert kv.kv_state_commit(w.states[0], length) == 0
        assert w.fork(0, 1) == -1 and b"every committed position" in kv.kv_last_error()
        assert w.used() == 1 and w.pages(1) == [] and kv.kv_state_length(w.states[1]) == 0
        assert w.owners(w.pages(0)[0]) == 1
    assert kv.kv_state_commit(w.states[0], 3) == 0
    assert w.fork(0, 1) == [(w.pages(0)[0], w.pages(1)[0])]
    w.close()


def test_own_pages_are_filled_before_they_take_the_shared_ones_places(filled):
    w = World(filled, pages=12)
    w.grow(0, 16)
    w.fork(0, 1)
    shared = w.pages(0)
    assert filled.kv_state_commit(w.states[1], 5) == 0
    out, then = (ctypes.c_int * 8)(), (ctypes.c_int * 8)()
    rows = filled.kv_sink_count(w.states[1])
    assert filled.kv_state_unshare_filled(w.states[1], 9, 1, out, then, 8) == -1  # the copy fails
    assert b"the copy failed" in filled.kv_last_error() and filled.kv_sink_count(w.states[1]) == rows
    assert w.pages(1) == shared and [w.owners(p) for p in shared] == [2] * 4 and w.used() == 4
    assert filled.kv_state_unshare_filled(w.states[1], 9, 0, out, then, 8) == 2
    mine = w.pages(1)
    assert list(then[:4]) == shared  # while the copy ran
    assert [(out[2 * i], out[2 * i + 1]) for i in range(2)] == list(zip(shared[1:3], mine[1:3]))
    assert mine[0] == shared[0] and mine[3] == shared[3] and [w.owners(p) for p in shared] == [2, 1, 1, 2]
    w.close()
