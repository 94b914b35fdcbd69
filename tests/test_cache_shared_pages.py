"""What several sequences share stays as it is, whatever lengths are set by hand: the KV
cache state on the CPU (through tests/kv_fork_shim.cpp)."""

from test_cache_fork import World, kv  # noqa: F401


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
