"""Shared pages of the decoder under lengths set by hand, against a decoder that shares nothing."""

import numpy as np
import pytest

from test_cache_decoder_gpu import Model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page_size", [4, 16])
@pytest.mark.parametrize("way", ["prefill", "generate", "decode"])
def test_appending_behind_a_lowered_length_leaves_the_other_sequence(rt, page_size, way):
    m = Model(rt, page_size=page_size)
    prompt, more = m.tokens(64), m.tokens(30, seed=9)
    m.dec.prefill(prompt)
    m.dec.fork(0, [1])
    before = [m.dec.read_kv(layer, 0) for layer in range(2)]
    m.dec.commit(1, 17)  # keeps the pages behind, which both sequences hold
    other = m.make()
    other.prefill(prompt[:17], slot=1)

    def go_on(d):
        if way == "prefill":
            return d.prefill(more, slot=1)
        if way == "generate":
            return d.generate([3], 30, slots=[1])[:1]
        return [d.decode([t], slots=[1])[0] for t in more[:20]]

    for got, want in zip(go_on(m.dec), go_on(other)):
        assert np.array_equal(got, want)
    for layer in range(2):
        for x, y in zip(m.dec.read_kv(layer, 0), before[layer]):
            assert np.array_equal(x, y)
        for x, y in zip(m.dec.read_kv(layer, 1), other.read_kv(layer, 1)):
            assert np.array_equal(x, y)


def test_committed_positions_without_pages_cannot_be_forked(rt):
    import tmc_cuda
    m = Model(rt)
    m.dec.stage(0, 20)
    m.dec.commit(0, 100)
    with pytest.raises(tmc_cuda.TmcError, match="every committed position"):
        m.dec.fork(0, [1, 2])
    assert m.dec.pool_stats()["used"] == 2 and m.dec.length(1) == m.dec.length(2) == 0


def test_committed_positions_without_pages_cannot_be_compacted(rt):
    import tmc_cuda
    m = Model(rt)
    m.dec.prefill(m.tokens(20))
    m.dec.commit(0, 100)  # two pages of 16 are there
    for keep in (list(range(40)) + [99], [3, 99], list(range(90))):
        with pytest.raises(tmc_cuda.TmcError, match="missing"):
            m.dec.compact(0, keep)
        assert m.dec.length(0) == 100 and m.dec.pool_stats()["used"] == 2
    m.dec.commit(0, 20)
    m.dec.compact(0, [0, 19])
    assert m.dec.length(0) == 2
