"""Forks, compaction and scores of one tensor-parallel rank's decoder (its share of the KV heads),
against a decoder that holds all heads. Nothing here takes a collective: the caches are filled
from the host, and each rank is a decoder by itself."""

import numpy as np
import pytest

import tmc_cuda
from oracle.decoder_ref import rope_tables

pytestmark = pytest.mark.gpu


def make(rt, rank, world, page_size=16):
    dec = tmc_cuda.Decoder(rt, 512, 8, 512, 1000, 2, 256, kv_heads=4, rope_theta=500000.0, page_size=page_size,
                           max_rows=8, max_slots=3, tp_rank=rank, tp_size=world)
    cos, sin = rope_tables(256, 64, 500000.0)
    dec.load_weight("rope.cosine", cos.numpy())
    dec.load_weight("rope.sine", sin.numpy())
    return dec


@pytest.mark.parametrize("world", [2, 4])
@pytest.mark.parametrize("page_size", [16, 7])
def test_a_ranks_heads_fork_and_compact_as_all_do(rt, world, page_size):
    rng = np.random.default_rng(world)
    keys, values = (rng.standard_normal((2, 4, 100, 64)).astype(np.float16).astype(np.float32) for _ in range(2))
    decoders = [make(rt, 0, 1, page_size)] + [make(rt, r, world, page_size) for r in range(world)]
    local = 4 // world
    for n, dec in enumerate(decoders):
        heads = slice(None) if n == 0 else slice((n - 1) * local, n * local)
        assert dec.local_kv_heads == (4 if n == 0 else local)
        dec.set_window(40, 4)
        dec.restore_kv(0, keys[:, heads], values[:, heads])
        dec.fork(0, [2, 1])
        dec.rollback(2, 50)
        dec.compact(1, list(range(4)) + list(range(60, 100)))
    for layer in range(2):
        for slot in range(3):
            whole = decoders[0].read_kv(layer, slot)
            parts = [d.read_kv(layer, slot) for d in decoders[1:]]
            for x, y in zip(whole, (np.concatenate(p) for p in zip(*parts))):
                assert np.array_equal(x, y)
        assert np.array_equal(decoders[0].read_kv(layer, 0)[0], keys[layer])
    assert len({tuple(d.pool_stats().items()) for d in decoders}) == 1


def test_scores_need_the_whole_vocabulary(rt):
    dec = make(rt, 0, 2)
    with pytest.raises(tmc_cuda.TmcError, match="whole vocabulary"):
        dec.score([1, 2, 3])
    assert dec.length(0) == 0 and dec.pool_stats()["used"] == 0
