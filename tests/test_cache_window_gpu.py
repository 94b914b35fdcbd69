"""Windows of the decoder beside its other calls."""

import numpy as np
import pytest

from test_cache_decoder_gpu import Model

pytestmark = pytest.mark.gpu


def test_kernels_of_any_number_of_rows(rt):
    m = Model(rt)
    off = [m.dec.kernels_per_step(r) for r in (0, 1, 64)]
    m.dec.set_window(48, 4)
    assert [m.dec.kernels_per_step(r) for r in (0, 1, 64)] == off  # these need no second kernel


def test_a_windowed_attentions_bytes_are_those_that_it_reads(rt):
    m = Model(rt)  # 2 KV heads and 8 heads of 64
    prompt = m.tokens(100)
    m.dec.prefill(prompt)
    m.dec.decode([1])
    queries = 2 * 2 * 8 * 64  # Q in, results out
    per_position = 2 * 2 * 2 * 64
    assert m.dec.profile_kernel(1, 1, 2)[1] == 101 * per_position + queries
    for window, sinks, seen in ((20, 3, 23), (200, 3, 101), (99, 1, 100), (100, 30, 101)):
        m.dec.set_window(window, sinks)
        assert m.dec.profile_kernel(1, 1, 2)[1] == seen * per_position + queries


def test_logits_of_a_profile_are_not_scored(rt):
    import tmc_cuda
    m = Model(rt)
    m.dec.prefill(m.tokens(20))
    m.dec.decode([1])
    first = m.dec.token_logprobs(1)["logprobs"]
    m.dec.profile_kernel(1, 1, 2)
    assert m.dec.token_logprobs(1)["logprobs"] == first  # attention leaves the logits
    m.dec.profile_kernel(0, 1, 2)
    m.dec.profile_kernel(5, 1, 2)
    with pytest.raises(tmc_cuda.TmcError, match="last step"):
        m.dec.token_logprobs(1)
    m.dec.decode([2])
    assert m.dec.token_logprobs(1)["ranks"][0] == 0


@pytest.mark.parametrize("window,sinks", [(512, 0), (600, 7), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (32, 8, 2), (128, 4, 4)])
def test_a_window_that_hides_nothing_is_none(rt, window, sinks, head_dim, heads, kv_heads):
    m = Model(rt, heads, kv_heads, head_dim)  # a capacity of 512
    other = m.make()
    other.set_window(window, sinks)
    for x, y in zip(m.dec.prefill(m.tokens(150)), other.prefill(m.tokens(150))):
        assert np.array_equal(x, y)
    for x, y in zip(m.dec.decode([5]), other.decode([5])):
        assert np.array_equal(x, y)
    for layer in range(2):
        for x, y in zip(m.dec.read_kv(layer), other.read_kv(layer)):
            assert np.array_equal(x, y)
