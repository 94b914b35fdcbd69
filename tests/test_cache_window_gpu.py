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
