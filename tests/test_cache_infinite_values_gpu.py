"""Infinite values that queries of the window attention see come out as the softmax weight in 32
bits makes them (an infinity, or NaN where infinities of both signs meet), by every kernel, and
leave the finite results right."""

import pytest
import torch

from test_cache_attention_gpu import BF16, F16, Case

pytestmark = pytest.mark.gpu

INF = float("inf")
SHAPES = [
    ("decode", (F16, 8, 2, 128, 16, [1, 1], [300, 41], 200, 4), None),
    ("decode bf16", (BF16, 4, 2, 64, 16, [1], [260], 1 << 20, 0), None),
    ("decode short heads", (F16, 2, 2, 16, 16, [1], [260], 1 << 20, 0), None),
    ("decode splits", (F16, 2, 1, 128, 64, [1], [20000], 16384, 64), None),
    ("few rows", (F16, 4, 2, 64, 16, [3], [290], 200, 2), None),
    ("few rows bf16", (BF16, 2, 1, 128, 8, [5], [290], 1 << 20, 0), None),
    ("boxes", (F16, 4, 2, 64, 16, [200], [150], 1 << 20, 0), 1 << 20),
    ("boxes bf16", (BF16, 2, 1, 128, 16, [150], [150], 250, 0), 1 << 20),
    ("copies", (F16, 2, 1, 128, 7, [150], [150], 1 << 20, 0), 1 << 20),
    ("prompt splits", (F16, 2, 1, 64, 64, [40], [900], 1 << 20, 0), None),
    ("short heads", (F16, 2, 1, 32, 16, [150], [150], 1 << 20, 0), 1 << 20),
    ("short heads bf16", (BF16, 2, 2, 16, 16, [150], [150], 200, 1), 1 << 20),
]


@pytest.mark.parametrize("low", [False, True], ids=["any weight", "a low weight"])
@pytest.mark.parametrize("over", [False, True], ids=["apart", "over the queries"])
@pytest.mark.parametrize("args,max_rows", [s[1:] for s in SHAPES], ids=[s[0] for s in SHAPES])
def test_infinite_values(rt, args, max_rows, over, low):
    if over and max_rows is None and args[5][0] > 16:
        pytest.skip("its results pass through the workspace")
    c = Case(*args, poison=False)
    n = len(c.rows)
    bad = 230  # the first sequence's position (of the splits' case: one of its window)
    if c.first[0] > 1000:
        bad = 19000
    elif c.first[0] > 800:
        bad = 870
    page = int(c.table[n - 1, bad // c.page])
    c.v[page, :, bad % c.page, 1] = INF
    c.v[page, :, bad % c.page, 3] = -INF
    c.v[page, :, bad % c.page, 5] = INF
    c.v[page, :, bad % c.page, c.d - 1] = INF
    other = int(c.table[n - 1, (bad - 9) // c.page])
    c.v[other, :, (bad - 9) % c.page, 5] = -INF
    if low:  # a weight of some e^-20 / keys: 0 in fp16, a normal number in fp32 and bf16
        c.q.fill_(1.0)
        c.k.mul_(0.01)
        c.k[page, :, bad % c.page] = -20.0 / c.d ** 0.5
    want, tol = c.exact()
    assert not torch.isfinite(want[:c.starts[1]]).all() and torch.isfinite(want[c.starts[1]:]).all()
    if over:
        want[c.starts[-1]:] = c.q[c.starts[-1]:].double()
        out = c.run(rt, out=c.q, max_rows=max_rows)
    else:
        out = c.run(rt, max_rows=max_rows)
    torch.cuda.synchronize()
    rt.synchronize()
    out = out.double()
    finite = torch.isfinite(want)
    assert ((out - want).abs() <= tol)[finite].all()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[out.isinf()], want[want.isinf()]) and torch.equal(out.isinf(), want.isinf())
