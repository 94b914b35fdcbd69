"""Prompts over pages that no TMA box fits (sizes that 8 does not divide), heads of 64 and 128: the
loader by 16-byte copies over many steps, with splits, windows, sinks, missing pages, captures."""

import pytest
import torch

import tmc_cuda
from test_cache_attention_gpu import BF16, F16, Case

pytestmark = pytest.mark.gpu

MANY = 1 << 20  # max_rows is only a bound: a large one asks for the prompt kernels
CASES = [
    ("two steps", (F16, 2, 1, 64, 7, [40], [200], 1 << 20, 0), MANY),
    ("as many steps as stages", (F16, 2, 1, 64, 12, [30], [354], 1 << 20, 0), MANY),
    ("one step more", (F16, 2, 1, 64, 12, [31], [354], 1 << 20, 0), MANY),
    ("stages of 128", (BF16, 2, 1, 128, 7, [40], [216], 1 << 20, 0), MANY),
    ("one step more, 128", (BF16, 2, 1, 128, 7, [41], [216], 1 << 20, 0), MANY),
    ("many steps", (F16, 2, 1, 128, 12, [20], [3000], 1 << 20, 0), MANY),
    ("many steps, two tiles", (BF16, 4, 1, 64, 5, [70], [2100], 1 << 20, 0), MANY),
    ("a causal prompt", (F16, 1, 1, 128, 7, [700], [0], 1 << 20, 0), MANY),
    ("window and sinks", (F16, 4, 2, 128, 20, [300], [900], 300, 37), MANY),
    ("window and sinks, 64", (BF16, 3, 1, 64, 1, [300], [700], 500, 130), MANY),
    ("ragged", (F16, 6, 2, 64, 7, [1, 0, 133, 290], [900, 3, 500, 11], 450, 2), None),
    ("splits", (F16, 4, 2, 64, 12, [300], [3000], 1 << 20, 3), None),
    ("splits, 128", (BF16, 8, 2, 128, 7, [150], [2500], 1500, 5), None),
    ("long pages", (F16, 2, 2, 128, 1001, [260], [900], 1 << 20, 0), MANY),
]


@pytest.mark.parametrize("args,max_rows", [c[1:] for c in CASES], ids=[c[0] for c in CASES])
def test_against_64_bits(rt, args, max_rows):
    c = Case(*args)
    before = c.out.clone()
    out = c.run(rt, max_rows=max_rows)
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(out)
    assert torch.equal(out[c.starts[-1]:], before[c.starts[-1]:])
    again = c.run(rt, max_rows=max_rows, workspace=None, out=torch.full_like(c.out, 7.0))
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(again)


@pytest.mark.parametrize("d,page", [(64, 7), (128, 12)])
def test_missing_pages_of_late_steps_are_skipped(rt, d, page):
    c = Case(F16, 4, 2, d, page, [200], [1500], 1 << 20, 0, poison=False)
    # The keys of some pages as far below the queries as fp16 goes: their weight is 0.
    c.q.copy_(c.q.abs() + 0.5)
    holes = [1, 60, 61, 90, 1400 // page]
    for i in holes:
        c.k[int(c.table[0, i])] = -1000.0
    want = c.run(rt, max_rows=MANY).clone()
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(want)
    for i in holes:
        c.table[0, i] = -1 if i % 2 else c.pool_pages
    out = c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError) as e:
        rt.synchronize()
    assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
    assert torch.equal(out, want)


@pytest.mark.parametrize("special", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", ["keys", "values"])
@pytest.mark.parametrize("d,page", [(64, 12), (128, 7)])
def test_what_a_row_does_not_see_cannot_reach_it(rt, where, special, d, page):
    first, rows, window = 600, 260, 200
    c = Case(F16, 2, 1, d, page, [rows], [first], window, 2, poison=False)
    bad = 610
    number = int(c.table[0, bad // page])
    pool = c.k if where == "keys" else c.v
    pool[number, :, bad % page] = special
    out = c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    rt.synchronize()
    at = torch.arange(first, first + rows, device="cuda")
    seen = (at >= bad) & (at - bad < window)
    pool[number, :, bad % page] = 0
    want, tol = c.exact()
    err = (out.double() - want).abs()[:rows]
    assert (err[~seen] <= tol[:rows][~seen]).all()
    if where == "values":
        assert not torch.isfinite(out[:rows][seen].float()).any()


@pytest.mark.parametrize("way", ["rising", "falling", "saw"])
@pytest.mark.parametrize("d,page", [(64, 7), (128, 20)])
def test_scores_that_run_away(rt, way, d, page):
    c = Case(BF16, 2, 1, d, page, [60], [1500], 1 << 20, 0, poison=False)
    length = c.first[0] + c.rows[0]
    at = torch.arange(length, device="cuda")
    a = {"rising": at / length * 2 - 1, "falling": 1 - at / length * 2, "saw": (at % 300) / 150 - 1}[way]
    number = c.table[0, at // c.page].long()
    c.k[number, :, at % c.page] = (a[:, None, None] * 300 / d ** 0.5 * (1 + 0.01 * torch.randn(
        (length, 1, d), device="cuda"))).to(c.dtype)
    c.q.fill_(1.0)
    out = c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(out)


def test_captured_replays_follow_their_inputs(rt):
    first = [1000, 700]
    c = Case(F16, 2, 1, 128, 7, [130, 260], first, 600, 4, poison=False, capacity=1500)
    c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(rt, max_rows=MANY, stream=torch.cuda.current_stream().cuda_stream)
    moved = [first[0] - 300, first[1] - 1]
    c.d_first.copy_(torch.tensor(moved, dtype=torch.int32))
    c.q.normal_()
    c.out.fill_(7.0)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    c.first = moved
    c.check(c.out)
