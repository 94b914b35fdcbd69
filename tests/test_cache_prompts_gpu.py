"""Window attention by the prompt kernels at sizes that would run as decoding does otherwise (max_rows
is only a bound: a large one asks for the prompt kernels), and short prompts beside it."""

import pytest
import torch

import tmc_cuda
from test_cache_attention_gpu import BF16, CASES, F16, Case

pytestmark = pytest.mark.gpu

MANY = 1 << 20
PROMPTS = [c for c in CASES if max(c[1][5]) > 1 or c[0] in ("ragged", "odd pages", "page of one", "sinks beyond the row")]


def loosened(c):
    """Case.exact with P rounded once, as the prompt kernels do for single rows too."""
    want, tol = c.exact()
    if max(c.rows) == 1:
        tol = tol + torch.finfo(c.dtype).eps / 2 * c.v.nan_to_num(0).abs().max().double()
    return want, tol


@pytest.mark.parametrize("args", [c[1] for c in PROMPTS], ids=[c[0] for c in PROMPTS])
def test_against_64_bits(rt, args):
    c = Case(*args)
    before = c.out.clone()
    out = c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    rt.synchronize()
    want, tol = loosened(c)
    assert torch.isfinite(out.float()).all()
    assert ((out.double() - want).abs() <= tol).all()
    assert torch.equal(out[c.starts[-1]:], before[c.starts[-1]:])


@pytest.mark.parametrize("args", [
    (F16, 4, 2, 128, 16, [300], [3000], 1 << 20, 0),   # boxes
    (BF16, 4, 2, 128, 24, [300], [3000], 2500, 5),     # copies
    (F16, 4, 4, 64, 64, [270, 130], [2900, 3100], 1 << 20, 3),
    (BF16, 8, 2, 32, 16, [500], [2000], 1 << 20, 0),   # mma.sync
], ids=["boxes", "copies", "ragged", "short heads"])
@pytest.mark.parametrize("workspace", ["full", None])
def test_splits_meet(rt, args, workspace):
    c = Case(*args)
    out = c.run(rt, workspace=workspace)
    torch.cuda.synchronize()
    rt.synchronize()
    if workspace:
        assert c.keep is not None  # the splits do meet there
    c.check(out)


@pytest.mark.parametrize("way", ["rising", "falling", "saw"])
@pytest.mark.parametrize("args", [
    (F16, 4, 2, 64, 16, [150], [700], 4000, 0),
    (BF16, 4, 2, 128, 24, [150], [700], 600, 3),
    (F16, 2, 1, 128, 16, [3], [3000], 1 << 20, 0),
    (BF16, 2, 2, 32, 16, [90], [700], 4000, 0),
], ids=["boxes", "copies", "few rows", "short heads"])
def test_scores_that_run_away(rt, way, args):
    c = Case(*args, poison=False)
    length = c.first[0] + c.rows[0]
    at = torch.arange(length, device="cuda")
    a = {"rising": at / length * 2 - 1, "falling": 1 - at / length * 2, "saw": (at % 300) / 150 - 1}[way]
    page = c.table[0, at // c.page].long()
    c.k[page, :, at % c.page] = (a[:, None, None] * 300 / c.d ** 0.5 * (1 + 0.01 * torch.randn(
        (length, c.hkv, c.d), device="cuda"))).to(c.dtype)
    c.q.fill_(1.0)
    out = c.run(rt, max_rows=MANY)
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(out)


@pytest.mark.parametrize("max_rows", [None, MANY], ids=["as it comes", "prompt kernels"])
@pytest.mark.parametrize("d,page,rows,first", [(64, 16, 60, 20), (128, 24, 60, 20), (32, 16, 60, 20), (128, 16, 5, 44)])
@pytest.mark.parametrize("special", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_what_a_row_does_not_see_cannot_reach_it(rt, where, special, d, page, rows, first, max_rows):
    c = Case(F16, 4, 2, d, page, [rows], [first], 16, 2, poison=False)
    bad = 45
    number = int(c.table[0, bad // page])
    pool = c.k if where == "keys" else c.v
    pool[number, :, bad % page] = special
    out = c.run(rt, max_rows=max_rows)
    torch.cuda.synchronize()
    seen = torch.tensor([first + r >= bad and first + r - bad < 16 for r in range(rows)], device="cuda")
    pool[number, :, bad % page] = 0
    want, tol = c.exact()
    err = (out.double() - want).abs()[:rows]
    assert (err[~seen] <= tol[:rows][~seen]).all()
    if where == "values":
        assert not torch.isfinite(out[:rows][seen].float()).any()


@pytest.mark.parametrize("max_rows", [None, MANY], ids=["as it comes", "prompt kernels"])
@pytest.mark.parametrize("rows", [[2, 3], [20, 20]])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 12), (16, 16)])
def test_missing_pages_are_reported_and_skipped(rt, d, page, rows, max_rows):
    c = Case(F16, 4, 2, d, page, rows, [64, 64], 40, 0, poison=False)
    # Sequence 1's keys of one page as far below its queries as fp16 goes: their weight is 0.
    mine = slice(rows[0], rows[0] + rows[1])
    c.q[mine] = c.q[mine].abs() + 0.5
    hole = int(c.table[0, 48 // page])
    c.k[hole] = -1000.0
    want = c.run(rt, max_rows=max_rows).clone()
    torch.cuda.synchronize()
    rt.synchronize()
    c.table[0, 48 // page] = -1  # without that page: the same
    c.table[1, :] = -1           # sequence 0 without any: zeros
    out = c.run(rt, max_rows=max_rows)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError) as e:
        rt.synchronize()
    assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
    assert (out[:rows[0]] == 0).all()
    assert torch.equal(out[mine], want[mine])


@pytest.mark.parametrize("args", [
    (F16, 8, 2, 128, 16, [4] * 20, [40 * i for i in range(20)], 300, 4),       # 16 tile rows: one tile
    (BF16, 6, 2, 64, 24, [1, 5, 0, 2], [900, 3, 40, 77], 64, 2),
    (F16, 4, 4, 32, 16, [16, 9], [500, 0], 1 << 20, 0),
    (F16, 8, 1, 128, 16, [6], [3000], 2000, 7),                                  # 48: three tiles, splits meet
    (BF16, 5, 1, 16, 8, [13], [700], 100, 130),                                  # tiles cut between a row's heads
    (F16, 24, 1, 128, 16, [3], [200], 50, 1),                                    # rows over several tiles
], ids=["a tile", "ragged", "one head a key", "three tiles", "cut rows", "wide rows"])
def test_few_rows(rt, args):
    c = Case(*args)
    before = c.out.clone()
    for workspace in ("full", None):
        out = c.run(rt, workspace=workspace)
        torch.cuda.synchronize()
        rt.synchronize()
        c.check(out)
        assert torch.equal(out[c.starts[-1]:], before[c.starts[-1]:])
