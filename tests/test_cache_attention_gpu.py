"""Window attention with sinks against a plain 64-bit implementation."""

import math

import pytest
import torch

import tmc_cuda

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Case:
    """Inputs of one call: pages in a random order, everything a query does not see poisoned."""

    def __init__(self, dtype, hq, hkv, d, page, rows, first, window, sinks, seed=0, pad=0, behind=2, capacity=None,
                 poison=True):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.page = dtype, hq, hkv, d, page
        self.rows, self.first, self.window, self.sinks = rows, first, window, sinks
        n = len(rows)
        lengths = [f + r for f, r in zip(first, rows)]
        self.capacity = capacity or max(max(lengths), 1)
        self.stride = -(-self.capacity // page)
        used = [-(-length // page) if r else 0 for length, r in zip(lengths, rows)]
        self.pool_pages = sum(used) + 2
        order = torch.randperm(self.pool_pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((n, self.stride), -1, dtype=torch.int32, device="cuda")
        at = 0
        for s, u in enumerate(used):
            table[n - 1 - s, :u] = order[at:at + u]
            at += u
        shape = (self.pool_pages, hkv, page, d)
        self.k = torch.randn(shape, generator=g, device="cuda").to(dtype)
        self.v = torch.randn(shape, generator=g, device="cuda").to(dtype)
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        self.starts = starts
        self.total = starts[-1] + behind
        self.width = hq * d + pad
        self.q = torch.randn((self.total, self.width), generator=g, device="cuda").to(dtype)
        self.out = torch.full((self.total, self.width), 7.0, dtype=dtype, device="cuda")
        self.table = table
        if poison:
            self._poison(lengths, used)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.d_starts, self.d_first, self.d_rows = i32(starts), i32(first), i32(list(range(n))[::-1])

    def _poison(self, lengths, used):
        """NaN wherever no query of the sequence looks, and no page at all where a whole page is unseen."""
        n = len(self.rows)
        for s, (length, r) in enumerate(zip(lengths, self.rows)):
            if r == 0:
                continue
            low = max(0, self.first[s] - self.window + 1)
            j = torch.arange(used[s] * self.page, device="cuda")
            seen = ((j >= low) | (j < self.sinks)) & (j < length)
            ids = self.table[n - 1 - s, :used[s]].long()
            hide = ~seen.view(used[s], self.page)
            for pool in (self.k, self.v):
                pages = pool[ids]
                pages.masked_fill_(hide[:, None, :, None], float("nan"))
                pool[ids] = pages
            unseen = hide.all(1)
            self.table[n - 1 - s, :used[s]] = torch.where(unseen, -1, self.table[n - 1 - s, :used[s]])
        free = torch.ones(self.pool_pages, dtype=torch.bool, device="cuda")
        free[self.table[self.table >= 0].long()] = False
        self.k[free] = float("nan")
        self.v[free] = float("nan")

    def run(self, rt, workspace="full", stream=None, out=None, max_rows=None, scale=0.0):
        out = self.out if out is None else out
        if max_rows is None:
            max_rows = max(1, max(self.rows))
        need = tmc_cuda.window_attention_workspace_bytes(len(self.rows), max_rows, self.hq, self.hkv, self.d, self.window,
                                                         self.sinks)
        ws = None
        if workspace == "full" and need:
            ws = torch.full((need // 4 + 4,), float("nan"), device="cuda")
        elif workspace == "half" and need:
            ws = torch.full((need // 8 + 4,), float("nan"), device="cuda")
        tmc_cuda.window_attention(rt, self.q, out, self.k, self.v, self.table, self.stride, self.d_rows, self.d_starts,
                                  self.d_first, len(self.rows), self.total, max_rows, self.hq, self.hkv, self.d,
                                  self.page, self.pool_pages, self.capacity, self.window, self.sinks, scale=scale,
                                  q_stride=self.width, out_stride=self.width, workspace=ws,
                                  stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
        self.keep = ws
        return out

    def exact(self, scale=None):
        """(values, tolerance) in 64 bits, laid out as out."""
        scale = scale or 1.0 / math.sqrt(self.d)
        want = self.out.double().clone()
        tol = torch.zeros_like(want)
        n, g = len(self.rows), self.hq // self.hkv
        eps = torch.finfo(self.dtype).eps / 2  # a rounding's relative error
        prompt = max(self.rows) > 1
        for s in range(n):
            for r in range(self.rows[s]):
                p = self.first[s] + r
                j = [x for x in range(p + 1) if p - x < self.window or x < self.sinks]
                jt = torch.tensor(j, device="cuda")
                page = self.table[n - 1 - s, jt // self.page].long()
                assert (page >= 0).all()
                for h in range(self.hkv):
                    k = self.k[page, h, jt % self.page].double()
                    v = self.v[page, h, jt % self.page].double()
                    lo = h * g * self.d
                    q = self.q[self.starts[s] + r, lo:lo + g * self.d].double().view(g, self.d)
                    sc = q @ k.T * scale
                    w = torch.softmax(sc, -1)
                    o = w @ v
                    # A dot product of d terms in fp32 is off by at most d 2^-24 sum |q k| (and its
                    # scaling, the maximum's subtraction and 2^x by a few roundings of numbers of that
                    # size); a weight's relative error is that much, and the normalised sum's twice it.
                    score = (q.abs() @ k.abs().T * scale).max() * (self.d + 8) * 2.0 ** -24 + 2.0 ** -20
                    spread = w @ v.abs()
                    # P: two parts (decode) leave eps^2 each, one part (prompts) eps; values below the
                    # storage type's normal range are off by half its smallest step.
                    part = eps if prompt else eps * eps
                    tiny = torch.finfo(self.dtype).tiny * eps
                    bound = eps * o.abs() * 1.01 + (part + 2 * score) * spread + tiny * (1 + v.abs().sum(0))
                    row = self.starts[s] + r
                    want[row, lo:lo + g * self.d] = o.reshape(-1)
                    tol[row, lo:lo + g * self.d] = bound.reshape(-1)
        return want, tol

    def check(self, out, scale=None):
        want, tol = self.exact(scale)
        err = (out.double() - want).abs()
        worst = (err - tol).max().item()
        assert torch.isfinite(out.float()).all()
        assert worst <= 0, (worst, err.max().item())


CASES = [
    # decode: one row per sequence
    ("one key", (F16, 4, 2, 128, 16, [1], [0], 1, 0)),
    ("window of one", (F16, 4, 2, 64, 16, [1, 1], [5, 40], 1, 0)),
    ("window of one, sinks", (BF16, 4, 2, 64, 16, [1, 1], [0, 40], 1, 3)),
    ("ragged", (F16, 8, 2, 128, 16, [1, 1, 1, 1], [0, 17, 255, 700], 200, 4)),
    ("ragged bf16", (BF16, 8, 2, 128, 16, [1, 1, 1], [3, 300, 911], 256, 5)),
    ("empty sequences", (F16, 4, 4, 64, 8, [0, 1, 0, 1], [0, 100, 7, 30], 64, 2)),
    ("odd pages", (F16, 6, 2, 32, 5, [1, 1], [99, 203], 64, 7)),
    ("page of one", (BF16, 2, 1, 16, 1, [1], [77], 50, 3)),
    ("sinks beyond the window", (F16, 2, 2, 64, 16, [1], [200], 16, 130)),
    ("sinks beyond the row", (F16, 2, 2, 64, 16, [1], [20], 4, 1000)),
    ("no window", (F16, 8, 8, 128, 16, [1], [500], 2 ** 31 - 1, 0)),
    ("17 heads a key", (F16, 17, 1, 64, 16, [1], [130], 100, 1)),
    ("32 heads a key", (BF16, 32, 1, 128, 16, [1], [333], 300, 0)),
    ("splits meet in the workspace", (F16, 2, 1, 128, 64, [1], [20000], 16384, 64)),
    # prompts
    ("short prompt", (F16, 4, 2, 128, 16, [3], [0], 100, 0)),
    ("one row, more allowed", (F16, 4, 2, 64, 16, [1, 2], [9, 70], 33, 1)),
    ("chunk", (F16, 8, 2, 128, 16, [70], [130], 64, 4)),
    ("chunk bf16", (BF16, 8, 8, 64, 24, [65], [200], 100, 17)),
    ("ragged prompts", (F16, 6, 2, 64, 16, [1, 0, 33, 129], [400, 3, 0, 11], 48, 2)),
    ("window of one prompt", (BF16, 2, 2, 32, 16, [40], [7], 1, 0)),
    ("window of one prompt, sinks", (F16, 2, 2, 32, 16, [40], [7], 1, 2)),
    ("three heads a key", (F16, 3, 1, 128, 7, [90], [41], 77, 9)),
    ("short heads", (BF16, 4, 1, 16, 16, [50], [0], 20, 1)),
    ("all keys", (F16, 4, 4, 128, 32, [140], [0], 1 << 20, 0)),
    ("prompt splits meet in the workspace", (F16, 2, 1, 64, 64, [5], [6000], 5000, 3)),
]


@pytest.mark.parametrize("args", [c[1] for c in CASES], ids=[c[0] for c in CASES])
def test_against_64_bits(rt, args):
    c = Case(*args)
    before = c.out.clone()
    out = c.run(rt)
    rt.synchronize()
    torch.cuda.synchronize()
    c.check(out)
    assert torch.equal(out[c.starts[-1]:], before[c.starts[-1]:])  # rows behind the last sequence


@pytest.mark.parametrize("rows,first", [([1], [300]), ([40], [300])])
def test_row_strides_and_scale(rt, rows, first):
    c = Case(F16, 4, 2, 64, 16, rows, first, 128, 4, pad=24)
    before = c.out.clone()
    out = c.run(rt, scale=0.31)
    torch.cuda.synchronize()
    c.check(out, 0.31)
    assert torch.equal(out[:, 4 * 64:], before[:, 4 * 64:])  # between the rows


@pytest.mark.parametrize("args", [(F16, 2, 1, 128, 64, [1], [20000], 16384, 64), (F16, 2, 1, 64, 64, [5], [6000], 5000, 3)])
def test_any_workspace_will_do(rt, args):
    c = Case(*args)
    for workspace in ("full", "half", None):
        out = c.run(rt, workspace=workspace, out=torch.full_like(c.out, 7.0))
        torch.cuda.synchronize()
        c.check(out)


def test_one_row_by_either_kernel(rt):
    # max_rows is only a bound: the prompt kernel answers single rows too.
    c = Case(BF16, 8, 2, 128, 16, [1, 1, 1], [3, 300, 911], 256, 5)
    out = c.run(rt, max_rows=9)
    torch.cuda.synchronize()
    c.rows = [1, 1, 1]
    want, tol = c.exact()
    eps = torch.finfo(BF16).eps / 2
    err = (out.double() - want).abs()
    # one part of P: eps of the weighted |v|, which is at most the largest |v|
    assert (err <= tol + eps * c.v.nan_to_num(0).abs().max().double()).all()


@pytest.mark.parametrize("special", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_what_a_row_does_not_see_cannot_reach_it(rt, where, special):
    # One position holds infinities or NaN: rows before it and rows whose window
    # has passed it stay finite and right, in the same tile as rows that see it.
    c = Case(F16, 4, 2, 64, 16, [60], [20], 16, 2, poison=False)
    bad = 45
    page = int(c.table[0, bad // 16])
    pool = c.k if where == "keys" else c.v
    pool[page, :, bad % 16] = special
    out = c.run(rt)
    torch.cuda.synchronize()
    seen = torch.tensor([20 + r >= bad and 20 + r - bad < 16 for r in range(60)], device="cuda")
    clean = pool.clone()
    clean[page, :, bad % 16] = 0
    if where == "keys":
        c.k = clean
    else:
        c.v = clean
    want, tol = c.exact()
    err = (out.double() - want).abs()[:60]
    assert (err[~seen] <= tol[:60][~seen]).all()
    if where == "values":
        assert not torch.isfinite(out[:60][seen].float()).any()


@pytest.mark.parametrize("rows", [[1, 1], [20, 20]])
def test_missing_pages_are_reported_and_skipped(rt, rows):
    c = Case(F16, 4, 2, 64, 16, rows, [64, 64], 40, 0, poison=False)
    good = c.run(rt).clone()
    torch.cuda.synchronize()
    rt.synchronize()
    c.table[1, :] = -1  # sequence 0 has no page at all
    out = c.run(rt)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError) as e:
        rt.synchronize()
    assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
    assert (out[:rows[0], :] == 0).all()
    assert torch.equal(out[rows[0]:], good[rows[0]:])
    c.table[1, :] = c.pool_pages
    c.run(rt)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError):
        rt.synchronize()


@pytest.mark.parametrize("change", [
    ("d_starts", [-1, 2, 4]), ("d_starts", [0, 7, 4]), ("d_starts", [3, 2, 4]), ("d_first", [-1, 64]),
    ("d_first", [79, 64]), ("d_rows", [-1, 0])])
def test_bad_sequences_are_reported_and_left_out(rt, change):
    c = Case(F16, 4, 2, 64, 16, [2, 2], [64, 64], 40, 0, poison=False, capacity=80, behind=0)
    want = c.run(rt).clone()
    rt.synchronize()
    setattr(c, change[0], torch.tensor(change[1], dtype=torch.int32, device="cuda"))
    out = c.run(rt, out=torch.full_like(c.out, 7.0), max_rows=2)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError) as e:
        rt.synchronize()
    assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
    assert (out[0] == 7.0).all()
    if change[1] == [-1, 2, 4] or change[0] != "d_starts":
        assert torch.equal(out[2:], want[2:])  # the other sequence is answered


@pytest.mark.parametrize("rows", [[1, 1, 1], [17, 1, 30]])
def test_captured_replays_follow_their_inputs(rt, rows):
    first = [200, 90, 333]
    c = Case(F16, 8, 2, 128, 16, rows, first, 96, 4, poison=False, capacity=400)
    c.run(rt)  # sets the kernels up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(rt, stream=torch.cuda.current_stream().cuda_stream)
    moved = [first[0] - 30, first[1], first[2] - 1]
    c.d_first.copy_(torch.tensor(moved, dtype=torch.int32))
    c.q.normal_()
    c.out.fill_(7.0)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    c.first = moved
    c.check(c.out)


def test_two_streams_at_once(rt):
    cases = [Case(F16, 2, 1, 128, 64, [1], [12000 + 64 * i], 8192, 8, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                c.run(rt)
    torch.cuda.synchronize()
    for c in cases:
        c.check(c.out)


def test_pool_beyond_32_bit_offsets(rt):
    hkv, page, d = 8, 16, 128
    pages = (1 << 32) // (hkv * page * d) + 8  # 2^32 elements and more
    c = Case(F16, 8, hkv, d, page, [1, 20], [100, 100], 64, 2, poison=False)
    k = torch.empty((pages, hkv, page, d), dtype=F16, device="cuda")
    v = torch.empty((pages, hkv, page, d), dtype=F16, device="cuda")
    ids = c.table[c.table >= 0].long()
    far = torch.arange(pages - len(ids), pages, device="cuda")
    k[far], v[far] = c.k[ids], c.v[ids]
    moved = c.table.clone()
    moved[c.table >= 0] = far.to(torch.int32)
    c.k, c.v, c.table, c.pool_pages = k, v, moved, pages
    out = c.run(rt)
    torch.cuda.synchronize()
    c.check(out)
