"""Serving-cache kernels as their documentation allows them to be called: scores that run away,
results over the queries, the package's own buffers, calls side by side, shared workspaces, long
lists. Checked by the same 64-bit definitions as the other tests."""

import numpy as np
import pytest
import torch

import tmc_cuda
from test_cache_attention_gpu import BF16, F16, Case
from test_cache_logprobs_gpu import call, check
from test_cache_ops_gpu import compacted, i32, make_pools, stream, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("way", ["rising", "falling", "saw"])
@pytest.mark.parametrize("args", [
    (F16, 4, 2, 128, 16, [1], [900], 4000, 0),
    (F16, 4, 2, 64, 16, [150], [700], 4000, 0),
    (BF16, 4, 2, 128, 24, [150], [700], 600, 3),
    (F16, 2, 1, 128, 16, [3], [5000], 1 << 20, 0),
    (BF16, 2, 2, 32, 16, [90], [700], 4000, 0),
], ids=["decode", "boxes", "copies", "splits", "short heads"])
def test_scores_that_run_away(rt, way, args):
    # Scores of about -300 .. 300: the running maximum of every row moves far, over and over or never.
    c = Case(*args, poison=False)
    lengths = [f + r for f, r in zip(c.first, c.rows)]
    n = len(c.rows)
    for s, length in enumerate(lengths):
        at = torch.arange(length, device="cuda")
        a = {"rising": at / length * 2 - 1, "falling": 1 - at / length * 2, "saw": (at % 300) / 150 - 1}[way]
        page = c.table[n - 1 - s, at // c.page].long()
        c.k[page, :, at % c.page] = (a[:, None, None] * 300 / c.d ** 0.5 * (1 + 0.01 * torch.randn(
            (length, c.hkv, c.d), device="cuda"))).to(c.dtype)
    c.q.fill_(1.0)
    out = c.run(rt)
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(out)


@pytest.mark.parametrize("args", [
    (F16, 8, 2, 128, 16, [1, 1], [300, 41], 200, 4),
    (F16, 2, 1, 128, 64, [1], [20000], 16384, 64),
    (F16, 8, 2, 128, 16, [70, 200], [130, 9], 64, 4),
    (BF16, 2, 1, 64, 24, [5], [6000], 5000, 3),
    (F16, 4, 1, 16, 16, [50], [0], 20, 1),
])
def test_results_over_the_queries(rt, args):
    c = Case(*args)
    want, tol = c.exact()
    want[c.starts[-1]:] = c.q[c.starts[-1]:].double()
    c.run(rt, out=c.q)
    torch.cuda.synchronize()
    assert ((c.q.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("args,max_rows", [
    ((F16, 4, 2, 64, 512, [1, 1], [100, 20], 50, 1), None),       # pages longer than the context
    ((F16, 4, 2, 64, 512, [40, 3], [100, 20], 50, 1), None),
    ((BF16, 4, 2, 128, 16, [33, 1, 7], [100, 20, 0], 64, 2), 700),  # more rows allowed than any sequence has
    ((F16, 2, 1, 16, 4, [1] * 1500, [i % 37 for i in range(1500)], 20, 2), None),
    ((F16, 2, 2, 64, 16, [1, 2] * 200, [i % 50 for i in range(400)], 20, 2), None),
], ids=["long pages", "long pages, prompt", "more rows allowed", "many rows", "many prompts"])
def test_other_shapes(rt, args, max_rows):
    c = Case(*args)
    out = c.run(rt, max_rows=max_rows)
    torch.cuda.synchronize()
    rt.synchronize()
    c.check(out)


def test_two_graphs_share_a_workspace(rt):
    cases = [Case(F16, 2, 1, 128, 64, rows, [12000], 8192, 8, seed=i) for i, rows in enumerate([[1], [6]])]
    need = [tmc_cuda.window_attention_workspace_bytes(1, c.rows[0], 2, 1, 128, 8192, 8) for c in cases]
    assert all(need)
    ws = torch.full((max(need) // 4,), float("nan"), device="cuda")
    graphs = []
    for c in cases:
        run = lambda: tmc_cuda.window_attention(  # noqa: E731
            rt, c.q, c.out, c.k, c.v, c.table, c.stride, c.d_rows, c.d_starts, c.d_first, 1, c.total, c.rows[0], 2, 1, 128,
            64, c.pool_pages, c.capacity, 8192, 8, workspace=ws, stream=torch.cuda.current_stream().cuda_stream)
        run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run()
    for _ in range(3):
        for c, g in zip(cases, graphs):
            c.out.fill_(7.0)
            g.replay()
    torch.cuda.synchronize()
    for c in cases:
        c.check(c.out)


def test_scores_and_copies_side_by_side(rt):
    streams = [torch.cuda.Stream() for _ in range(3)]
    x = [torch.randn((3, 60000), device="cuda") for _ in streams]
    t = [i32([i, 59999, -1]) for i in range(3)]
    pools, addresses = make_pools(2, 60, 2, 16, 64, F16)
    cos, sin = tables(400, 64)
    keep = list(range(3, 100, 2))
    source, target = list(range(7)), list(range(20, 24))
    want, tol = compacted(pools, 2, source, target, keep, 0, 16, cos, sin)
    for w in want:
        w[30], w[31] = w[10], w[10]  # one source, two targets
    d_source, d_target, d_keep, src, dst = i32(source), i32(target), i32(keep), i32([10, 10]), i32([30, 31])
    torch.cuda.synchronize()
    out = [None] * 3
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i] = call(rt, x[i], t[i], 60000, 32)
        with torch.cuda.stream(streams[0]):
            tmc_cuda.kv_compact(rt, addresses, 2, 60, 2, 64, 16, d_source, 7, d_target, 4, d_keep, len(keep), 0, cos, sin,
                                400, stream=stream())
        with torch.cuda.stream(streams[1]):
            tmc_cuda.kv_copy_pages(rt, addresses, 4, 60, 2 * 16 * 64 * 2, src, dst, 2, stream=stream())
    torch.cuda.synchronize()
    rt.synchronize()
    for i in range(3):
        check(out[i], x[i], t[i], 60000, 32)
    for p, w, e in zip(pools, want, tol):
        assert ((p.double() - w).abs() <= e).all()


@pytest.mark.parametrize("keep", [[9, 9, 2, 9], [40, 3, 17, 2, 39]], ids=["repeated", "in any order"])
def test_compaction_of_any_list(rt, keep):
    pools, addresses = make_pools(2, 9, 3, 7, 24, F16)
    cos, sin = tables(64, 24)
    source, target = [8, 1, 2, 0, 5, 6], [3]
    want, tol = compacted(pools, 2, source, target, keep, 2, 7, cos, sin)
    tmc_cuda.kv_compact(rt, addresses, 2, 9, 3, 24, 7, i32(source), 6, i32(target), 1, i32(keep), len(keep), 2, cos, sin, 64,
                        stream=stream())
    torch.cuda.synchronize()
    rt.synchronize()
    for p, w, e in zip(pools, want, tol):
        assert ((p.double() - w).abs() <= e).all()


def test_many_short_rows(rt):
    rows = 70000
    x = torch.randn((rows, 9), device="cuda").to(BF16)
    t = torch.randint(-1, 9, (rows,), dtype=torch.int32, device="cuda")
    out = call(rt, x, t, 9, 9)
    torch.cuda.synchronize()
    check(out, x, t, 9, 9)


def test_buffers_of_the_package(rt):
    # One row of two heads over seven keys, then its scores, a page copy and a compaction, on the runtime's stream.
    rng = np.random.default_rng(5)
    d, page, n = 16, 4, 7
    buf = lambda a, dtype: tmc_cuda.Buffer(rt, a.size, dtype, a)  # noqa: E731
    ints = lambda v: buf(np.asarray(v, np.int32), tmc_cuda.I32)  # noqa: E731
    half = lambda a: a.astype(np.float16).astype(np.float32)  # noqa: E731
    q = half(rng.standard_normal((1, 2, d), dtype=np.float32))
    k, v = (half(rng.standard_normal((3, 1, page, d), dtype=np.float32)) for _ in range(2))
    bq, bk, bv = (buf(a, tmc_cuda.F16) for a in (q, k, v))
    bo = tmc_cuda.Buffer(rt, 2 * d, tmc_cuda.F16)
    tmc_cuda.window_attention(rt, bq, bo, bk, bv, ints([2, 0]), 2, ints([0]), ints([0, 1]), ints([n - 1]), 1, 1, 1, 2, 1, d,
                              page, 3, 8, 8)
    rt.synchronize()
    keys = np.concatenate([k[2, 0], k[0, 0]])[:n].astype(np.float64)
    values = np.concatenate([v[2, 0], v[0, 0]])[:n].astype(np.float64)
    s = q[0].astype(np.float64) @ keys.T / np.sqrt(d)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    got = bo.read().reshape(2, d)
    # the output's rounding (2^-11 of values below 4) and far smaller errors of the sums
    assert np.abs(got - w @ values).max() <= 4 * 2.0 ** -11

    x = rng.standard_normal((2, 50), dtype=np.float32)
    bx, lp = buf(x, tmc_cuda.F32), tmc_cuda.Buffer(rt, 2, tmc_cuda.F32)
    tmc_cuda.token_logprobs(rt, bx, ints([3, 49]), 2, 50, lp)
    rt.synchronize()
    exact = x.astype(np.float64)
    exact = (exact - np.log(np.exp(exact).sum(1, keepdims=True)))[[0, 1], [3, 49]]
    assert np.abs(lp.read() - exact).max() <= 2.0 ** -20

    addresses = np.asarray([bk.ptr, bv.ptr], np.int64)
    pools = ints(addresses.view(np.int32))
    tmc_cuda.kv_copy_pages(rt, pools, 2, 3, page * d * 2, ints([2]), ints([1]), 1)
    rt.synchronize()
    assert (bk.read().reshape(k.shape)[1] == k[2]).all() and (bv.read().reshape(v.shape)[1] == v[2]).all()
    tmc_cuda.kv_compact(rt, pools, 1, 3, 1, d, page, ints([2, 0]), 2, ints([1]), 1, ints([6, 0]), 2)
    rt.synchronize()
    after = bk.read().reshape(k.shape)
    assert (after[1, 0, 0] == k[0, 0, 2]).all() and (after[1, 0, 1] == k[2, 0, 0]).all()
