"""Page copies and cache compaction against plain indexing and 64-bit rotations."""

import pytest
import torch

import tmc_cuda

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_pools(layers, pages, hkv, page, d, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pools = [torch.randn((pages, hkv, page, d), generator=g, device="cuda").to(dtype) for _ in range(2 * layers)]
    return pools, torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("layers,pages,hkv,page,d,pairs", [
    (1, 2, 1, 1, 8, [(0, 1)]),
    (2, 9, 3, 5, 8, [(1, 0), (1, 2), (8, 7)]),
    (3, 40, 8, 16, 128, [(i % 20, 20 + i) for i in range(20)]),
    (32, 6, 2, 128, 64, [(5, 0), (4, 1)]),
    (1, 4, 4, 7, 24, [(3, 3), (2, 1)]),
])
def test_page_copies(rt, layers, pages, hkv, page, d, pairs):
    pools, addresses = make_pools(layers, pages, hkv, page, d, F16)
    want = [p.clone() for p in pools]
    for w in want:
        for s, t in pairs:
            w[t] = w[s]
    tmc_cuda.kv_copy_pages(rt, addresses, 2 * layers, pages, hkv * page * d * 2, i32([s for s, _ in pairs]),
                           i32([t for _, t in pairs]), len(pairs), stream=stream())
    torch.cuda.synchronize()
    rt.synchronize()
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_bad_pages_are_reported_and_skipped(rt):
    pools, addresses = make_pools(2, 8, 2, 16, 64, F16)
    want = [p.clone() for p in pools]
    for w in want:
        w[5] = w[4]
    for bad in ([-1, 0], [8, 0], [0, -3], [0, 9]):
        tmc_cuda.kv_copy_pages(rt, addresses, 4, 8, 2 * 16 * 64 * 2, i32([bad[0], 4]), i32([bad[1], 5]), 2,
                               stream=stream())
        torch.cuda.synchronize()
        with pytest.raises(tmc_cuda.TmcError) as e:
            rt.synchronize()
        assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
        assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_pages_beyond_32_bit_offsets(rt):
    pages, elems = 140000, 8 * 16 * 128  # 4.6 GB a pool
    pool = torch.empty((pages, elems), dtype=F16, device="cuda")
    pool[3].normal_()
    addresses = torch.tensor([pool.data_ptr()], dtype=torch.int64, device="cuda")
    tmc_cuda.kv_copy_pages(rt, addresses, 1, pages, elems * 2, i32([3]), i32([pages - 1]), 1, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(pool[pages - 1], pool[3])


def tables(rows, d, theta=10000.0):
    f = theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float(), a.sin().float()


def compacted(pools, layers, source, target, keep, first, page, cos, sin):
    """(values, tolerances) of every pool in 64 bits."""
    want, tol = [p.double() for p in pools], [torch.zeros_like(p, dtype=torch.float64) for p in pools]
    eps = torch.finfo(pools[0].dtype).eps / 2
    for n in range(2 * layers):
        for i, p in enumerate(keep):
            t = first + i
            row = pools[n][source[p // page], :, p % page].double()
            new, slack = row.clone(), torch.zeros_like(row)
            if n % 2 == 0 and cos is not None and p != t:
                c, s = cos[abs(p - t)].double(), sin[abs(p - t)].double() * (1 if p > t else -1)
                a, b = row[:, 0::2], row[:, 1::2]
                new[:, 0::2], new[:, 1::2] = a * c + b * s, b * c - a * s
                # two fp32 roundings of products no larger than |a| + |b|, then one to storage
                size = (a.abs() + b.abs()) * 2.0 ** -23
                slack = eps * new.abs() * 1.001 + torch.finfo(pools[0].dtype).tiny * eps
                slack[:, 0::2] += size
                slack[:, 1::2] += size
            want[n][target[t // page], :, t % page] = new
            tol[n][target[t // page], :, t % page] = slack
    return want, tol


@pytest.mark.parametrize("dtype,layers,hkv,d,page,length,first,keep", [
    (F16, 1, 1, 8, 1, 4, 0, [3]),
    (F16, 2, 2, 64, 16, 100, 0, list(range(40, 100))),
    (BF16, 2, 8, 128, 16, 200, 4, list(range(120, 200))),
    (F16, 3, 3, 24, 7, 90, 5, [5, 6, 8, 9, 30, 31, 55, 89]),
    (BF16, 1, 4, 32, 24, 60, 0, [0, 1, 2, 3, 50, 58, 59]),
    (F16, 1, 2, 64, 16, 64, 40, [3, 9, 41, 63]),  # rows that move to later positions
    (F16, 2, 16, 16, 5, 33, 0, list(range(0, 33, 2))),
])
@pytest.mark.parametrize("turned", [True, False])
def test_compaction(rt, dtype, layers, hkv, d, page, length, first, keep, turned):
    old, new = -(-length // page), -(-(first + len(keep)) // page)
    pools, addresses = make_pools(layers, old + new + 1, hkv, page, d, dtype, seed=length)
    order = torch.randperm(old + new + 1).tolist()
    source, target = order[:old], order[old:old + new]
    cos, sin = tables(length, d) if turned else (None, None)
    want, tol = compacted(pools, layers, source, target, keep, first, page, cos, sin)
    tmc_cuda.kv_compact(rt, addresses, layers, old + new + 1, hkv, d, page, i32(source), old, i32(target), new, i32(keep),
                        len(keep), first, cos, sin, length, dtype=tmc_cuda.F16 if dtype == F16 else tmc_cuda.BF16,
                        stream=stream())
    torch.cuda.synchronize()
    rt.synchronize()
    for p, w, t in zip(pools, want, tol):
        assert ((p.double() - w).abs() <= t).all()


def test_compaction_reports_bad_rows(rt):
    pools, addresses = make_pools(1, 9, 2, 16, 64, F16)
    cos, sin = tables(30, 64)
    before = [p.clone() for p in pools]
    # outside the source pages, a missing page, a page beyond the pool, a distance beyond the tables
    for source, keep in (([0, 1], [32]), ([0, 1], [-1]), ([0, -1], [20]), ([0, 9], [20]), ([0, 1, 2, 3], [50])):
        tmc_cuda.kv_compact(rt, addresses, 1, 9, 2, 64, 16, i32(source), len(source), i32([5]), 1, i32(keep), 1, 0, cos,
                            sin, 30, stream=stream())
        torch.cuda.synchronize()
        with pytest.raises(tmc_cuda.TmcError) as e:
            rt.synchronize()
        assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
        assert all(torch.equal(p, b) for p, b in zip(pools, before))


def test_captured_replays_follow_their_inputs(rt):
    pools, addresses = make_pools(2, 12, 2, 16, 64, F16)
    cos, sin = tables(64, 64)
    keep, src, dst = i32(list(range(20, 60))), i32([0]), i32([11])
    compact = lambda: tmc_cuda.kv_compact(rt, addresses, 2, 12, 2, 64, 16, i32_source, 4, i32_target, 3, keep, 40, 0,  # noqa: E731
                                          cos, sin, 64, stream=stream())
    copy = lambda: tmc_cuda.kv_copy_pages(rt, addresses, 4, 12, 2 * 16 * 64 * 2, src, dst, 1, stream=stream())  # noqa: E731
    i32_source, i32_target = i32([3, 1, 2, 0]), i32([7, 8, 5])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        compact()
        copy()
    keep.copy_(i32(list(range(4, 44))))
    src.copy_(i32([8]))  # a page that the compaction has just filled
    source, target = [3, 1, 2, 0], [7, 8, 5]
    want, tol = compacted(pools, 2, source, target, list(range(4, 44)), 0, 16, cos, sin)
    graph.replay()
    torch.cuda.synchronize()
    for p, w, t in zip(pools, want, tol):
        w[11], t[11] = w[8], t[8]
        assert ((p.double() - w).abs() <= t).all()
