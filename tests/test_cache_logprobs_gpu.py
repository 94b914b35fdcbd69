"""Token log probabilities, entropy, rank and top alternatives against 64 bits."""

import math

import pytest
import torch

import tmc_cuda

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


def call(rt, x, targets, vocab, top, stream=None, rows=None):
    rows = x.shape[0] if rows is None else rows
    f = lambda *s: torch.full(s, 9.0, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, 9, dtype=torch.int32, device="cuda")  # noqa: E731
    out = dict(logprobs=f(rows), entropy=f(rows), ranks=i(rows), ids=i(rows, top), top=f(rows, top))
    tmc_cuda.token_logprobs(rt, x, targets, rows, vocab, out["logprobs"], out["entropy"], out["ranks"], top, out["ids"],
                            out["top"], row_stride=x.stride(0),
                            stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
    return out


def check(out, x, targets, vocab, top):
    """Every row against the definition. The sums of a thread are of at most vocab / 256 + 40
    positive terms in fp32; each term's exponent is off by three roundings of its distance
    to the maximum (whose weighted mean is the entropy at most) and 2^-22 of 2^x."""
    x = x[:, :vocab].double()
    m = x.amax(1, keepdim=True)
    log_p = x - m - (x - m).exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    rel = (vocab / 256 + 40) * 2.0 ** -24 + 3 * (entropy + 1) * 2.0 ** -24 + 2.0 ** -21
    t = targets.long()
    given = (t >= 0)
    rows = torch.arange(x.shape[0], device="cuda")
    want = log_p[rows, t.clamp(min=0)]
    tol = rel + 4 * 2.0 ** -24 * (want.abs() + entropy + 1)
    got = out["logprobs"].double()
    assert (got[~given] == 0).all()
    same = got == want  # infinities
    assert (same | ((got - want).abs() <= tol))[given].all(), (got - want).abs().max()
    ht = rel * (2 + 2 * entropy) + 2.0 ** -22 * (entropy + 1)
    assert ((out["entropy"].double() - entropy).abs() <= ht).all(), (out["entropy"].double() - entropy).abs().max()
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    place = (order == t.clamp(min=0)[:, None]).int().argmax(1)
    assert torch.equal(out["ranks"].long(), torch.where(given, place, -1))
    assert torch.equal(out["ids"].long(), order[:, :top])
    best = log_p.gather(1, order[:, :top])
    diff = (out["top"].double() - best).abs()
    limit = rel[:, None] + 4 * 2.0 ** -24 * (best.abs() + entropy[:, None] + 1)
    assert ((out["top"].double() == best) | (diff <= limit)).all()


CASES = [
    # dtype, rows, vocab, stride, top, offset of the first logit in elements
    (F32, 1, 1, 1, 1, 0), (F32, 3, 2, 2, 2, 0), (F16, 2, 5, 7, 3, 1), (BF16, 4, 40, 41, 32, 0), (F32, 5, 40, 40, 32, 3),
    (F16, 3, 257, 257, 20, 0), (F32, 2, 1000, 1003, 32, 1), (BF16, 9, 4099, 4100, 5, 5), (F16, 1, 8191, 8192, 0, 0),
    (F32, 7, 32000, 32000, 20, 0), (BF16, 300, 5001, 5001, 1, 0), (F32, 1, 128256, 128256, 20, 0),
    (F16, 2, 128256, 128256, 32, 0), (BF16, 1, 200003, 200003, 32, 7), (F32, 700, 1537, 1600, 4, 2),
]


@pytest.mark.parametrize("dtype,rows,vocab,stride,top,offset", CASES)
@pytest.mark.parametrize("std", [0.5, 6.0])
def test_against_64_bits(rt, dtype, rows, vocab, stride, top, offset, std):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows * vocab + top)
    flat = torch.full((rows * stride + offset,), float("nan"), dtype=dtype, device="cuda")
    x = flat[offset:].view(rows, stride)
    x[:, :vocab] = (torch.randn((rows, vocab), generator=g, device="cuda") * std).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    t[::3] = x[::3, :vocab].float().argmax(1).to(torch.int32)
    if rows > 2:
        t[1] = -1
    out = call(rt, x, t, vocab, top)
    torch.cuda.synchronize()
    rt.synchronize()
    check(out, x, t, vocab, top)


def rows_of(kind, vocab, dtype, g):
    x = torch.randn((vocab,), generator=g, device="cuda").to(dtype)
    index = torch.arange(vocab, device="cuda")
    if kind == "equal":
        x = torch.zeros_like(x)
    elif kind == "signed zeros":
        x = torch.where(index % 2 == 0, -0.0, 0.0).to(dtype)
    elif kind == "falling":
        x = (-(index // 7).float() / 100).to(dtype)
    elif kind == "rising":
        x = (index.float() / 100).to(dtype)
    elif kind == "few left":
        x = torch.where(index % (vocab // 3) == 2, x.float(), -INF).to(dtype)
    elif kind == "one left":
        x = torch.where(index == vocab - 1, x.float(), -INF).to(dtype)
    elif kind == "lowest":
        x = torch.where(index % 5 == 0, x.float(), torch.finfo(dtype).min).to(dtype)
    elif kind == "nothing but lowest":
        x = torch.full_like(x, torch.finfo(dtype).min)
    elif kind == "one thread holds the top":
        x = torch.where((index // 8) % 256 == 3, x.float() + 30, x.float()).to(dtype)
    elif kind == "peaked":
        x = torch.where(index == vocab // 2, 60.0, x.float()).to(dtype)
    return x


KINDS = ["equal", "signed zeros", "falling", "rising", "few left", "one left", "lowest", "nothing but lowest",
         "one thread holds the top", "peaked"]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [300, 9001, 70000])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows_of_every_kind(rt, dtype, vocab, top):
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab)
    x = torch.stack([rows_of(k, vocab, dtype, g) for k in KINDS])
    t = torch.randint(0, vocab, (len(KINDS),), generator=g, device="cuda", dtype=torch.int32)
    t[5] = vocab - 1
    out = call(rt, x, t, vocab, top)
    torch.cuda.synchronize()
    rt.synchronize()
    check(out, x, t, vocab, top)


@pytest.mark.parametrize("vocab", [40, 9001, 70000])
def test_rows_without_an_answer(rt, vocab):
    x = torch.randn((4, vocab), device="cuda")
    x[0] = -INF
    x[1, vocab // 2] = float("nan")
    x[2, 3] = INF
    t = torch.tensor([3, 5, 3, 5], dtype=torch.int32, device="cuda")
    out = call(rt, x, t, vocab, 5)
    torch.cuda.synchronize()
    rt.synchronize()
    assert out["logprobs"][0] == -INF and out["entropy"][0] == 0 and out["ranks"][0] == 3
    assert out["ids"][0].tolist() == [0, 1, 2, 3, 4] and (out["top"][0] == -INF).all()
    assert out["logprobs"][1:3].isnan().all() and out["entropy"][1:3].isnan().all()
    assert out["ids"][2, 0] == 3
    order = torch.sort(x[1].nan_to_num(nan=-INF), descending=True, stable=True)[1]
    assert torch.equal(out["ids"][1].long(), order[:5])
    check({k: v[3:] for k, v in out.items()}, x[3:], t[3:], vocab, 5)


def test_targets_out_of_range_are_reported(rt):
    x = torch.randn((4, 500), device="cuda")
    t = torch.tensor([7, 500, -2, -1], dtype=torch.int32, device="cuda")
    out = call(rt, x, t, 500, 2)
    torch.cuda.synchronize()
    with pytest.raises(tmc_cuda.TmcError) as e:
        rt.synchronize()
    assert e.value.code == tmc_cuda.ERR_DEVICE_STATUS
    assert out["logprobs"][1:3].isnan().all() and out["ranks"].tolist()[1:] == [-1, -1, -1]
    assert out["logprobs"][3] == 0
    ok = {k: v[[0, 3]] for k, v in out.items()}
    check(ok, x[[0, 3]], t[[0, 3]], 500, 2)


def test_rows_behind_the_last_are_left(rt):
    x = torch.randn((6, 300), device="cuda")
    t = torch.zeros(6, dtype=torch.int32, device="cuda")
    f = torch.full((6,), 9.0, device="cuda")
    tmc_cuda.token_logprobs(rt, x, t, 4, 300, f, stream=0)
    torch.cuda.synchronize()
    assert (f[4:] == 9.0).all() and (f[:4] < 0).all()


@pytest.mark.parametrize("skip", ["logprobs", "entropy", "ranks"])
def test_results_may_be_left_out(rt, skip):
    x = torch.randn((3, 3000), device="cuda")
    t = torch.tensor([1, 2, 2999], dtype=torch.int32, device="cuda")
    full = call(rt, x, t, 3000, 0)
    part = {k: torch.zeros_like(v) for k, v in full.items()}
    give = {k: (None if k == skip else part[k]) for k in ("logprobs", "entropy", "ranks")}
    tmc_cuda.token_logprobs(rt, x, t, 3, 3000, give["logprobs"], give["entropy"], give["ranks"], stream=0)
    torch.cuda.synchronize()
    for k in ("logprobs", "entropy", "ranks"):
        assert (part[k] == 0).all() if k == skip else torch.equal(part[k], full[k])


def test_captured_replays_follow_their_inputs(rt):
    x = torch.randn((5, 50000), device="cuda")
    t = torch.tensor([1, 2, 3, 49999, -1], dtype=torch.int32, device="cuda")
    call(rt, x, t, 50000, 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(rt, x, t, 50000, 20)
    for _ in range(2):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, t, 50000, 20)


def test_logits_beyond_32_bit_offsets(rt):
    stride = (1 << 31) + 8
    flat = torch.empty((stride + 5000,), dtype=BF16, device="cuda")
    x = flat.as_strided((2, 5000), (stride, 1))
    x.copy_(torch.randn((2, 5000), device="cuda"))
    t = torch.tensor([17, 4999], dtype=torch.int32, device="cuda")
    out = call(rt, x, t, 5000, 3)
    torch.cuda.synchronize()
    check(out, x, t, 5000, 3)


def test_entropy_is_the_mean_of_minus_log_p():
    # the identity the kernel uses: H = log s - u / s with s, u about the maximum
    x = torch.randn(1000, dtype=torch.float64) * 3
    d = x - x.max()
    s, u = d.exp().sum(), (d.exp() * d).sum()
    p = torch.softmax(x, 0)
    assert math.isclose((s.log() - u / s).item(), -(p * p.log()).sum().item(), rel_tol=1e-12)
