"""NaN and infinite values where the documentation says what becomes of them: ranks of masked and
NaN logits, against a stable sort."""

import pytest
import torch

from test_cache_logprobs_gpu import BF16, F16, F32, call

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,offset,rows", [(1, 0, 2), (5, 1, 6), (300, 0, 6), (9001, 3, 6), (70001, 5, 6), (5001, 0, 300)])
@pytest.mark.parametrize("top", [0, 5])
def test_nan_ranks_as_minus_infinity(rt, dtype, vocab, offset, rows, top):
    top = min(top, vocab)
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab)
    x = torch.empty((rows * vocab + offset,), dtype=dtype, device="cuda")[offset:].view(rows, vocab)
    x.copy_(torch.randn((rows, vocab), generator=g, device="cuda"))
    kind = torch.randint(0, 6, (rows, vocab), generator=g, device="cuda")
    x[kind == 0] = NAN
    x[kind == 1] = -INF
    if rows > 5:
        x[3] = NAN
        x[4] = torch.where(kind[4] < 3, NAN, -INF)
        x[5] = -INF
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    # targets at NaN, at -inf (somewhere, and the row's last one), at anything
    for r in range(min(rows, 100)):
        of = [x[r].isnan(), x[r] == -INF, x[r] == x[r], x[r].isnan() | (x[r] == -INF)][r % 4]
        at = of.nonzero()[:, 0]
        if len(at):
            t[r] = at[len(at) // 2 if r % 8 < 4 else -1]
    out = call(rt, x, t, vocab, top)
    torch.cuda.synchronize()
    rt.synchronize()
    order = torch.sort(torch.where(x.isnan(), -INF, x.double()), dim=1, descending=True, stable=True)[1]
    place = (order == t.long()[:, None]).int().argmax(1)
    assert torch.equal(out["ranks"].long(), place)
    assert torch.equal(out["ids"].long(), order[:, :top])
    assert torch.equal(out["logprobs"].isnan(), x.isnan().any(1))
