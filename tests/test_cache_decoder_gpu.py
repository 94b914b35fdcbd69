"""Windows, forks, compaction and token scores of the decoder executor, against
the CPU oracle with a windowed attention and against the decoder itself."""

import math

import numpy as np
import pytest
import torch

import oracle.decoder_ref as ref
from oracle.decoder_ref import DecoderOracle, DecoderSpec, random_weights, rope_tables
from test_decoder_gpu import rms_close

pytestmark = pytest.mark.gpu


def windowed(window, sinks):
    """causal_gqa_attention with a window and sinks."""
    def attention(q, k, v, start):
        rows, d = q.shape[2], q.shape[3]
        group = q.shape[1] // k.shape[1]
        kk, vv = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
        scores = torch.matmul(q.float(), kk.float().transpose(-2, -1)) / math.sqrt(d)
        p = torch.arange(start, start + rows).view(rows, 1)
        j = torch.arange(kk.size(2)).view(1, -1)
        hidden = (j > p) | ((p - j >= window) & (j >= sinks))
        return torch.matmul(torch.softmax(scores.masked_fill(hidden, float("-inf")), -1), vv.float())
    return attention


class Model:
    def __init__(self, rt, heads=8, kv_heads=2, head_dim=64, capacity=512, page_size=16, max_rows=64, max_slots=4, seed=3,
                 pool_pages=0):
        import tmc_cuda
        self.spec = DecoderSpec(hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, intermediate=512, vocab=1000,
                                layers=2, capacity=capacity, rope_theta=500000.0)
        self.weights = random_weights(self.spec, seed, std=0.05)
        self.cos, self.sin = rope_tables(capacity, head_dim, 500000.0)
        self.make = lambda: self._decoder(tmc_cuda, rt, page_size, max_rows, max_slots, pool_pages)
        self.dec = self.make()
        self.oracle = DecoderOracle(self.spec, self.weights, self.cos, self.sin)
        self.twin = DecoderOracle(self.spec, self.weights, self.cos, self.sin, summation_order_seed=7)

    def _decoder(self, tmc_cuda, rt, page_size, max_rows, max_slots, pool_pages):
        s = self.spec
        dec = tmc_cuda.Decoder(rt, s.hidden, s.heads, s.intermediate, s.vocab, s.layers, s.capacity,
                               kv_heads=s.kv_heads, rope_theta=s.rope_theta, page_size=page_size, max_rows=max_rows,
                               max_slots=max_slots, pool_pages=pool_pages)
        dec.load_weights(self.weights)
        dec.load_weight("rope.cosine", self.cos.numpy())
        dec.load_weight("rope.sine", self.sin.numpy())
        return dec

    def tokens(self, n, seed=1):
        return np.random.default_rng(seed).integers(0, self.spec.vocab, n).astype(np.int32)

    def step(self, logits):
        return 4.5 * 0.05 * math.sqrt(self.spec.hidden) * 2.0 ** -10 + 2.0 ** -10 * float(np.abs(logits).max())

    def expect(self, got, tokens, what, seq=0):
        """Logits of `tokens` appended to the oracle's sequence, within its noise floor.

        A single row's twin often rounds exactly alike, so the floor is at least what one
        step of fp16 in the normalised hidden state makes of a logit: two correct sums may
        round each of its `hidden` entries (of size 1: a step is 2^-10) to neighbours, which
        moves a logit of weights N(0, 0.05) by 0.05 sqrt(hidden) 2^-10, 4.5 standard
        deviations of that being the largest of some 10^5 logits; and the logit itself is
        rounded, to neighbours 2^-10 of its size apart. rms_close allows three times the
        floor, so a third of the two together is the floor."""
        want, _ = self.oracle.forward(seq, tokens)
        other, _ = self.twin.forward(seq, tokens)
        floor = max(float((want.float() - other.float()).abs().max()), self.step(want.float().numpy()) / 3)
        rms_close(got, want.float().numpy(), what, floor)


@pytest.mark.parametrize("head_dim,heads,kv_heads,page_size", [(64, 8, 2, 16), (128, 4, 4, 24), (32, 8, 2, 0), (64, 3, 1, 5)])
@pytest.mark.parametrize("window,sinks", [(48, 4), (1, 0), (200, 30)])
def test_windowed_decoder_against_the_oracle(rt, monkeypatch, head_dim, heads, kv_heads, page_size, window, sinks):
    if heads * head_dim % 8 != 0:
        pytest.skip("hidden size")
    m = Model(rt, heads, kv_heads, head_dim, page_size=page_size)
    m.dec.set_window(window, sinks)
    monkeypatch.setattr(ref, "causal_gqa_attention", windowed(window, sinks))
    prompt = m.tokens(150)  # chunks of 64, 64 and 22 rows
    got, _ = m.dec.prefill(prompt)
    m.expect(got, prompt, "prompt")
    for i, t in enumerate(m.tokens(5, seed=2)):
        got, _ = m.dec.decode([t])
        m.expect(got, [t], f"step {i}")


def test_window_on_and_off(rt):
    m = Model(rt)
    prompt, step = m.tokens(100), m.tokens(1, seed=2)
    full, _ = m.dec.prefill(prompt)
    for window in (512, 2 ** 31 - 1):
        other = m.make()
        other.set_window(window)
        got, _ = other.prefill(prompt)
        # each of the two is a step (see expect) from the exact logits
        rms_close(got, full, "whole window", floor=2 * m.step(full) / 3)
    m.dec.set_window(10, 2)
    narrow, _ = m.dec.decode(step)
    m.dec.rollback(0, 100)
    m.dec.set_window(0)
    wide, _ = m.dec.decode(step)
    assert np.abs(narrow - wide).max() > 1e-2 * np.abs(wide).max()
    fresh = m.make()
    fresh.prefill(prompt)
    again, _ = fresh.decode(step)
    assert np.array_equal(wide, again)  # turned off, the decoder is what it was


@pytest.mark.parametrize("length", [1, 16, 37, 64])
def test_forks_answer_as_separate_prompts(rt, length):
    m = Model(rt)
    prompt = m.tokens(length)
    m.dec.prefill(prompt)
    used = m.dec.pool_stats()["used"]
    m.dec.fork(0, [2, 1])
    assert m.dec.pool_stats()["used"] == used + (2 if length % 16 else 0)
    other = m.make()
    for s in (0, 1, 2):
        other.prefill(prompt, slot=s)
    for i in range(20):  # over the page's end
        t = m.tokens(3, seed=10 + i)
        a, na = m.dec.decode(t, slots=[0, 1, 2])
        b, nb = other.decode(t, slots=[0, 1, 2])
        assert np.array_equal(a, b) and np.array_equal(na, nb)
    for layer in range(2):
        for s in (0, 1, 2):
            for x, y in zip(m.dec.read_kv(layer, s), other.read_kv(layer, s)):
                assert np.array_equal(x, y)
    m.dec.release(0)
    other.release(0)
    out_a, _ = m.dec.generate(m.tokens(2, seed=5), 30, slots=[2, 1])
    out_b, _ = other.generate(m.tokens(2, seed=5), 30, slots=[2, 1])
    assert np.array_equal(out_a, out_b)
    for s in (1, 2):
        m.dec.release(s)
    assert m.dec.pool_stats()["used"] == 0


def test_a_fork_rolled_back_writes_its_own_pages(rt):
    m = Model(rt)
    prompt = m.tokens(48)
    m.dec.prefill(prompt)
    m.dec.fork(0, [1])
    before = [m.dec.read_kv(layer, 0) for layer in range(2)]
    m.dec.rollback(1, 20)
    got, _ = m.dec.prefill(m.tokens(25, seed=9), slot=1)
    for layer in range(2):
        for x, y in zip(m.dec.read_kv(layer, 0), before[layer]):
            assert np.array_equal(x, y)
    other = m.make()
    other.prefill(prompt[:20])
    want, _ = other.prefill(m.tokens(25, seed=9))
    assert np.array_equal(got, want)
    m.dec.rollback(0, 30)  # the owner that is left now writes in place
    m.dec.decode([5])


def compact_oracle(o, keep):
    """The oracle's cache with only the rows `keep`, keys turned back."""
    back = torch.tensor(keep) - torch.arange(len(keep))
    c, s = o.rope_cos[back].double(), o.rope_sin[back].double()
    new = []
    for k, v in o.caches[0]:
        kk = k[:, keep].double()
        a, b = kk[..., 0::2], kk[..., 1::2]
        turned = torch.stack([a * c + b * s, b * c - a * s], -1).flatten(-2)
        new.append((turned.to(k.dtype), v[:, keep]))
    o.caches[0] = new


@pytest.mark.parametrize("keep", [list(range(4)) + list(range(60, 100)), [99], list(range(0, 100, 3)),
                                  list(range(33)) + [50, 51, 98], list(range(100)), list(range(40))])
@pytest.mark.parametrize("page_size", [16, 7])
def test_compaction(rt, keep, page_size):
    m = Model(rt, page_size=page_size)
    prompt = m.tokens(100)
    m.dec.prefill(prompt)
    m.oracle.forward(0, prompt)
    m.twin.forward(0, prompt)
    before = [m.dec.read_kv(layer) for layer in range(2)]
    m.dec.compact(0, keep)
    assert m.dec.length(0) == len(keep)
    assert m.dec.pool_stats()["used"] == -(-len(keep) // page_size)
    back = torch.tensor(keep) - torch.arange(len(keep))
    c, s = m.cos[back].double().numpy(), m.sin[back].double().numpy()
    for layer in range(2):
        k, v = m.dec.read_kv(layer)
        assert np.array_equal(v, before[layer][1][:, keep])
        old = before[layer][0][:, keep].astype(np.float64)
        a, b = old[..., 0::2], old[..., 1::2]
        want = np.stack([a * c + b * s, b * c - a * s], -1).reshape(old.shape)
        # one rounding to fp16, after two fp32 roundings of numbers no larger than |a| + |b|
        size = np.repeat(np.abs(a) + np.abs(b), 2, axis=-1)
        assert (np.abs(k - want) <= 2.0 ** -11 * np.abs(want) * 1.001 + 2.0 ** -23 * size + 2.0 ** -25).all()
    compact_oracle(m.oracle, keep)
    compact_oracle(m.twin, keep)
    for t in m.tokens(3, seed=4):
        got, _ = m.dec.decode([t])
        m.expect(got, [t], "after compaction")


def test_compaction_of_a_fork_leaves_the_other(rt):
    m = Model(rt)
    m.dec.prefill(m.tokens(64))
    m.dec.fork(0, [1])
    before = [m.dec.read_kv(layer, 0) for layer in range(2)]
    m.dec.compact(1, list(range(20)) + list(range(50, 64)))
    for layer in range(2):
        for x, y in zip(m.dec.read_kv(layer, 0), before[layer]):
            assert np.array_equal(x, y)
    assert m.dec.length(1) == 34 and m.dec.pool_stats()["used"] == 4 + 2


@pytest.mark.parametrize("count", [1, 50, 150])
@pytest.mark.parametrize("top", [0, 5])
def test_scored_prompts_against_their_logits(rt, count, top):
    m = Model(rt)
    prompt = m.tokens(count)
    logits, nxt = m.dec.prefill(prompt)
    other = m.make()
    got, next_scored = other.score(prompt, top=top)
    assert next_scored == nxt and other.length(0) == count
    x = torch.tensor(logits.astype(np.float64))
    lp = torch.log_softmax(x, -1)
    target = torch.tensor(np.append(prompt[1:], 0).astype(np.int64))
    want = lp.gather(1, target[:, None])[:, 0].numpy()
    want[-1] = 0.0
    # sums of 1000 positive terms in fp32 and a few roundings of numbers up to the log's size
    tol = 50 * 2.0 ** -24 + 8 * 2.0 ** -24 * (np.abs(want) + 7)
    assert (np.abs(got["logprobs"] - want) <= tol).all()
    entropy = -(lp.exp() * lp).sum(-1).numpy()
    assert (np.abs(got["entropy"] - entropy) <= 50 * 2.0 ** -24 * 16).all()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ranks = (order == target[:, None]).int().argmax(-1).numpy()
    ranks[-1] = -1
    assert np.array_equal(got["ranks"], ranks)
    assert np.array_equal(got["top_ids"], order[:, :top].numpy())
    best = lp.gather(1, order[:, :top]).numpy()
    assert (np.abs(got["top_logprobs"] - best) <= 50 * 2.0 ** -24 + 8 * 2.0 ** -24 * (np.abs(best) + 7)).all()


def test_scores_of_the_last_step(rt):
    m = Model(rt)
    for s in range(3):
        m.dec.prefill(m.tokens(20 + s, seed=s), slot=s)
    logits, nxt = m.dec.decode([1, 2, 3], slots=[0, 1, 2])
    lp = torch.log_softmax(torch.tensor(logits.astype(np.float64)), -1)
    greedy = m.dec.token_logprobs(3, top=2)
    assert np.array_equal(greedy["top_ids"][:, 0], nxt) and (greedy["ranks"] == 0).all()
    assert np.allclose(greedy["logprobs"], lp.max(-1)[0].numpy(), atol=1e-5, rtol=0)
    given = m.dec.token_logprobs(2, targets=[7, -1])
    assert abs(given["logprobs"][0] - lp[0, 7].item()) < 1e-5 and given["logprobs"][1] == 0 and given["ranks"][1] == -1
    out, _ = m.dec.generate([4, 5], 6, slots=[1, 2])
    last = m.dec.token_logprobs(2)
    assert (last["ranks"] == 0).all() and np.array_equal(m.dec.token_logprobs(2, targets=out[-1])["logprobs"],
                                                         last["logprobs"])


def test_generation_beyond_the_capacity(rt, monkeypatch):
    # All together: a windowed prompt, a fork, scores, and compaction whenever
    # the cache is full, against the oracle going the same way.
    window, sinks, cap = 40, 4, 96
    m = Model(rt, capacity=cap, max_slots=2)
    m.dec.set_window(window, sinks)
    monkeypatch.setattr(ref, "causal_gqa_attention", windowed(window, sinks))
    prompt = m.tokens(80)
    m.dec.score(prompt, top=3)
    m.dec.fork(0, [1])
    m.oracle.forward(0, prompt)
    m.twin.forward(0, prompt)
    keep = list(range(sinks)) + list(range(cap - window, cap))
    for i, t in enumerate(m.tokens(cap, seed=6)):
        if m.dec.length(1) == cap:
            m.dec.compact(1, keep)
            compact_oracle(m.oracle, keep)
            compact_oracle(m.twin, keep)
        got, _ = m.dec.decode([t], slots=[1])
        m.expect(got, [t], f"token {i}")
        if i == 40:
            m.dec.release(0)  # the prompt's other owner leaves
    assert m.dec.length(1) < cap


def test_refusals(rt):
    import tmc_cuda
    m = Model(rt, max_slots=3, pool_pages=40, capacity=512)
    d = m.dec
    refuse = lambda f, *a, **k: pytest.raises(tmc_cuda.TmcError, f, *a, **k)  # noqa: E731
    for bad in ((-1, 0), (5, -1)):
        refuse(d.set_window, *bad)
    refuse(d.fork, 0, [1])  # nothing to fork
    d.prefill(m.tokens(20))
    refuse(d.fork, 0, [0])
    refuse(d.fork, 0, [1, 1])
    refuse(d.fork, 0, [3])
    refuse(d.fork, -1, [1])
    refuse(d.fork, 0, [])
    d.prefill(m.tokens(5), slot=1)
    refuse(d.fork, 0, [2, 1])  # slot 1 is taken: slot 2 is given back
    assert d.length(2) == 0 and d.pool_stats()["used"] == 3
    for bad in ([], [20], [-1, 3], [3, 3], [4, 2], list(range(21))):
        refuse(d.compact, 0, bad)
    assert d.length(0) == 20
    refuse(d.compact, 5, [0])
    refuse(d.token_logprobs, 6)  # the last step had five rows
    refuse(d.token_logprobs, 0)
    refuse(d.token_logprobs, 1, targets=[1000])
    refuse(d.token_logprobs, 1, targets=[-2])
    refuse(d.token_logprobs, 1, top=33)
    refuse(d.score, [1000])
    refuse(d.score, [])
    d.inject_page_failures(1)
    refuse(d.compact, 0, [0, 19])
    assert d.length(0) == 20 and d.pool_stats()["used"] == 3
    d.inject_page_failures(1)
    refuse(d.fork, 0, [2])
    assert d.length(2) == 0 and d.pool_stats()["used"] == 3
