"""The measured attention call as two streams make it at the same time."""

import pytest
import torch

import perf.operators as operators

pytestmark = pytest.mark.gpu


def test_attention_calls_of_two_streams_keep_apart(monkeypatch):
    case = next(c for c in operators.listed() if c["name"] == "attention decode long")
    monkeypatch.setattr(operators, "own", True)
    states = [operators.prepare(case, seed) for seed in (1, 2)]
    want = [operators.run(st).clone() for st in states]  # one after the other
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                operators.run(st)
    torch.cuda.synchronize()
    for st, w in zip(states, want):
        assert torch.equal(st["out"], w)
    spaces = []
    for stream in streams:
        with torch.cuda.stream(stream):
            spaces.append([operators._workspace(1 << 20) for _ in range(2)])
    assert len({s.data_ptr() for pair in spaces for s in pair}) == 4  # none is shared while it is held
    assert operators._workspace(0) is None
