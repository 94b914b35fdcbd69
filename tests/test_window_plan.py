"""How window attention calls are split (window_plan.hpp through tests/window_plan_shim.cpp), on
the CPU: the workspace that the library asks for, which does not know a call's capacity, holds
the partial states of whatever the call is split into."""

import ctypes
import os
import random
import shutil
import subprocess

import pytest

import tmc_cuda

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMS = 148


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("plan") / "libplan.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "aicompiler-test_b200", "csrc"),
                    os.path.join(ROOT, "tests", "window_plan_shim.cpp"), "-o", out], check=True, capture_output=True)
    lib = ctypes.CDLL(out)
    lib.plan.argtypes = [ctypes.c_int] * 5 + [ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    lib.most_splits.argtypes = [ctypes.c_int] * 5 + [ctypes.c_longlong, ctypes.c_int]
    return lib


def plan(lib, shape, keys):
    out = (ctypes.c_int * 5)()
    lib.plan(*shape, keys, SMS, out)
    return dict(zip(("decode", "tensor", "tiles", "cluster", "outer"), out))


def partial_bytes(shape, outer):
    sequences, rows, hq, _, d = shape
    return 0 if outer <= 1 else outer * sequences * rows * hq * (d + 2) * 4


SHAPES = [(1, 255, 16, 16, 64), (1, 64, 32, 8, 128), (1, 512, 32, 8, 128), (2, 1, 4, 1, 128), (1, 2, 32, 8, 128),
          (1, 40, 2, 1, 64), (3, 130, 24, 3, 128), (1, 90, 8, 8, 32), (64, 4, 32, 8, 128), (1, 700, 4, 1, 64)]


@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_the_workspace_holds_what_any_capacity_is_split_into(lib, shape):
    for bound in (100, 640, 1255, 5000, 70000):
        most = lib.most_splits(*shape, bound, SMS)
        keys = list(range(1, min(bound, 3000) + 1)) + list(range(3000, bound + 1, 97)) + [bound]
        assert most >= max(plan(lib, shape, k)["outer"] for k in keys if k <= bound)


def test_drawn_shapes(lib):
    rng = random.Random(7)
    for _ in range(400):
        hkv, d = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([16, 32, 64, 128])
        rows = rng.choice([1, 1, 2, 5, int(2 ** rng.uniform(1, 12))])
        shape = (int(2 ** rng.uniform(0, 7)), rows, hkv * rng.randint(1, 8), hkv, d)
        bound = int(2 ** rng.uniform(5, 17))
        most = lib.most_splits(*shape, bound, SMS)
        for k in [bound] + [rng.randint(1, bound) for _ in range(200)]:
            assert most >= plan(lib, shape, k)["outer"]


def test_the_librarys_answer_is_this_bound(lib):
    for sequences, rows, hq, hkv, d in SHAPES:
        for window, sinks in ((100, 4), (1000, 0), (65536, 64)):
            keys = window + sinks + (rows if rows > 1 else 0)
            got = tmc_cuda.lib.tmc_k_window_attention_workspace_bytes(sequences, rows, hq, hkv, d, window, sinks)
            shape = (sequences, rows, hq, hkv, d)
            assert got == partial_bytes(shape, lib.most_splits(*shape, keys, SMS))


def test_a_shorter_capacity_can_mean_more_splits(lib):
    # what the bound is for: room for four, five steps take three, four steps take four
    shape = (1, 1000, 8, 8, 64)
    assert [plan(lib, shape, 128 * steps)["outer"] for steps in (4, 5)] == [4, 3]
    assert lib.most_splits(*shape, 640, SMS) == 4


@pytest.mark.parametrize("sequences,max_rows,hq,hkv,d", [
    (1, 2 ** 30, 1024, 1, 64), (1, 2 ** 31 - 1, 512, 1, 128), (2 ** 31 - 1, 1, 32, 8, 128), (65536, 1, 4, 1, 64),
    (1, 1, 2 ** 31 - 1, 1, 64), (1, 2 ** 26, 1, 1, 32), (60000, 60000, 65535, 1, 16), (1, 1, 65535 * 17, 65535, 64)])
def test_calls_that_cannot_be_launched_need_no_workspace(sequences, max_rows, hq, hkv, d):
    assert tmc_cuda.lib.tmc_k_window_attention_workspace_bytes(sequences, max_rows, hq, hkv, d, 1024, 0) == 0
