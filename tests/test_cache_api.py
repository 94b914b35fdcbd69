"""Refusals of the serving-cache kernels: argument checks on the host, before any
launch (placeholder pointers are never dereferenced). CPU only."""

import pytest

import tmc_cuda

P = 0x1000


def attention(q=P, q_stride=512, out=P, out_stride=512, k=P, v=P, dtype=tmc_cuda.F16, table=P, table_stride=4,
              table_rows=P, row_starts=P, first=P, sequences=1, rows=1, max_rows=1, hq=4, hkv=2, d=128, page=16,
              pool_pages=8, capacity=64, window=16, sinks=0, scale=0.0, workspace=None, workspace_bytes=0):
    return tmc_cuda.lib.tmc_k_window_attention(
        q, q_stride, out, out_stride, k, v, dtype, table, table_stride, table_rows, row_starts, first, sequences, rows,
        max_rows, hq, hkv, d, page, pool_pages, capacity, window, sinks, scale, workspace, workspace_bytes, None, None)


def logprobs(logits=P, dtype=tmc_cuda.F32, stride=100, targets=P, rows=1, vocab=100, out=P, entropy=P, ranks=P, top=4,
             ids=P, values=P):
    return tmc_cuda.lib.tmc_k_token_logprobs(logits, dtype, stride, targets, rows, vocab, out, entropy, ranks, top, ids,
                                             values, None, None)


def copy(pools=P, pool_count=2, pool_pages=8, page_bytes=64, src=P, dst=P, count=1):
    return tmc_cuda.lib.tmc_k_kv_copy_pages(pools, pool_count, pool_pages, page_bytes, src, dst, count, None, None)


def compact(pools=P, layers=1, dtype=tmc_cuda.F16, pool_pages=8, hkv=2, d=64, page=16, src=P, src_count=4, dst=P,
            dst_count=4, keep=P, count=8, first=0, cos=P, sin=P, rope_rows=64):
    return tmc_cuda.lib.tmc_k_kv_compact(pools, layers, dtype, pool_pages, hkv, d, page, src, src_count, dst, dst_count,
                                         keep, count, first, cos, sin, rope_rows, None, None)


REFUSALS = [
    (attention, dict(q=None), "INVALID", "null"),
    (attention, dict(row_starts=None), "INVALID", "null"),
    (attention, dict(dtype=tmc_cuda.F32), "UNSUPPORTED", "fp16 or bf16"),
    (attention, dict(sequences=-1), "INVALID", "sequences"),
    (attention, dict(max_rows=0), "INVALID", "max_rows"),
    (attention, dict(hq=3), "INVALID", "multiple of hkv"),
    (attention, dict(hkv=0), "INVALID", "multiple of hkv"),
    (attention, dict(d=96), "UNSUPPORTED", "head dimension"),
    (attention, dict(page=0), "INVALID", "page_size"),
    (attention, dict(capacity=0), "INVALID", "capacity"),
    (attention, dict(window=0), "INVALID", "window >= 1"),
    (attention, dict(sinks=-1), "INVALID", "sinks >= 0"),
    (attention, dict(scale=-1.0), "INVALID", "scale"),
    (attention, dict(scale=float("nan")), "INVALID", "scale"),
    (attention, dict(scale=float("inf")), "INVALID", "scale"),
    (attention, dict(q_stride=511), "INVALID", "strides"),
    (attention, dict(out_stride=516), "INVALID", "strides"),
    (attention, dict(q=P + 8), "INVALID", "aligned"),
    (attention, dict(workspace=P + 4), "INVALID", "aligned"),
    (logprobs, dict(logits=None), "INVALID", "null"),
    (logprobs, dict(out=None, entropy=None, ranks=None, top=0), "INVALID", "null"),
    (logprobs, dict(targets=None), "INVALID", "need targets"),
    (logprobs, dict(ids=None), "INVALID", "null"),
    (logprobs, dict(dtype=tmc_cuda.I32), "UNSUPPORTED", "dtype"),
    (logprobs, dict(rows=-1), "INVALID", "rows >= 0"),
    (logprobs, dict(stride=99), "INVALID", "row_stride"),
    (logprobs, dict(top=33), "UNSUPPORTED", "top"),
    (logprobs, dict(top=5, vocab=4), "UNSUPPORTED", "top"),
    (logprobs, dict(logits=P + 2), "INVALID", "aligned"),
    (copy, dict(pools=None), "INVALID", "null"),
    (copy, dict(pool_count=0), "INVALID", "pool_count"),
    (copy, dict(count=-1), "INVALID", "count >= 0"),
    (copy, dict(page_bytes=24), "INVALID", "multiple of 16"),
    (copy, dict(page_bytes=0), "INVALID", "multiple of 16"),
    (copy, dict(count=9), "INVALID", "more targets"),
    (compact, dict(keep=None), "INVALID", "null"),
    (compact, dict(sin=None), "INVALID", "both rope tables"),
    (compact, dict(dtype=tmc_cuda.F32), "UNSUPPORTED", "fp16 or bf16"),
    (compact, dict(layers=0), "INVALID", "layers"),
    (compact, dict(d=12), "UNSUPPORTED", "multiple of 8"),
    (compact, dict(count=65), "INVALID", "must hold"),
    (compact, dict(first=2147483647), "INVALID", "must hold"),
    (compact, dict(rope_rows=0), "INVALID", "rope_rows"),
]


@pytest.mark.parametrize("call,change,code,fragment", REFUSALS,
                         ids=[f"{c.__name__}-{'-'.join(f'{k}={v}' for k, v in a.items())}" for c, a, _, _ in REFUSALS])
def test_bad_arguments_are_refused_on_the_host(call, change, code, fragment):
    assert call(**change) == getattr(tmc_cuda, "ERR_" + code)
    assert fragment in tmc_cuda.last_error()


@pytest.mark.parametrize("call,change", [(attention, dict(sequences=0)), (attention, dict(rows=0)),
                                         (logprobs, dict(rows=0)), (copy, dict(count=0)), (compact, dict(count=0))])
def test_empty_calls_do_nothing(call, change):
    assert call(**change) == tmc_cuda.OK


def test_window_attention_workspace_grows_only_where_splits_meet():
    need = tmc_cuda.window_attention_workspace_bytes
    assert need(64, 1, 32, 8, 128, 4096, 4) == 0  # enough CTAs without further splits
    assert need(1, 1, 4, 1, 128, 64, 4) == 0  # nothing to split
    assert need(1, 1, 4, 1, 128, 65536, 4) > 0
    assert need(0, 1, 4, 1, 128, 65536, 4) == 0 == need(1, 1, 4, 3, 128, 65536, 4)


def test_integers_beyond_32_bits_are_refused():
    class Array:
        def __init__(self, dtype=tmc_cuda.F16):
            self.dtype, self.nbytes = dtype, 64

        def data_ptr(self):
            return P

    class Runtime:
        stream = status_ptr = None

    a, n, f, rt = Array(), Array(tmc_cuda.I32), Array(tmc_cuda.F32), Runtime()
    with pytest.raises(tmc_cuda.TmcError, match="32 bits"):
        tmc_cuda.window_attention(rt, a, a, a, a, n, 4, n, n, n, 1, 1, 1, 4, 2, 128, 16, 8, 64, 1 << 32, 0)
    with pytest.raises(tmc_cuda.TmcError, match="32 bits"):
        tmc_cuda.kv_copy_pages(rt, a, 2, 8, 64, n, n, (1 << 32) + 1)
    with pytest.raises(tmc_cuda.TmcError, match="32 bits"):
        tmc_cuda.token_logprobs(rt, a, n, 1 << 33, 100, f)
    with pytest.raises(tmc_cuda.TmcError, match="32 bits"):
        tmc_cuda.kv_compact(rt, a, 1, 8, 2, 64, 16, n, 4, n, 4, n, 1 << 32)
    # the same refusals as the C entries give, through the packed form
    with pytest.raises(tmc_cuda.TmcError, match="window >= 1"):
        tmc_cuda.window_attention(rt, a, a, a, a, n, 4, n, n, n, 1, 1, 1, 4, 2, 128, 16, 8, 64, 0, 0)
    with pytest.raises(tmc_cuda.TmcError, match="scale"):
        tmc_cuda.window_attention(rt, a, a, a, a, n, 4, n, n, n, 1, 1, 1, 4, 2, 128, 16, 8, 64, 9, 0, scale=-0.5)
    with pytest.raises(tmc_cuda.TmcError, match="top"):
        tmc_cuda.token_logprobs(rt, a, n, 1, 100, f, top=33, top_ids=n, top_logprobs=f)
    with pytest.raises(tmc_cuda.TmcError, match="multiple of 8"):
        tmc_cuda.kv_compact(rt, a, 1, 8, 2, 12, 16, n, 4, n, 4, n, 1)
    for name in ("window_attention", "token_logprobs", "kv_copy_pages", "kv_compact"):
        assert getattr(tmc_cuda.lib, f"tmc_k_{name}_slots")(None) == tmc_cuda.ERR_INVALID


class Array:
    """Stands for a tensor of another library; nothing reads its memory."""

    def __init__(self, dtype):
        self.dtype, self.nbytes = dtype, 64

    def data_ptr(self):
        return P


class Handles:
    stream = status_ptr = None


@pytest.mark.parametrize("wrong", ["out", "k", "table", "starts"])
def test_attention_arrays_of_another_type_are_refused(wrong):
    types = dict(q="torch.float16", out="torch.float16", k="torch.float16", v="torch.float16", table="torch.int32",
                 rows="torch.int32", starts="torch.int32", first="torch.int32")
    types[wrong] = "torch.bfloat16" if types[wrong] == "torch.float16" else "torch.int64"
    a = {k: Array(t) for k, t in types.items()}
    with pytest.raises(TypeError):
        tmc_cuda.window_attention(Handles, a["q"], a["out"], a["k"], a["v"], a["table"], 4, a["rows"], a["starts"],
                                  a["first"], 0, 0, 1, 4, 2, 128, 16, 8, 64, 16)


def test_other_arrays_of_another_type_are_refused():
    f, i, wide = Array("torch.float32"), Array("torch.int32"), Array("torch.int64")
    with pytest.raises(TypeError):  # token ids as they come from an embedding's input
        tmc_cuda.token_logprobs(Handles, f, wide, 0, 100, f)
    with pytest.raises(TypeError):
        tmc_cuda.token_logprobs(Handles, f, i, 0, 100, Array("torch.bfloat16"))
    with pytest.raises(TypeError):
        tmc_cuda.token_logprobs(Handles, wide, i, 0, 100, f)
    with pytest.raises(TypeError):
        tmc_cuda.token_logprobs(Handles, Array("torch.float64"), i, 0, 100, f)
    with pytest.raises(TypeError):
        tmc_cuda.kv_copy_pages(Handles, wide, 2, 8, 64, wide, i, 0)
    with pytest.raises(TypeError):
        tmc_cuda.kv_compact(Handles, wide, 1, 8, 2, 64, 16, i, 4, i, 4, wide, 0)
    tmc_cuda.token_logprobs(Handles, f, i, 0, 100, f)
    tmc_cuda.kv_copy_pages(Handles, wide, 2, 8, 64, i, i, 0)
