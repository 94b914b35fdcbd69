"""Sizes, plain forms and exact values of the serving-cache operators.

Four operators over the paged key/value cache and over what a decoder answers:

- ``attention``: causal attention of ragged query rows over cache pages, with a
  sliding window and a few first positions (sinks) that stay visible;
- ``logprobs``: log probabilities of given tokens with entropy, rank and the
  top alternatives;
- ``copy``: copies of whole pages in every layer (forking a sequence);
- ``compact``: kept rows of a sequence moved together into other pages, keys
  re-rotated to their new positions.

``run`` computes them with elementary torch operations, or with the library's
kernels where ``own`` is true.
"""

import functools
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- the library's calls ------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _library():
    """The binding and one runtime, kept as a program keeps them."""
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aicompiler-test_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import tmc_cuda
    return tmc_cuda, tmc_cuda.Runtime(0)


def _workspace(nbytes):
    """A call's own workspace, of the current stream: calls may overlap on the GPU."""
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---- sizes --------------------------------------------------------------------

def _spread(n, low, high):
    """n whole numbers between low and high, the largest first: ragged lengths."""
    return [high - (high - low) * ((s * 37) % 101) // 100 for s in range(n)]


def _sequences(c):
    """Query rows and last position + 1 (context) of every sequence of an attention case."""
    contexts = _spread(c["seqs"], c["context_low"], c["context"])
    rows = [min(r, n) for r, n in zip(_spread(c["seqs"], c["rows_low"], c["rows"]), contexts)]
    return rows, contexts


def listed():
    attention = dict(op="attention", dtype="f16", hq=32, hkv=8, d=128, page=16, sinks=4, rows=1, rows_low=1, behind=0)
    logprobs = dict(op="logprobs", dtype="f32", vocab=128256, stride=128256, masked=0)
    pages = dict(op="copy", dtype="f16", layers=32, hkv=8, d=128, page=16)
    compact = dict(op="compact", dtype="f16", layers=32, hkv=8, d=128, page=16)
    return [
        # One sequence answers one token: the launch and the reads' latency are what counts.
        dict(attention, name="attention decode 1", seqs=1, context=2048, context_low=2048, window=1024),
        # A full batch of sequences of different lengths, most of them longer than the window.
        dict(attention, name="attention decode 64", seqs=64, context=8192, context_low=700, window=4096),
        # One rank's share (one key/value head) of two very long contexts, read in a wide window.
        dict(attention, name="attention decode long", dtype="bf16", seqs=2, hq=4, hkv=1, page=64, context=100003,
             context_low=90001, window=65536, sinks=64),
        # One chunk of a prompt, multi-head attention with short heads, pages that are no power of two.
        dict(attention, name="attention chunk 255", seqs=1, hq=16, hkv=16, d=64, page=24, rows=255, rows_low=255,
             context=1791, context_low=1791, window=1000),
        # Several prompts in one call, some continuing a cached prefix, rows behind the last one unused.
        dict(attention, name="attention prompts 4", dtype="bf16", seqs=4, page=32, rows=2600, rows_low=500,
             context=4100, context_low=900, window=2048, behind=13),
        # The log probability of one answered token, with five alternatives.
        dict(logprobs, name="logprobs 1", rows=1, top=5),
        # A batch of answered tokens, with twenty alternatives; a third of the vocabulary is masked out.
        dict(logprobs, name="logprobs 64", rows=64, top=20, masked=33),
        # A prompt is scored: every position's next token, no alternatives; odd vocabulary, padded rows.
        dict(logprobs, name="logprobs 1500", rows=1500, dtype="bf16", vocab=50021, stride=50048, top=0),
        # A sequence is forked once: its last, partly filled page is copied in every layer.
        dict(pages, name="copy 1", pages=2, count=1),
        # Many sequences are forked or moved at once.
        dict(pages, name="copy 400", pages=1024, count=400),
        # A short sequence of a small model drops its middle.
        dict(compact, name="compact 60", layers=2, hkv=4, d=64, length=128, first=4, count=60),
        # A sequence at its capacity keeps its first positions and its newest half.
        dict(compact, name="compact 2044", length=4096, first=4, count=2044),
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention", "attention", "logprobs", "copy", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    hkv = rng.choice([1, 2, 4, 8, 16])
    d = rng.choice([32, 64, 128])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "attention":
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        prompts = rng.random() < 0.5
        seqs = _log_uniform(rng, 1, 6) if prompts else _log_uniform(rng, 1, 64)
        rows = _log_uniform(rng, 2, 1200) if prompts else 1
        context = rows + _log_uniform(rng, 1, 2500 if prompts else 8000)
        return dict(op=op, dtype=dtype, seqs=seqs, hq=hq, hkv=hkv, d=d, page=page, rows=rows,
                    rows_low=rng.randint(1, rows), context=context, context_low=rng.randint(1, context),
                    window=_log_uniform(rng, 1, 5000), sinks=rng.choice([0, 1, 4, 17, 64]), behind=rng.choice([0, 3]))
    if op == "logprobs":
        vocab = _log_uniform(rng, 40, 200000)
        rows = min(_log_uniform(rng, 1, 1500), max(1, 75000000 // vocab))
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=rows, vocab=vocab,
                    stride=vocab + rng.choice([0, 1, 8, 100]), top=rng.choice([0, 1, 5, 20, 32]),
                    masked=rng.choice([0, 0, 10, 90]))
    layers = _log_uniform(rng, 1, 32)
    if op == "copy":
        pages = _log_uniform(rng, 4, 800)
        while layers * pages * hkv * page * d > 1 << 28:
            pages = max(4, pages // 2)
            page = max(8, page // 2)
        return dict(op=op, dtype=dtype, layers=layers, hkv=hkv, d=d, page=page, pages=pages,
                    count=rng.randint(1, pages // 2))
    length = _log_uniform(rng, 20, 4000)
    first = rng.choice([0, 1, 4, 19])
    return dict(op=op, dtype=dtype, layers=layers, hkv=hkv, d=d, page=page, length=length, first=first,
                count=rng.randint(1, max(1, (length - first) // 2)))


# ---- inputs -------------------------------------------------------------------

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, shape, dtype, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    out.normal_(0.0, std, generator=g)
    return out


def _prepare_attention(c, g, seed):
    rows, contexts = _sequences(c)
    seqs, page = c["seqs"], c["page"]
    stride = -(-c["context"] // page)
    used = [-(-n // page) for n in contexts]
    pool_pages = sum(used) + 3
    pages = np.random.RandomState(seed % (1 << 31)).permutation(pool_pages)
    table = np.full((seqs, stride), -1, np.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = pages[at:at + n]
        at += n
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    total = starts[-1] + c["behind"]
    dtype = _DTYPES[c["dtype"]]
    shape = (pool_pages, c["hkv"], page, c["d"])
    return {
        "q": _normal(g, (total, c["hq"], c["d"]), dtype), "k": _normal(g, shape, dtype), "v": _normal(g, shape, dtype),
        "out": torch.full((total, c["hq"], c["d"]), 0.25, dtype=dtype, device="cuda"),
        "table": _i32(table), "table_rows": _i32(list(range(seqs))[::-1]), "starts": _i32(starts),
        "first": _i32([n - r for n, r in zip(contexts, rows)]), "most_rows": max(rows), "total": total,
        # the longest run of visible positions behind the sinks, over the sequences
        "span": max(n - max(0, n - r - c["window"] + 1) for n, r in zip(contexts, rows)),
        "pool_pages": pool_pages, "stride": stride,
    }


def _attention_tables(c, st):
    """The table row of sequence s is row seqs - 1 - s: rows need not come in order."""
    return st["table"].flip(0)


def _prepare_logprobs(c, g, seed):
    x = _normal(g, (c["rows"], c["stride"]), _DTYPES[c["dtype"]], 2.5)
    if c["masked"]:
        hidden = torch.rand((c["stride"],), generator=g, device="cuda") < c["masked"] / 100.0
        x[:, hidden] = float("-inf")
    targets = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
    # likely tokens, as answered ones are: the largest of a few
    seen = torch.randint(0, c["vocab"], (c["rows"], 64), generator=g, device="cuda")
    best = seen.gather(1, x.gather(1, seen).float().argmax(1, keepdim=True))[:, 0].to(torch.int32)
    even = torch.arange(c["rows"], device="cuda") % 2 == 0
    targets = torch.where(even, best, targets)
    if c["rows"] > 4:
        targets[-1] = -1  # the last position of a prompt has no next token
    new = functools.partial(torch.empty, device="cuda")
    return {"x": x, "targets": targets, "logprobs": new(c["rows"]), "entropy": new(c["rows"]),
            "ranks": new(c["rows"], dtype=torch.int32), "ids": new((c["rows"], c["top"]), dtype=torch.int32),
            "top": new((c["rows"], c["top"]))}


def _pools(kv):
    """The device array of pool addresses: K, V of layer 0, K, V of layer 1, ..."""
    step = kv[0].numel() * kv.element_size()
    return torch.tensor([kv.data_ptr() + i * step for i in range(kv.shape[0])], dtype=torch.int64, device="cuda")


def _prepare_copy(c, g, seed):
    kv = _normal(g, (2 * c["layers"], c["pages"], c["hkv"], c["page"], c["d"]), _DTYPES[c["dtype"]])
    order = np.random.RandomState(seed % (1 << 31)).permutation(c["pages"])
    count = c["count"]
    # sources may repeat (one prompt forked often), targets do not
    source = order[count:][np.random.RandomState((seed + 1) % (1 << 31)).randint(0, c["pages"] - count, count)]
    return {"kv": kv, "pools": _pools(kv), "source": _i32(source), "target": _i32(order[:count])}


def _compact_pages(c):
    return -(-c["length"] // c["page"]), -(-(c["first"] + c["count"]) // c["page"])


def _prepare_compact(c, g, seed):
    old, new = _compact_pages(c)
    kv = _normal(g, (2 * c["layers"], old + new + 1, c["hkv"], c["page"], c["d"]), _DTYPES[c["dtype"]])
    order = np.random.RandomState(seed % (1 << 31)).permutation(old + new + 1)
    angle = torch.arange(c["length"], dtype=torch.float64, device="cuda")[:, None] * 500000.0 ** (
        -torch.arange(0, c["d"], 2, dtype=torch.float64, device="cuda") / c["d"])
    count = c["count"]
    # two thirds are the newest positions, the others are chosen from before them
    newest = count - count // 3
    middle = np.random.RandomState((seed + 1) % (1 << 31)).permutation(
        np.arange(c["first"], max(c["length"] - newest, c["first"])))[:count // 3]
    keep = np.sort(np.concatenate([middle, np.arange(c["length"] - (count - len(middle)), c["length"])]))
    return {"kv": kv, "pools": _pools(kv), "source": _i32(order[:old]), "target": _i32(order[old:old + new]),
            "keep": _i32(keep), "cos": angle.cos().float(), "sin": angle.sin().float()}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    make = {"attention": _prepare_attention, "logprobs": _prepare_logprobs, "copy": _prepare_copy,
            "compact": _prepare_compact}[case["op"]]
    return dict(make(case, g, seed), case=case)


# ---- plain forms ----------------------------------------------------------------

def _plain_attention(c, st):
    seqs, g = c["seqs"], c["hq"] // c["hkv"]
    starts, first = st["starts"].long(), st["first"].long()
    rows = starts[1:] - starts[:-1]
    last = first + rows - 1
    # query rows of each sequence, padded to the longest one
    i = torch.arange(st["most_rows"], device="cuda")
    at = (starts[:-1, None] + i).clamp(max=st["total"] - 1)
    q = st["q"][at].float().view(seqs, -1, c["hkv"], g, c["d"]).permute(0, 2, 1, 3, 4).flatten(2, 3)
    # positions that some row of the sequence sees: the sinks, then a run up to the last
    low = (first - c["window"] + 1).clamp(min=0)
    j = torch.cat([torch.arange(c["sinks"], device="cuda").expand(seqs, -1),
                   low[:, None] + torch.arange(st["span"], device="cuda")], 1)
    once = torch.cat([j[:, :c["sinks"]] < low[:, None], j[:, c["sinks"]:] <= last[:, None]], 1)
    j = torch.where(once, j, 0)
    tables = _attention_tables(c, st)
    page = tables.gather(1, j // c["page"]).long()
    k = st["k"][page, :, j % c["page"]].float().permute(0, 2, 3, 1)
    v = st["v"][page, :, j % c["page"]].float().permute(0, 2, 1, 3)
    position = (first[:, None] + i)[:, :, None]
    seen = once[:, None] & (j[:, None] <= position) & ((j[:, None] > position - c["window"]) | (j[:, None] < c["sinks"]))
    seen = seen.repeat_interleave(g, 1)[:, None]
    s = torch.matmul(q, k) * c["d"] ** -0.5
    s = s.masked_fill(~seen, float("-inf"))
    s = s - s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.exp()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out = st["out"].clone()
    here = i < rows[:, None]
    out[at[here]] = o[here].to(out.dtype)
    return out


def _plain_logprobs(c, st):
    x = st["x"][:, :c["vocab"]].float()
    lse = x.amax(1, keepdim=True)
    lse = lse + (x - lse).exp().sum(1, keepdim=True).log()
    log_p = x - lse
    entropy = -torch.where(log_p > float("-inf"), log_p.exp() * log_p, 0.0).sum(1)
    given = st["targets"] >= 0
    t = st["targets"].long().clamp(min=0)[:, None]
    index = torch.arange(c["vocab"], device="cuda")
    xt = x.gather(1, t)
    ranks = (x > xt).sum(1) + ((x == xt) & (index < t)).sum(1)
    # larger values first, then lower indices: one whole number that orders both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 20) + ((1 << 20) - 1 - index)
    ids = (1 << 20) - 1 - (key.topk(c["top"], 1)[0] & ((1 << 20) - 1))
    return {"logprobs": torch.where(given, log_p.gather(1, t)[:, 0], 0.0), "entropy": entropy,
            "ranks": torch.where(given, ranks, -1).to(torch.int32), "ids": ids.to(torch.int32),
            "top": log_p.gather(1, ids)}


def _plain_copy(c, st):
    st["kv"][:, st["target"].long()] = st["kv"][:, st["source"].long()]
    return st["kv"]


def _plain_compact(c, st):
    keep = st["keep"].long()
    to = c["first"] + torch.arange(c["count"], device="cuda")
    rows = st["kv"][:, st["source"].long()[keep // c["page"]], :, keep % c["page"]].float()
    back = keep - to
    cos, sin = st["cos"][back.abs()], st["sin"][back.abs()] * back.sign()[:, None]
    cos, sin = cos[:, None, None], sin[:, None, None]
    a, b = rows[:, 0::2, :, 0::2], rows[:, 0::2, :, 1::2]
    rows[:, 0::2] = torch.stack([a * cos + b * sin, b * cos - a * sin], -1).flatten(-2)
    st["kv"][:, st["target"].long()[to // c["page"]], :, to % c["page"]] = rows.to(st["kv"].dtype)
    return st["kv"]


# ---- the library's kernels ------------------------------------------------------

def _own_attention(c, st):
    tmc, rt = _library()
    need = tmc.window_attention_workspace_bytes(c["seqs"], st["most_rows"], c["hq"], c["hkv"], c["d"], c["window"],
                                                c["sinks"])
    # Table rows shorter than their sequence name the pool's last page (-1, as an index), by its own
    # number here; the table of a single sequence is whole.
    table = st["table"] if c["seqs"] == 1 else st["table"].remainder(st["pool_pages"])
    tmc.window_attention(rt, st["q"], st["out"], st["k"], st["v"], table, st["stride"], st["table_rows"],
                         st["starts"], st["first"], c["seqs"], st["total"], st["most_rows"], c["hq"], c["hkv"], c["d"],
                         c["page"], st["pool_pages"], c["context"], c["window"], c["sinks"],
                         workspace=_workspace(need), stream=_stream())
    return st["out"]


def _own_logprobs(c, st):
    tmc, rt = _library()
    tmc.token_logprobs(rt, st["x"], st["targets"], c["rows"], c["vocab"], st["logprobs"], st["entropy"], st["ranks"],
                       c["top"], st["ids"], st["top"], row_stride=c["stride"], stream=_stream())
    return {k: st[k] for k in ("logprobs", "entropy", "ranks", "ids", "top")}


def _own_copy(c, st):
    tmc, rt = _library()
    tmc.kv_copy_pages(rt, st["pools"], 2 * c["layers"], c["pages"], c["hkv"] * c["page"] * c["d"] * 2, st["source"],
                      st["target"], c["count"], stream=_stream())
    return st["kv"]


def _own_compact(c, st):
    tmc, rt = _library()
    old, new = _compact_pages(c)
    tmc.kv_compact(rt, st["pools"], c["layers"], old + new + 1, c["hkv"], c["d"], c["page"], st["source"], old,
                   st["target"], new, st["keep"], c["count"], c["first"], st["cos"], st["sin"], c["length"],
                   dtype={"f16": tmc.F16, "bf16": tmc.BF16}[c["dtype"]], stream=_stream())
    return st["kv"]


def run(state):
    c = state["case"]
    if own:
        return {"attention": _own_attention, "logprobs": _own_logprobs, "copy": _own_copy,
                "compact": _own_compact}[c["op"]](c, state)
    return {"attention": _plain_attention, "logprobs": _plain_logprobs, "copy": _plain_copy,
            "compact": _plain_compact}[c["op"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "attention":
        rows, contexts = _sequences(c)
        w, sinks = c["window"], c["sinks"]
        read = seen = 0
        for r, n in zip(rows, contexts):
            low = max(0, n - r - w + 1)
            read += n - low + min(sinks, low)
            for p in range(n - r, n):
                own_low = max(0, p - w + 1)
                seen += p - own_low + 1 + min(sinks, own_low)
        return {"bytes": 2 * read * c["hkv"] * c["d"] * size + 2 * sum(rows) * c["hq"] * c["d"] * size,
                "flops": 4 * seen * c["hq"] * c["d"]}
    if c["op"] == "logprobs":
        return {"bytes": c["rows"] * (c["vocab"] * size + 16 + 8 * c["top"]), "flops": 6 * c["rows"] * c["vocab"]}
    if c["op"] == "copy":
        page_bytes = c["hkv"] * c["page"] * c["d"] * size
        return {"bytes": 2 * 2 * c["layers"] * c["count"] * page_bytes, "flops": 0}
    row_bytes = 2 * c["layers"] * c["hkv"] * c["d"] * size
    return {"bytes": c["count"] * (2 * row_bytes + 4 + 4 * c["d"]),
            "flops": 3 * c["count"] * c["layers"] * c["hkv"] * c["d"]}


# ---- exact values -----------------------------------------------------------------

def _exact_attention(c, st):
    """Each sequence by itself over its whole context, by the definition, in 64 bits."""
    out = st["out"].double()
    table = st["table"].cpu().numpy()
    starts, first = st["starts"].tolist(), st["first"].tolist()
    g = c["hq"] // c["hkv"]
    for s in range(c["seqs"]):
        a, b, p0 = starts[s], starts[s + 1], first[s]
        n = p0 + b - a
        ids = torch.tensor(table[int(st["table_rows"][s]), :-(-n // c["page"])].astype(np.int64), device="cuda")
        j = torch.arange(n, device="cuda")
        p = torch.arange(p0, n, device="cuda")[:, None]
        seen = (j <= p) & ((p - j < c["window"]) | (j < c["sinks"]))
        for h in range(c["hkv"]):
            k = st["k"][ids, h].reshape(-1, c["d"])[:n].double()
            v = st["v"][ids, h].reshape(-1, c["d"])[:n].double()
            for head in range(h * g, (h + 1) * g):
                score = (st["q"][a:b, head].double() @ k.T) / c["d"] ** 0.5
                weight = torch.softmax(score.masked_fill(~seen, float("-inf")), -1)
                out[a:b, head] = weight @ v
    return out


def _exact_logprobs(c, st):
    x = st["x"][:, :c["vocab"]].double()
    log_p = torch.log_softmax(x, 1)
    p = log_p.exp()
    rows = torch.arange(c["rows"], device="cuda")
    target = st["targets"].long()
    given = target >= 0
    safe = torch.where(given, target, 0)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    place = (order == safe[:, None]).int().argmax(1)
    return {"logprobs": torch.where(given, log_p[rows, safe], 0.0),
            "entropy": torch.special.entr(p).sum(1),
            "ranks": torch.where(given, place, -1).to(torch.int32),
            "ids": order[:, :c["top"]].to(torch.int32),
            "top": log_p.gather(1, order[:, :c["top"]])}


def _exact_copy(c, st):
    source = torch.arange(c["pages"], device="cuda")
    source[st["target"].long()] = st["source"].long()
    return torch.index_select(st["kv"], 1, source).double()


def _exact_compact(c, st):
    kv = st["kv"].double()
    source, target = st["source"].tolist(), st["target"].tolist()
    angle = torch.atan2(st["sin"].double(), st["cos"].double())
    # the tables hold cosine and sine rounded to 32 bits: their own length goes with them
    length = torch.hypot(st["sin"].double(), st["cos"].double())
    for i, p in enumerate(st["keep"].tolist()):
        to = c["first"] + i
        row = kv[:, source[p // c["page"]], :, p % c["page"]].clone()
        turn = torch.polar(length[abs(p - to)], -angle[abs(p - to)] * (1 if p >= to else -1))
        key = torch.view_as_complex(row[0::2].unflatten(-1, (-1, 2)).contiguous())
        row[0::2] = torch.view_as_real(key * turn).flatten(-2)
        kv[:, target[to // c["page"]], :, to % c["page"]] = row
    return kv


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "logprobs": _exact_logprobs, "copy": _exact_copy,
            "compact": _exact_compact}[case["op"]](case, st)
