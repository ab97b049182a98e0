"""Workloads of a decoder's step over a paged cache.

A decoder that searches for a transcript norms and turns its queries and keys,
writes keys and values into a paged cache of 16 or 8 bits, attends with one
token, a run of tokens or a tree of drafted ones over it, and steers its logits
by what was said and by a grammar before it chooses.  Each case is one
pass through one of the operators on that way.

With ``own`` false, ``run`` computes an operator from elementary torch
operations in 32 bits; with ``own`` true, it calls the framework's kernels.
"""
from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
TOP = {"e4m3": 448.0, "int8": 127.0}  # largest code
LEAST = 2.0 ** -96                    # rows below it are quantised as if it were their largest value
TWO64 = 1 << 64


# ---- the cases ------------------------------------------------------------------


def listed():
    return [
        # a decoder's step of 16 streams of 4 beams: the smallest call, where latency counts
        _rotary("norm_rotary_step", rows=64, heads=16, kv_heads=4, dim=128, rotary=128, far=2000),
        # queries and keys of the 280 chunks (188 encoder frames each) of a 1 h recording, three quarters of a head turned
        _rotary("norm_rotary_long_form", rows=52_640, heads=8, kv_heads=8, dim=128, rotary=96, layout="interleaved",
                norm="layer", far=45_000),
        # a step of 16 streams of 4 beams: a token of each written, and read back as it is kept
        _cache("cache_step", seqs=64, lo=126, hi=1500, new=1, kv_heads=4, dim=128, page=64, kind="e4m3", read="new"),
        # the last 512 tokens of 8 prompts written, the whole prompts read back for attention over them
        _cache("cache_prompts", seqs=8, lo=700, hi=8192, new=512, kv_heads=8, dim=128, page=64, kind="int8", read="all"),
        # the encoder frames of 256 clips of 1 to 20 s written once for all of a decoder's steps, and read back
        _cache("cache_clips", seqs=256, lo=13, hi=251, new=0, kv_heads=8, dim=64, page=16, kind="e4m3", dtype="f16",
               read="all"),
        # a step of one stream: one token over 126, in the model's own type
        _attention("tree_one", seqs=1, lo=126, hi=126, new=1, heads=16, kv_heads=4, dim=128, page=64, kind="bf16"),
        # a step of 64 streams of 4 beams, each beam over a cache of its own
        _attention("tree_beams", seqs=256, lo=126, hi=1500, new=1, heads=16, kv_heads=4, dim=128, page=64, kind="e4m3"),
        # trees of 16 drafted tokens over 32 prompts
        _attention("tree_drafts", seqs=32, lo=700, hi=8192, new=16, heads=32, kv_heads=8, dim=128, page=64, kind="int8",
                   tree=True),
        # a run of 5 tokens of 2 streams over a whole 1 h recording's frames, pages of 16
        _attention("tree_recording", seqs=2, lo=45_000, hi=45_000, new=5, heads=8, kv_heads=8, dim=64, page=16,
                   kind="f16", dtype="f16"),
        # a transducer's step: 16 streams of 4 beams, 1,024 pieces and the blank, the pieces said so far
        _logits("logits_transducer", rows=64, vocab=1025, history=64, dtype="f32", bias="none", states=0),
        # a text decoder's step: 64 streams of 8 beams, a large vocabulary, a grammar of 100 states
        _logits("logits_text", rows=512, vocab=128_000, history=1500, dtype="bf16", bias="all", states=100),
        # as many streams without a grammar, penalties of their own
        _logits("logits_streams", rows=64, vocab=128_000, history=8192, dtype="f16", bias="none", states=0, each=True),
    ]


def _named(name, case):
    return {"name": name, **case} if name else case


def _rotary(name, rows, heads, kv_heads, dim, rotary, far, layout="half", norm="rms", dtype="bf16"):
    return _named(name, {"op": "rotary", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
                         "far": far, "layout": layout, "norm": norm, "dtype": dtype})


def _cache(name, seqs, lo, hi, new, kv_heads, dim, page, kind, read, dtype="bf16", pick=1):
    """Sequences of lo to hi tokens, of which the last ``new`` (0: all) are written, and ``read`` ("new" or "all") read."""
    return _named(name, {"op": "cache", "seqs": seqs, "lo": lo, "hi": hi, "new": new, "kv_heads": kv_heads, "dim": dim,
                         "page": page, "kind": kind, "dtype": dtype, "read": read, "pick": pick})


def _attention(name, seqs, lo, hi, new, heads, kv_heads, dim, page, kind, dtype="bf16", tree=False, pick=1):
    """Sequences of lo to hi tokens, the last ``new`` of them the queries."""
    return _named(name, {"op": "attention", "seqs": seqs, "lo": lo, "hi": hi, "new": new, "heads": heads,
                         "kv_heads": kv_heads, "dim": dim, "page": page, "kind": kind, "dtype": dtype, "tree": tree,
                         "pick": pick})


def _logits(name, rows, vocab, history, dtype, bias, states, each=False):
    """``bias``: "none", "all" (one for all rows) or "rows"; ``states``: of a grammar, or 0; ``each``: penalties of
    each row's own."""
    return _named(name, {"op": "logits", "rows": rows, "vocab": vocab, "history": history, "dtype": dtype, "bias": bias,
                         "states": states, "each": each})


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "attention", "attention", "attention", "logits"])
    return {"rotary": _draw_rotary, "cache": _draw_cache, "attention": _draw_attention, "logits": _draw_logits}[op](rng)


def _draw_rotary(rng):
    dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([0, 1, 2, 4, 8])
    heads = rng.choice([1, 8, 16])
    return _rotary(None, rows=_log_int(rng, 1, 52_640 * 16 * 128 // ((heads + kv_heads) * dim * 2)), heads=heads,
                   kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2]), far=_log_int(rng, 16, 1_000_000),
                   layout=rng.choice(["half", "interleaved"]), norm=rng.choice(["rms", "rms", "layer"]),
                   dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))


def _draw_cache(rng):
    hi = _log_int(rng, 1, 8192)
    kv_heads = rng.choice([1, 2, 4, 8])
    return _cache(None, seqs=_log_int(rng, 1, max(1, min(300, 30_000 // hi))), lo=rng.randrange(0, hi + 1), hi=hi,
                  new=rng.choice([0, 1, _log_int(rng, 1, 512)]), kv_heads=kv_heads, dim=rng.choice([32, 64, 80, 128, 128]),
                  page=rng.choice([16, 32, 64, 128]), kind=rng.choice(["e4m3", "e4m3", "int8", "int8", "bf16"]),
                  dtype=rng.choice(["f32", "bf16", "bf16", "f16"]), read=rng.choice(["new", "all"]),
                  pick=rng.randrange(1 << 20))


def _draw_attention(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = min(32, kv_heads * rng.choice([1, 2, 4, 4, 8]))
    new = rng.choice([1, 1, 1, 2, 4, 5, 8, 16, 33, 64])
    hi = _log_int(rng, new, 45_000)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    return _attention(None, seqs=_log_int(rng, 1, max(1, min(256, 100_000 // hi))), lo=rng.randrange(0, hi + 1), hi=hi,
                      new=new, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 80, 96, 128, 128]),
                      page=rng.choice([16, 32, 64, 128]), kind=rng.choice([dtype, "e4m3", "e4m3", "int8", "int8"]),
                      dtype=dtype, tree=rng.choice([False, True]), pick=rng.randrange(1 << 20))


def _draw_logits(rng):
    vocab = rng.choice([1025, _log_int(rng, 40, 128_000), 8 * _log_int(rng, 5, 16_000)])
    return _logits(None, rows=_log_int(rng, 1, max(1, min(2048, 60_000_000 // vocab))), vocab=vocab,
                   history=rng.choice([0, _log_int(rng, 1, 8192)]), dtype=rng.choice(["f32", "bf16", "bf16", "f16"]),
                   bias=rng.choice(["none", "none", "all", "rows"]), states=rng.choice([0, 1, 7, 100]),
                   each=rng.choice([False, True]))


# ---- what a program has in hand before the call ------------------------------------


@functools.lru_cache(maxsize=None)
def _ops():
    """The handle a program keeps for all its calls."""
    from scriptrs_amd import ModelOps
    return ModelOps()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    return {"rotary": _rotary_inputs, "cache": _cache_inputs, "attention": _attention_inputs,
            "logits": _logits_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if case["op"] == "rotary":
        if own:
            from scriptrs_amd import RotaryTable
            x["table"] = RotaryTable(case["rotary"], layout=case["layout"])
        else:
            step = [round(f / (2 * math.pi) * TWO64) for f in _frequencies(case)]
            x["steps"] = torch.tensor([s - TWO64 if s >= TWO64 // 2 else s for s in step], device="cuda")
    if case["op"] in ("cache", "attention"):
        _prepare_cache(case, x)
    return x


def run(state):
    return {"rotary": _run_rotary, "cache": _run_cache, "attention": _run_attention,
            "logits": _run_logits}[state["case"]["op"]](state)


def work(case):
    return {"rotary": _rotary_work, "cache": _cache_work, "attention": _attention_work,
            "logits": _logits_work}[case["op"]](case)


def exact(case, seed):
    with torch.no_grad():
        return {"rotary": _rotary_exact, "cache": _cache_exact, "attention": _attention_exact,
                "logits": _logits_exact}[case["op"]](case, _inputs(case, seed))


# ---- norms of queries and keys, and their rotary positions ----------------------------

EPS = 1e-5
BASE = 10_000.0


def _frequencies(case):
    """Radians a position for each pair of channels."""
    return [BASE ** (-2 * p / case["rotary"]) for p in range(case["rotary"] // 2)]


def _rotary_inputs(case, seed):
    g = _gen(seed)
    n, H, K, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    # queries, keys and values of one projection; a few channels are far larger than the rest, with an offset
    loud = torch.where(torch.rand(H + 2 * K, D, device="cuda", generator=g) < 0.03, 10.0, 1.0)
    x = ((torch.randn(n, H + 2 * K, D, device="cuda", generator=g) + 0.2) * loud).to(DTYPES[case["dtype"]])
    if n >= 1024:  # packed sequences, each from a place of its own
        first = torch.randint(0, case["far"], (n // 188 + 1,), device="cuda", generator=g)
        at = first.repeat_interleave(188)[:n] + torch.arange(n, device="cuda") % 188
    else:          # a step: a token of each stream
        at = torch.randint(0, case["far"], (n,), device="cuda", generator=g)
    q_weight, k_weight = (1 + 0.1 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    return {"q": x[:, :H], "k": x[:, H:H + K] if K else None, "positions": at.int(), "q_weight": q_weight,
            "k_weight": k_weight if K else None}


def _rotary_work(case):
    values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    return {"bytes": 2 * values * ESIZE[case["dtype"]] + 4 * case["rows"] + 8 * case["dim"], "flops": 7 * values}


def _pairs(x, case):
    R = case["rotary"]
    return (x[..., :R // 2], x[..., R // 2:R]) if case["layout"] == "half" else (x[..., 0:R:2], x[..., 1:R:2])


def _joined(a, b, rest, case):
    return torch.cat([torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2), rest], -1)


def _run_rotary(state):
    case = state["case"]
    if own:
        return _ops().norm_rotary(state["table"], state["positions"], state["q"], state["k"], norm=case["norm"],
                                  q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS)
    # the angle as a fraction of a turn, whole turns dropped: products modulo 2^64
    turn = (state["positions"].long()[:, None] * state["steps"][None, :]) >> 32
    angle = (turn.float() * (2 * math.pi / 2 ** 32))[:, None, :]
    cos, sin = angle.cos(), angle.sin()

    def one(x, weight):
        if x is None:
            return None
        y = x.float()
        if case["norm"] == "layer":
            y = y - y.mean(-1, keepdim=True)
        y = y / ((y * y).mean(-1, keepdim=True) + EPS).sqrt() * weight
        a, b = _pairs(y, case)
        return _joined(a * cos - b * sin, b * cos + a * sin, y[..., case["rotary"]:], case).to(x.dtype)
    return [one(state["q"], state["q_weight"]), one(state["k"], state["k_weight"])]


def _rotary_exact(case, x):
    f = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    turn = torch.exp(1j * (x["positions"].double()[:, None] * f))[:, None, :]

    def one(t, weight):
        if t is None:
            return None
        y = t.double()
        centre = y.mean(2, keepdim=True) if case["norm"] == "layer" else 0.0
        spread = y.var(2, unbiased=False, keepdim=True) if case["norm"] == "layer" else y.square().mean(2, keepdim=True)
        y = (y - centre) * (spread + EPS).rsqrt() * weight.double()
        z = torch.complex(*(t.contiguous() for t in _pairs(y, case))) * turn
        return _joined(z.real, z.imag, y[..., case["rotary"]:], case)
    return [one(x["q"], x["q_weight"]), one(x["k"], x["k_weight"])]


# ---- a paged cache ----------------------------------------------------------------------


def _lengths(case):
    rng = random.Random(case["pick"])
    lo, hi = max(case["lo"], case["new"]), case["hi"]
    lo = min(lo, hi)
    n = [lo if lo == hi else int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1
         for _ in range(case["seqs"])]
    n[-1] = hi
    return n


def _new(case):
    """How many tokens of each sequence are new."""
    return [min(case["new"], n) if case["new"] else n for n in _lengths(case)]


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def _cache_inputs(case, seed):
    """Keys and values of all tokens, and where their pages are: in any order, room for a quarter more."""
    g = _gen(seed)
    lengths, page, K, D = _lengths(case), case["page"], case["kv_heads"], case["dim"]
    total = sum(lengths)
    # (keys have a few channels larger than the rest)
    loud = torch.where(torch.rand(K, D, device="cuda", generator=g) < 1 / 16, 3.0, 1.0)
    kv = torch.randn(total, 2 * K, D, device="cuda", generator=g)
    kv[:, :K] *= loud
    kv = kv.to(DTYPES[case["dtype"]])
    rng = np.random.RandomState((seed ^ case["pick"]) % (1 << 31))
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + 3
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((case["seqs"], max(1, -(-case["hi"] * 5 // (4 * page)))), -1, np.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = order[at:at + n]
        at += n
    return {"k": kv[:, :K], "v": kv[:, K:], "pages": pages, "table": torch.from_numpy(table).cuda(),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def _places(lengths, counts):
    """(sequence, position) of the last counts[s] tokens of each sequence, on the GPU."""
    s = np.repeat(np.arange(len(counts)), counts)
    first = np.asarray(lengths) - np.asarray(counts) - _offsets(counts)[:-1]
    return torch.from_numpy(s).cuda(), torch.from_numpy(np.arange(len(s)) + np.repeat(first, counts)).cuda()


def _quantised(x, kind):
    """Codes and scales of rows of 32-bit values."""
    if kind not in TOP:
        return x.to(DTYPES[kind]), None
    top = x.abs().amax(-1).clamp(min=LEAST)
    y = x * TOP[kind] / top[..., None]
    return (y.to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().to(torch.int8)), top / TOP[kind]


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales[..., None]


def _prepare_cache(case, x):
    """The cache with what was written before: all tokens but the new ones (cache), or all (attention)."""
    lengths, new = _lengths(case), _new(case)
    page, K, D = case["page"], case["kv_heads"], case["dim"]
    total = _offsets(lengths)
    if case["op"] == "cache":
        where = np.concatenate([np.arange(b - n, b) for b, n in zip(total[1:], new)] + [np.zeros(0, np.int64)])
        where = torch.from_numpy(where).cuda()
        written = x["k"], x["v"]
        x["k_new"], x["v_new"] = torch.cat(written, 1)[where].split(K, 1)  # (views of one projection's output)
        x["new_at"] = _places(lengths, new)
    read = lengths if case.get("read") != "new" else new
    if own:
        from scriptrs_amd import KvCache
        x["cache"] = KvCache(x["pages"], page, K, D, dtype=case["kind"])
        x["plan"] = _ops().cache_plan(_offsets(new), case.get("heads", K), K, D)
        x["read_plan"] = _ops().cache_plan(_offsets(read), case.get("heads", K), K, D) if case["op"] == "cache" else None
        _ops().cache_write(_ops().cache_plan(total, K, K, D), x["cache"], x["table"], x["lengths"], x["k"], x["v"])
    else:
        s, at = _places(lengths, lengths)
        x["read_at"] = (s, at) if case.get("read") != "new" else _places(lengths, new)
        x["cache"] = []
        for t in (x["k"], x["v"]):
            codes, scales = _quantised(t.float(), case["kind"])
            kept = codes.new_zeros(x["pages"], page, K, D) if codes.dtype != torch.float8_e4m3fn else \
                torch.zeros(x["pages"], page, K, D, dtype=torch.int8, device="cuda").view(torch.float8_e4m3fn)
            _put(kept, x["table"][s, at // page], at % page, codes)
            scaled = None
            if scales is not None:
                scaled = torch.zeros(x["pages"], page, K, device="cuda")
                scaled[x["table"][s, at // page], at % page] = scales
            x["cache"].append((kept, scaled))


def _put(kept, page, slot, codes):
    """kept[page, slot] = codes (8 bits as whole numbers: their indexing is the same)."""
    if codes.element_size() == 1:
        kept, codes = kept.view(torch.int8), codes.view(torch.int8)
    kept[page, slot] = codes


def _taken(kept, page, slot):
    if kept.element_size() == 1:
        return kept.view(torch.int8)[page, slot].view(kept.dtype)
    return kept[page, slot]


def _run_cache(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if dtype == torch.float32:
        dtype = torch.bfloat16  # (what attention takes)
    if own:
        _ops().cache_write(state["plan"], state["cache"], state["table"], state["lengths"], state["k_new"], state["v_new"])
        return list(_ops().cache_read(state["read_plan"], state["cache"], state["table"], state["lengths"], dtype=dtype))
    page = case["page"]
    s, at = state["new_at"]
    into, slot = state["table"][s, at // page], at % page
    outs = []
    for x, (kept, scaled) in zip((state["k_new"], state["v_new"]), state["cache"]):
        codes, scales = _quantised(x.float(), case["kind"])
        _put(kept, into, slot, codes)
        if scaled is not None:
            scaled[into, slot] = scales
    s, at = state["read_at"]
    out_of, slot = state["table"][s, at // page], at % page
    for kept, scaled in state["cache"]:
        outs.append(_values(_taken(kept, out_of, slot), None if scaled is None else scaled[out_of, slot]).to(dtype))
    return outs


def _cache_work(case):
    new, lengths = sum(_new(case)), sum(_lengths(case))
    read = new if case["read"] == "new" else lengths
    values = 2 * case["kv_heads"] * case["dim"]
    kept = values * ESIZE[case["kind"]] + (8 * case["kv_heads"] if case["kind"] in TOP else 0)
    return {"bytes": new * (values * ESIZE[case["dtype"]] + kept) + read * (2 * values + kept),
            "flops": values * (4 * new + read)}


def _kept_exact(x, kind):
    """What a cache gives back of rows of 64-bit values, from the codes' definition."""
    if kind in DTYPES:
        return x.to(DTYPES[kind]).double()
    largest = torch.maximum(x.abs().max(-1, keepdim=True).values, torch.full((), LEAST, dtype=torch.float64, device="cuda"))
    y = x * TOP[kind] / largest
    # a step of the codes at y: 1 for whole numbers; 2^-3 of its power of two, not below 2^-6's, with 3 bits behind the first
    step = torch.ones_like(y) if kind == "int8" else torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)
    return torch.round(y / step) * step * largest / TOP[kind]


def _cache_exact(case, x):
    lengths, new = _lengths(case), _new(case)
    ends = np.cumsum(lengths)
    read = lengths if case["read"] == "all" else new
    rows = torch.cat([torch.arange(e - n, e, device="cuda") for e, n in zip(ends, read)])
    # (a cache in 16 bits rounds to them once, whatever it is read as)
    return [_kept_exact(x[name].double()[rows], case["kind"]) for name in ("k", "v")]


# ---- attention of new tokens over the cache -----------------------------------------------


def _attention_inputs(case, seed):
    x = _cache_inputs(case, seed)
    g = _gen(seed + 1)
    new = _new(case)
    n = sum(new)
    x["q"] = torch.randn(n, case["heads"], case["dim"], device="cuda", generator=g).to(DTYPES[case["dtype"]])
    x["tree"] = None
    if case["tree"]:
        # a draft's parent is any earlier one, or the context; it sees itself and those above it
        rng = np.random.RandomState(seed % (1 << 31))
        rows = []
        for m in new:
            seen = []
            for i in range(m):
                parent = int(rng.randint(-1, i)) if i else -1
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            rows += seen
        x["tree"] = torch.from_numpy(np.array(rows, np.uint64).astype(np.int64)).cuda()
    return x


def _attention_work(case):
    lengths, new = _lengths(case), _new(case)
    rows, K, D = sum(new), case["kv_heads"], case["dim"]
    token = 2 * K * D * ESIZE[case["kind"]] + (8 * K if case["kind"] in TOP else 0)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lengths, new))
    return {"bytes": sum(lengths) * token + 2 * rows * case["heads"] * D * 2, "flops": 4 * D * case["heads"] * pairs}


SCORES = 1 << 27  # score elements, or gathered values, of the plain form at a time


def _run_attention(state):
    case = state["case"]
    q, tree = state["q"], state["tree"]
    if own:
        return _ops().cache_attention(state["plan"], state["cache"], state["table"], state["lengths"], q, tree=tree)
    H, K, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths, new = _lengths(case), _new(case)
    offsets = _offsets(new)
    out = torch.zeros_like(q)
    first = 0
    while first < len(new):  # as many sequences at a time, padded together, as fit
        last, m, n = first, 0, 0
        while last < len(new):
            m2, n2 = max(m, new[last]), max(n, lengths[last])
            if last > first and (last - first + 1) * n2 * max(m2 * H, K * D) > SCORES:
                break
            m, n, last = m2, n2, last + 1
        b = last - first
        if m:
            at = torch.arange(n, device="cuda")
            some = torch.tensor(new[first:last], device="cuda")[:, None]
            length = state["lengths"][first:last, None].long()
            i = torch.arange(m, device="cuda")[None, :]
            rows = torch.where(i < some, torch.from_numpy(offsets[first:last]).cuda()[:, None] + i, 0)
            pages = state["table"][first:last][:, at // page].clamp(min=0)
            held = at < length
            k, v = (torch.where(held[..., None, None], _values(_taken(kept, pages, (at % page).expand(b, n)),
                                                               None if scaled is None else scaled[pages, at % page]), 0.0)
                    for kept, scaled in state["cache"])
            draft = at - (length - some)  # [b, n]: which of the new tokens, negative for the context
            if tree is None:
                see = draft[:, None, :] <= i[:, :, None]
            else:
                bits = tree[rows][:, :, None] >> draft.clamp(0, 63)[:, None, :] & 1
                see = (draft < 0)[:, None, :] | (bits != 0)
            see = (see & held[:, None, :])[:, None, None]
            qb = q[rows].float().view(b, m, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(b * K, H // K * m, D)
            s = torch.bmm(qb, k.permute(0, 2, 3, 1).reshape(b * K, D, n).contiguous()).view(b, K, H // K, m, n) / math.sqrt(D)
            s = torch.where(see, s, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.where(see, (s - torch.where(top == float("-inf"), 0.0, top)).exp(), 0.0)
            o = torch.bmm(p.view(b * K, H // K * m, n), v.permute(0, 2, 1, 3).reshape(b * K, n, D).contiguous())
            o = o.view(b, K, H // K, m, D) / p.sum(-1, keepdim=True).clamp(min=1e-30)
            o = o.permute(0, 3, 1, 2, 4).reshape(b, m, H, D)
            is_row = i < some
            out[rows[is_row]] = o[is_row].to(q.dtype)
        first = last
    return out


def _attention_exact(case, x):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    lengths, new = _lengths(case), _new(case)
    if sum(n * m for n, m in zip(lengths, new)) * H * D > 1 << 40:
        return None
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    ends, rows = np.cumsum(lengths), np.cumsum(new)
    for n, m, end, row in zip(lengths, new, ends, rows):
        if m == 0:
            continue
        keys, values = (_kept_exact(x[t][end - n:end].double(), case["kind"]).transpose(0, 1).contiguous() for t in ("k", "v"))
        hidden = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        for i in range(m):
            if x["tree"] is None:
                hidden[i, n - m + i + 1:] = True
            else:
                bits = int(x["tree"][row - m + i]) % TWO64
                hidden[i, n - m:] = torch.tensor([not bits >> j & 1 for j in range(m)], device="cuda")
        for h in range(H):
            w = x["q"][row - m:row, h].double() @ keys[h // (H // K)].T.contiguous() / math.sqrt(D)
            out[row - m:row, h] = torch.softmax(w.masked_fill(hidden, float("-inf")), -1) @ values[h // (H // K)]
    return out


# ---- steering the logits --------------------------------------------------------------------


def _logits_inputs(case, seed):
    g = _gen(seed)
    n, V, L = case["rows"], case["vocab"], case["history"]

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)
    x = {"logits": torch.empty(n, V, dtype=DTYPES[case["dtype"]], device="cuda")}
    for r in range(0, n, 64):
        m = min(64, n - r)
        x["logits"][r:r + m] = torch.randn(m, V, device="cuda", generator=g).mul_(3).to(x["logits"].dtype)
    x["history"] = x["lengths"] = None
    if L:  # what was said: few tokens often, most once; rows are as far as they are
        said = (V * rand(n, L).pow(4)).long().clamp(max=V - 1)
        said = torch.where(rand(n, L) < 0.5, said, torch.randint(0, V, (n, L), device="cuda", generator=g))
        x["history"] = said.int()
        x["lengths"] = (L * rand(n)).ceil().int()
        x["lengths"][0] = L
    one = {"repetition": 1.2, "presence": 0.3, "frequency": 0.1}
    for name, value in one.items():
        x[name] = value * (0.5 + rand(n)) + (0.6 if name == "repetition" else 0.0) if case["each"] else value
    x["bias"] = None
    if case["bias"] != "none":
        shape = (V,) if case["bias"] == "all" else (n, V)
        x["bias"] = torch.where(rand(*shape) < 0.05, 4 * rand(*shape) - 2, 0.0)
    x["allowed"] = x["states"] = None
    if case["states"]:  # a grammar lets a quarter of the tokens through; a row in 8 has none
        words = -(-V // 32)
        a, b = (torch.randint(-(1 << 31), 1 << 31, (case["states"], words), device="cuda", generator=g) for _ in range(2))
        x["allowed"] = (a & b).int()
        x["states"] = torch.randint(0, case["states"], (n,), device="cuda", generator=g)
        x["states"] = torch.where(rand(n) < 1 / 8, -1, x["states"]).int()
    return x


def _logits_work(case):
    n, V, L = case["rows"], case["vocab"], case["history"]
    bias = 4 * V * {"none": 0, "all": 1, "rows": n}[case["bias"]]
    masks = 4 * (-(-V // 32)) * min(case["states"], n) + (4 * n if case["states"] else 0)
    said = (2 * L + 4) * n if L else 0  # (4 bytes a token, rows half full)
    return {"bytes": 2 * n * V * ESIZE[case["dtype"]] + bias + masks + said, "flops": n * V * (1 + (case["bias"] != "none"))}


def _column(value, rows):
    return value[:, None] if isinstance(value, torch.Tensor) else torch.full((rows, 1), value, device="cuda")


def _run_logits(state):
    case = state["case"]
    if own:
        return _ops().adjust_logits(state["logits"], history=state["history"], lengths=state["lengths"],
                                    repetition=state["repetition"], presence=state["presence"],
                                    frequency=state["frequency"], bias=state["bias"], allowed=state["allowed"],
                                    states=state["states"])
    n, V = case["rows"], case["vocab"]
    z = state["logits"].float()
    if state["history"] is not None:
        said = torch.arange(case["history"], device="cuda") < state["lengths"][:, None]
        count = torch.zeros(n, V, device="cuda").scatter_add_(1, state["history"].long(), said.float())
        repetition = _column(state["repetition"], n)
        z = torch.where(count > 0, torch.where(z > 0, z / repetition, z * repetition), z)
        z = z - (_column(state["presence"], n) * (count > 0) + _column(state["frequency"], n) * count)
    if state["bias"] is not None:
        z = z + state["bias"]
    if state["allowed"] is not None:
        t = torch.arange(V, device="cuda")
        bits = state["allowed"][:, t // 32] >> (t % 32).int() & 1
        free = state["states"] < 0
        ok = bits.bool()[state["states"].clamp(min=0).long()] | free[:, None]
        z = torch.where(ok, z, float("-inf"))
    return z.to(state["logits"].dtype)


def _logits_exact(case, x):
    n, V = case["rows"], case["vocab"]
    out = torch.empty(n, V, dtype=torch.float64, device="cuda")

    def of(name, r):
        return float(x[name][r]) if isinstance(x[name], torch.Tensor) else x[name]
    for r in range(n):
        z = x["logits"][r].double()
        if x["history"] is not None:
            said = x["history"][r, :int(x["lengths"][r])]
            token, count = torch.unique(said, return_counts=True)
            token = token.long()
            old = z[token]
            z[token] = torch.where(old < 0, old * of("repetition", r), old / of("repetition", r)) - of("presence", r) \
                - of("frequency", r) * count
        if x["bias"] is not None:
            z += (x["bias"] if case["bias"] == "all" else x["bias"][r]).double()
        out[r] = z
    if x["states"] is not None:
        shifts = torch.arange(32, device="cuda", dtype=torch.int32)
        for s in range(case["states"]):
            mine = x["states"] == s
            if bool(mine.any()):
                bits = (torch.bitwise_right_shift(x["allowed"][s][:, None], shifts) % 2).flatten()[:V]
                out[mine] = out[mine].masked_fill(bits == 0, float("-inf"))
    return out
