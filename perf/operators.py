"""Workloads of the operators that a recogniser runs behind the log-mel features.

The features of a batch of clips or chunks go through an encoder's blocks and
a decoder that searches for the transcript.  Each case is one pass through one
of the operators on that way: attention over packed sequences, rotary
positions, the norms around a block with its gate and residual scale, and a
step of beam search.  An encoder frame is 8 feature frames (1280 samples, 80 ms).

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
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}
SCORES = 1 << 27  # score elements of the plain attention at a time
TWO64 = 1 << 64


# ---- the cases ------------------------------------------------------------------


def listed():
    return [
        # the encoder of one 10 s clip: the smallest call, where latency counts
        _attention("attention_clip", seqs=1, lo=126, hi=126, heads=8, kv_heads=8, dim=128),
        # the encoder over the 280 chunks (188 encoder frames each) of a 1 h recording
        _attention("attention_long_form", seqs=280, lo=188, hi=188, heads=8, kv_heads=8, dim=128),
        # a ragged batch of clips of 1 to 20 s, frames without speech hidden
        _attention("attention_ragged", seqs=256, lo=13, hi=251, heads=8, kv_heads=8, dim=64, dtype="f16", mask=0.3),
        # a whole 1 h recording through an encoder with local attention (about 10 s to either side)
        _attention("attention_local", seqs=1, lo=45_000, hi=45_000, heads=8, kv_heads=8, dim=128, left=128, right=128),
        # a decoder over packed prompts of different lengths, causal, grouped heads
        _attention("attention_prompts", seqs=8, lo=700, hi=8192, heads=32, kv_heads=8, dim=128, right=0),
        # a decoder's step: one token of each of 4 beams over the encoder frames of 64 streams
        _attention("attention_step", seqs=64, lo=126, hi=1500, q=4, heads=16, kv_heads=4, dim=128),
        # a decoder's step of 16 streams of 4 beams: the smallest call
        {"name": "rotary_step", "op": "rotary", "rows": 64, "heads": 16, "kv_heads": 4, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "none", "far": 2000, "dtype": "bf16"},
        # queries and keys of the 280 chunks, part of the head rotated
        {"name": "rotary_long_form", "op": "rotary", "rows": 52_640, "heads": 8, "kv_heads": 8, "dim": 128,
         "rotary": 96, "layout": "interleaved", "scaling": "parts", "far": 45_000, "dtype": "bf16"},
        # one clip's block: half the feed-forward's output added, then the next block's norm
        {"name": "norm_clip", "op": "norm", "rows": 126, "width": 1024, "stream": "bf16", "dtype": "bf16",
         "post": "none", "pre": "layer", "gate": "none", "scale": 0.5},
        # the 280 chunks, a 32-bit residual stream, norms on both sides and a gate for each channel
        {"name": "norm_long_form", "op": "norm", "rows": 52_640, "width": 1024, "stream": "f32", "dtype": "bf16",
         "post": "rms", "pre": "rms", "gate": "channel", "scale": 1.0},
        # a transducer's step: 16 streams of 4 beams, 1,024 pieces and the blank, a recurrent state
        {"name": "beam_transducer", "op": "beam", "streams": 16, "beams": 4, "vocab": 1025, "dtype": "f32",
         "state": "recurrent", "length": 2, "channels": 640, "first": False},
        # a text decoder's step: 64 streams of 8 beams, a large vocabulary, its own keys and values reordered
        {"name": "beam_text", "op": "beam", "streams": 64, "beams": 8, "vocab": 128_000, "dtype": "bf16",
         "state": "cache", "length": 48, "channels": 512, "first": False},
    ]


def _attention(name, seqs, lo, hi, heads, kv_heads, dim, dtype="bf16", q=0, left=-1, right=-1, mask=0.0, pick=1):
    """Sequences of lo to hi keys; q: queries of each (0: as many as keys)."""
    case = {"op": "attention", "seqs": seqs, "lo": lo, "hi": hi, "q": q, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "left": left, "right": right, "mask": mask, "pick": pick}
    return {"name": name, **case} if name else case


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "norm", "beam"])
    return {"attention": _draw_attention, "rotary": _draw_rotary, "norm": _draw_norm, "beam": _draw_beam}[op](rng)


def _draw_attention(rng):
    kind = rng.choice(["encoder", "local", "prompts", "step"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 1, 2, 4, 8])
    heads = min(32, kv_heads * group)
    dim = rng.choice([64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    pick = rng.randrange(1 << 20)
    common = dict(heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, pick=pick)
    if kind == "encoder":
        hi = _log_int(rng, 1, 1500)
        return _attention(None, seqs=_log_int(rng, 1, max(1, min(300, 60_000 // hi))), lo=rng.randrange(0, hi + 1),
                          hi=hi, mask=rng.choice([0.0, 0.3]), **common)
    if kind == "local":
        hi = _log_int(rng, 500, 45_000)
        return _attention(None, seqs=rng.choice([1, 1, 2]), lo=hi, hi=hi, left=_log_int(rng, 16, 512),
                          right=rng.choice([0, _log_int(rng, 1, 256)]), **common)
    if kind == "prompts":
        hi = _log_int(rng, 2, 8192)
        return _attention(None, seqs=_log_int(rng, 1, max(1, min(64, 16_000 // hi))), lo=max(1, hi // rng.choice([1, 8])),
                          hi=hi, right=0, **common)
    hi = _log_int(rng, 1, 45_000)
    return _attention(None, seqs=_log_int(rng, 1, max(1, min(256, 100_000 // hi))), lo=rng.randrange(0, hi + 1), hi=hi,
                      q=rng.choice([1, 1, 2, 4, 5, 8]), mask=rng.choice([0.0, 0.0, 0.3]), **common)


def _draw_rotary(rng):
    dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([0, 1, 2, 4, 8])
    heads = rng.choice([1, 8, 16])
    return {"op": "rotary", "rows": _log_int(rng, 1, 52_640 * 16 * 128 // ((heads + kv_heads) * dim * 2)),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
            "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "base", "parts"]),
            "far": _log_int(rng, 16, 1_000_000), "dtype": rng.choice(["f32", "bf16", "f16"])}


def _draw_norm(rng):
    width = rng.choice([_log_int(rng, 16, 8192), 8 * _log_int(rng, 8, 1024)])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    return {"op": "norm", "rows": _log_int(rng, 1, max(2, 52_640 * 512 // width)), "width": width,
            "stream": rng.choice(["f32", dtype]), "dtype": dtype, "post": rng.choice(["none", "layer", "rms"]),
            "pre": rng.choice(["layer", "rms"]), "gate": rng.choice(["none", "channel", "rows"]),
            "scale": rng.choice([1.0, 0.5])}


def _draw_beam(rng):
    beams = rng.choice([1, 2, 4, 5, 8, 16])
    vocab = max(2 * beams + 2, rng.choice([1025, _log_int(rng, 40, 128_000)]))
    return {"op": "beam", "streams": _log_int(rng, 1, max(1, min(128, 50_000_000 // (beams * vocab)))), "beams": beams,
            "vocab": vocab, "dtype": rng.choice(["f32", "bf16", "f16"]), "state": rng.choice(["recurrent", "cache"]),
            "length": rng.choice([1, 2, 7, 16]), "channels": rng.choice([64, 333, 512, 640]),
            "first": rng.random() < 0.25}


# ---- what a program has in hand before the call ------------------------------------


@functools.lru_cache(maxsize=None)
def _ops():
    """The handle a program keeps for all its calls."""
    from scriptrs_amd import ModelOps
    return ModelOps()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "attention":
        if own:
            state["plan"] = _ops().attention_plan(state["q_offsets"], state["k_offsets"], case["heads"],
                                                  case["kv_heads"], case["dim"], left=case["left"],
                                                  right=case["right"])
        else:
            state["plan"] = _plain_plan(case, state["q_offsets"], state["k_offsets"])
    if case["op"] == "rotary":
        if own:
            from scriptrs_amd import RotaryTable
            state["table"] = RotaryTable(case["rotary"], layout=case["layout"], **_rotary_scaling(case))
        else:
            step = [round(f / (2 * math.pi) * TWO64) for f in _frequencies(case)]
            state["steps"] = torch.tensor([s - TWO64 if s >= TWO64 // 2 else s for s in step], device="cuda")
    return state


def _inputs(case, seed):
    return {"attention": _attention_inputs, "rotary": _rotary_inputs, "norm": _norm_inputs,
            "beam": _beam_inputs}[case["op"]](case, seed)


def run(state):
    return {"attention": _run_attention, "rotary": _run_rotary, "norm": _run_norm,
            "beam": _run_beam}[state["case"]["op"]](state)


def work(case):
    return {"attention": _attention_work, "rotary": _rotary_work, "norm": _norm_work, "beam": _beam_work}[case["op"]](case)


def exact(case, seed):
    with torch.no_grad():
        return {"attention": _attention_exact, "rotary": _rotary_exact, "norm": _norm_exact,
                "beam": _beam_exact}[case["op"]](case, _inputs(case, seed))


# ---- attention over packed sequences ------------------------------------------------


def _lengths(case):
    rng = random.Random(case["pick"])
    lo, hi = case["lo"], case["hi"]
    k = [lo if lo == hi else int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1
         for _ in range(case["seqs"])]
    k[-1] = hi
    return [case["q"] or n for n in k], k


def _attention_inputs(case, seed):
    lq, lk = _lengths(case)
    q_off, k_off = np.concatenate([[0], np.cumsum(lq)]), np.concatenate([[0], np.cumsum(lk)])
    g = _gen(seed)
    H, K, D, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]

    def rows(n, heads):
        return torch.randn(n, heads, D, device="cuda", generator=g, dtype=torch.float32).to(dtype)
    if case["q"]:  # queries of the decoder, keys and values projected from the encoder's frames
        q, kv = rows(int(q_off[-1]), H), rows(int(k_off[-1]), 2 * K)
        k, v = kv[:, :K], kv[:, K:]
    else:          # one projection
        x = rows(int(q_off[-1]), H + 2 * K)
        q, k, v = x[:, :H], x[:, H:H + K], x[:, H + K:]
    mask = None
    if case["mask"]:
        # 200 ms bursts of speech and pauses; one sequence in 16 has no speech at all
        n = int(k_off[-1])
        mask = (torch.rand(n // 3 + 1, device="cuda", generator=g) >= case["mask"]).repeat_interleave(3)[:n]
        speech = torch.rand(case["seqs"], device="cuda", generator=g) >= 1 / 16
        mask = mask & speech.repeat_interleave(torch.tensor(lk, device="cuda"))
    return {"q": q, "k": k, "v": v, "mask": mask, "q_offsets": q_off, "k_offsets": k_off}


def _visible_pairs(lq, lk, left, right):
    """(query, key) pairs that the window leaves: query i sees keys i + lk - lq - left .. i + lk - lq + right."""
    at = np.arange(lq, dtype=np.int64) + (lk - lq)
    first = np.maximum(at - left, 0) if left >= 0 else np.zeros(lq, np.int64)
    last = np.minimum(at + right, lk - 1) if right >= 0 else np.full(lq, lk - 1)
    return int(np.maximum(last - first + 1, 0).sum())


def _attention_work(case):
    lq, lk = _lengths(case)
    pairs = sum(_visible_pairs(a, b, case["left"], case["right"]) for a, b in zip(lq, lk))
    if case["mask"]:
        pairs = int(pairs * (1 - case["mask"]) * 15 / 16)
    e, D = ESIZE[case["dtype"]], case["dim"]
    moved = e * D * (2 * sum(lq) * case["heads"] + 2 * sum(lk) * case["kv_heads"]) + (sum(lk) if case["mask"] else 0)
    return {"bytes": moved, "flops": 4 * D * case["heads"] * pairs}


def _plain_plan(case, q_off, k_off):
    """Blocks of the plain form: short sequences padded together, long ones in
    blocks of queries with the keys that their window leaves; the rows they
    gather and what the window lets through."""
    left, right, heads = case["left"], case["right"], case["heads"]
    spans, group = [], []  # groups of (q0, q1, k0, k1, first query's place among the keys)

    def close():
        if group:
            spans.append(list(group))
            group.clear()
    for s in range(len(q_off) - 1):
        q0, q1, k0, k1 = int(q_off[s]), int(q_off[s + 1]), int(k_off[s]), int(k_off[s + 1])
        lq, lk = q1 - q0, k1 - k0
        if lq == 0:
            continue
        block = lq
        if lq * lk * heads > SCORES:
            block = max(64, min(1024, SCORES // (heads * lk))) if left < 0 or right < 0 else 512
        for b in range(0, lq, block):
            e = min(lq, b + block)
            lo, hi = 0, lk
            if block < lq:
                close()
                lo = max(0, b + lk - lq - left) if left >= 0 else 0
                hi = min(lk, e + lk - lq + right) if right >= 0 else lk
                lo, hi = min(lo, hi), max(lo, hi)
            group.append((q0 + b, q0 + e, k0 + lo, k0 + hi, b + lk - lq - lo))
            mq, mk = max(x[1] - x[0] for x in group), max(x[3] - x[2] for x in group)
            if block < lq:
                close()
            elif len(group) > 1 and len(group) * mq * mk * heads > SCORES:
                last = group.pop()
                close()
                group.append(last)
    close()
    plan = []
    for spans_of in spans:
        t = torch.tensor(spans_of, device="cuda")
        mq, mk = int((t[:, 1] - t[:, 0]).max()), int((t[:, 3] - t[:, 2]).max())
        i, j = torch.arange(mq, device="cuda"), torch.arange(mk, device="cuda")
        qi, kj = t[:, :1] + i, t[:, 2:3] + j
        in_q, in_k = qi < t[:, 1:2], kj < t[:, 3:4]
        see = in_k[:, None, :] & in_q[:, :, None]
        at = (t[:, 4:5] + i)[:, :, None]
        if left >= 0:
            see = see & (j >= at - left)
        if right >= 0:
            see = see & (j <= at + right)
        plan.append((qi[in_q], in_q, torch.where(in_q, qi, t[:, :1]), torch.where(in_k, kj, 0), see))
    return plan


def _run_attention(state):
    case = state["case"]
    q, k, v, mask = state["q"], state["k"], state["v"], state["mask"]
    if own:
        return _ops().attention(state["plan"], q, k, v, key_mask=mask)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if k.shape[0] == 0:
        return out
    for rows, in_q, qi, kj, see in state["plan"]:
        n, mq, mk = qi.shape[0], qi.shape[1], kj.shape[1]
        if mask is not None:
            see = see & mask[kj][:, None, :]
        see = see[:, None, None]
        qb = q[qi].float().permute(0, 2, 1, 3).reshape(n * K, H // K * mq, D)
        kb = k[kj].float().permute(0, 2, 3, 1).reshape(n * K, D, mk)
        vb = v[kj].float().permute(0, 2, 1, 3).reshape(n * K, mk, D)
        s = torch.bmm(qb, kb).mul_(1 / math.sqrt(D)).view(n, K, H // K, mq, mk)
        s = torch.where(see, s, float("-inf"))
        top = s.amax(-1, keepdim=True) if mk else s.new_full((n, K, H // K, mq, 1), float("-inf"))
        p = torch.where(see, s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_(), 0.0)
        o = torch.bmm(p.view(n * K, H // K * mq, mk), vb).view(n, K, H // K, mq, D)
        o = o / p.sum(-1, keepdim=True).clamp_(min=1e-30)
        out[rows] = o.permute(0, 3, 1, 2, 4).reshape(n, mq, H, D)[in_q].to(q.dtype)
    return out


def _attention_exact(case, x):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    lq, lk = _lengths(case)
    if sum(_visible_pairs(a, b, -1, -1) for a, b in zip(lq, lk)) * H * D > 1 << 44:
        return None
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for s, (a, b) in enumerate(zip(lq, lk)):
        if a == 0 or b == 0:
            continue
        q0, k0 = int(x["q_offsets"][s]), int(x["k_offsets"][s])
        keys = x["k"][k0:k0 + b].double().transpose(0, 1).contiguous()      # [K, b, D]
        values = x["v"][k0:k0 + b].double().transpose(0, 1).contiguous()
        speech = x["mask"][k0:k0 + b] if x["mask"] is not None else torch.ones(b, dtype=torch.bool, device="cuda")
        step = max(1, min(a, (1 << 27) // (b * H)))
        for i in range(0, a, step):
            m = min(step, a - i)
            place = torch.arange(i, i + m, device="cuda")[:, None] + (b - a)
            lo = max(0, i + b - a - case["left"]) if case["left"] >= 0 else 0
            hi = min(b, i + m + b - a + case["right"]) if case["right"] >= 0 else b
            if hi <= lo:
                continue
            j = torch.arange(lo, hi, device="cuda")[None, :]
            see = speech[None, lo:hi].expand(m, hi - lo)
            if case["left"] >= 0:
                see = see & (place - j <= case["left"])
            if case["right"] >= 0:
                see = see & (j - place <= case["right"])
            for h in range(K):
                query = x["q"][q0 + i:q0 + i + m, h * (H // K):(h + 1) * (H // K)].double()
                w = torch.tensordot(query, keys[h, lo:hi], dims=([2], [1])) / math.sqrt(D)  # [m, group, keys]
                w = w.masked_fill(~see[:, None, :], float("-inf"))
                logz = torch.logsumexp(w, -1, keepdim=True)
                w = torch.exp(w - torch.where(torch.isinf(logz), torch.zeros_like(logz), logz))
                out[q0 + i:q0 + i + m, h * (H // K):(h + 1) * (H // K)] = torch.tensordot(w, values[h, lo:hi], dims=1)
    return out


# ---- rotary positions -----------------------------------------------------------------

PARTS = {"factor": 8.0, "original": 4096, "low": 1.0, "high": 32.0}


def _rotary_scaling(case):
    kind = case["scaling"]
    if kind == "none":
        return {"base": 10_000.0}
    if kind in ("linear", "base"):
        return {"base": 10_000.0, "scaling": kind, "factor": 4.0}
    return {"base": 500_000.0, "scaling": "parts", "factor": PARTS["factor"], "original_length": PARTS["original"],
            "low": PARTS["low"], "high": PARTS["high"], "magnitude": 1 + 0.1 * math.log(PARTS["factor"])}


def _frequencies(case):
    """Radians a position for each pair of channels."""
    R = case["rotary"]
    s = _rotary_scaling(case)
    base = s["base"] * (s["factor"] ** (R / (R - 2)) if case["scaling"] == "base" else 1.0)
    f = [base ** (-2 * p / R) for p in range(R // 2)]
    if case["scaling"] == "linear":
        return [x / s["factor"] for x in f]
    if case["scaling"] == "parts":
        def keep(x):  # 1: turns often within the original length, kept; 0: slower than that, interpolated
            turns = PARTS["original"] * x / (2 * math.pi)
            return min(1.0, max(0.0, (turns - PARTS["low"]) / (PARTS["high"] - PARTS["low"])))
        return [x * ((1 - keep(x)) / PARTS["factor"] + keep(x)) for x in f]
    return f


def _rotary_inputs(case, seed):
    g = _gen(seed)
    n, H, K, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn(n, H + 2 * K, D, device="cuda", generator=g).to(DTYPES[case["dtype"]])
    if n >= 1024:  # packed sequences, each from a place of its own
        first = torch.randint(0, case["far"], (n // 188 + 1,), device="cuda", generator=g)
        at = first.repeat_interleave(188)[:n] + torch.arange(n, device="cuda") % 188
    else:          # a step: a token of each stream
        at = torch.randint(0, case["far"], (n,), device="cuda", generator=g)
    return {"q": x[:, :H], "k": x[:, H:H + K] if K else None, "positions": at.int()}


def _rotary_work(case):
    moved = 2 * case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"] * ESIZE[case["dtype"]]
    return {"bytes": moved + 4 * case["rows"],
            "flops": 3 * case["rows"] * (case["heads"] + case["kv_heads"]) * case["rotary"]}


def _pairs(x, R, layout):
    if layout == "half":
        return x[..., :R // 2], x[..., R // 2:R]
    return x[..., 0:R:2], x[..., 1:R:2]


def _join(a, b, rest, layout):
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _run_rotary(state):
    case = state["case"]
    q, k, at = state["q"], state["k"], state["positions"]
    if own:
        return _ops().rotary(state["table"], at, q, k)
    # the angle as a fraction of a turn, whole turns dropped: products modulo 2^64
    turn = (at.long()[:, None] * state["steps"][None, :]) >> 32
    angle = (turn.float() * (2 * math.pi / 2 ** 32))[:, None, :]
    m = _rotary_scaling(case).get("magnitude", 1.0)
    cos, sin = angle.cos() * m, angle.sin() * m
    outs = []
    for x in (q, k):
        if x is None:
            outs.append(None)
            continue
        a, b = _pairs(x.float(), case["rotary"], case["layout"])
        outs.append(_join(a * cos - b * sin, b * cos + a * sin, x[..., case["rotary"]:].float(), case["layout"]).to(x.dtype))
    return outs


def _rotary_exact(case, x):
    f = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(f, _rotary_scaling(case).get("magnitude", 1.0)).expand(case["rows"], -1).contiguous(),
                       x["positions"].double()[:, None] * f)[:, None, :]
    outs = []
    for t in (x["q"], x["k"]):
        if t is None:
            outs.append(None)
            continue
        a, b = _pairs(t.double(), case["rotary"], case["layout"])
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        outs.append(_join(z.real, z.imag, t[..., case["rotary"]:].double(), case["layout"]))
    return outs


# ---- norms around a block, its gate and residual scale -----------------------------------

EPS = 1e-5


def _norm_inputs(case, seed):
    g = _gen(seed)
    n, w, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    # a residual stream has a few channels far larger than the rest and an offset
    loud = torch.where(torch.rand(w, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    x = {"residual": ((normal(n, w) + 0.3) * loud).to(DTYPES[case["stream"]]), "block": normal(n, w).to(dtype)}
    x["gate"] = {"none": lambda: None, "channel": lambda: normal(w).mul(0.1).to(dtype),
                 "rows": lambda: normal(n, w).to(dtype)}[case["gate"]]()
    for side in ("post", "pre"):
        kind = case[side]
        x[side + "_weight"] = 1 + 0.1 * normal(w) if kind != "none" else None
        x[side + "_bias"] = 0.1 * normal(w) if kind == "layer" else None
    return x


def _norm_work(case):
    e, s = ESIZE[case["dtype"]], ESIZE[case["stream"]]
    each = 2 * s + 2 * e + (e if case["gate"] == "rows" else 0)
    weights = 4 * sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("post", "pre"))
    weights += e if case["gate"] == "channel" else 0
    return {"bytes": case["width"] * (case["rows"] * each + weights), "flops": 12 * case["rows"] * case["width"]}


def _run_norm(state):
    case = state["case"]
    r, y, gate = state["residual"], state["block"], state["gate"]
    if own:
        def kind(name):
            return None if case[name] == "none" else case[name]
        return _ops().residual_norm(r, y, scale=case["scale"], gate=gate,
                                    gate_activation="sigmoid" if case["gate"] == "rows" else None,
                                    post=kind("post"), post_weight=state["post_weight"], post_bias=state["post_bias"],
                                    pre=kind("pre"), pre_weight=state["pre_weight"], pre_bias=state["pre_bias"], eps=EPS)

    def norm(x, kind, weight, bias):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / (x * x).mean(-1, keepdim=True).add(EPS).sqrt() * weight
        return x + bias if kind == "layer" else x
    h = y.float()
    if case["post"] != "none":
        h = norm(h, case["post"], state["post_weight"], state["post_bias"])
    if gate is not None:
        h = h * (1 / (1 + (-gate.float()).exp()) if case["gate"] == "rows" else gate.float())
    x = r.float() + case["scale"] * h
    z = norm(x, case["pre"], state["pre_weight"], state["pre_bias"])
    return [x.to(r.dtype), z.to(y.dtype)]


def _norm_exact(case, s):
    def normed(x, side):
        kind = case[side]
        if kind == "none":
            return x
        centre = x.mean(1) if kind == "layer" else torch.zeros(len(x), dtype=x.dtype, device=x.device)
        spread = (x.square().mean(1) - 0 if kind == "rms" else x.var(1, unbiased=False)) + EPS
        out = torch.addcmul(torch.zeros_like(x), (x - centre[:, None]) * spread.rsqrt()[:, None], s[side + "_weight"].double())
        return out if s[side + "_bias"] is None else out + s[side + "_bias"].double()
    h = normed(s["block"].double(), "post")
    if case["gate"] == "channel":
        h = h * s["gate"].double()
    if case["gate"] == "rows":
        h = h * torch.sigmoid(s["gate"].double())
    stream = torch.add(s["residual"].double(), h, alpha=case["scale"])
    return [stream, normed(stream, "pre")]


# ---- a step of beam search -----------------------------------------------------------------


def _beam_inputs(case, seed):
    """A decoder's peaked distributions: two likely tokens a beam over a
    background, the totals of a stream's likely candidates at least 1/16
    apart, so that the choice does not hang on a rounding.  One beam in 10 has
    ended.  On a stream's first step only its first beam is alive and the
    background (on a grid of 1/64, with ties) is chosen from."""
    g = _gen(seed)
    B, W, V, dtype = case["streams"], case["beams"], case["vocab"], DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)
    logits = torch.empty(B * W, V, dtype=dtype, device="cuda")
    for r in range(0, B * W, 64):
        n = min(64, B * W - r)
        logits[r:r + n] = ((torch.randn(n, V, device="cuda", generator=g).clamp_(-5, 5) * 64).round_() / 64).to(dtype)
    gap = 0.25 if W <= 8 else 0.125
    slot = rand(B, 2 * W).argsort(-1).view(B * W, 2).sort(-1).values
    token = torch.stack([torch.randint(0, V // 2, (B * W,), device="cuda", generator=g),
                         torch.randint(V // 2, V - 1, (B * W,), device="cuda", generator=g)], 1)
    token = torch.where(rand(B * W, 1) < 0.5, token, token.flip(1))  # the likeliest token in either half
    likely = 14 - gap * (slot - slot[:, :1])
    logits.scatter_(1, token, likely.to(dtype))
    logz = torch.cat([torch.logsumexp(logits[r:r + 64].double(), 1) for r in range(0, B * W, 64)])
    best = -5 - gap * slot[:, 0] + (rand(B * W) - 0.5) / 32
    scores = (best - (14 - logz)).float().view(B, W)
    ended = rand(B, W) < 0.1
    scores = torch.where(ended, best.float().view(B, W), scores)
    if case["first"]:
        ended = torch.zeros_like(ended)
        scores = torch.full_like(scores, float("-inf"))
        scores[:, 0] = 0.0
    if case["state"] == "recurrent":
        shape, kind = (case["length"], B * W, case["channels"]), torch.float32
    else:
        shape, kind = (B * W, case["length"], case["channels"]), torch.bfloat16
    states = [torch.randn(shape, device="cuda", generator=g).to(kind) for _ in range(2)]
    return {"logits": logits, "scores": scores, "finished": ended, "states": states, "end": V - 1}


def _beam_work(case):
    rows = case["streams"] * case["beams"]
    states = 2 * 2 * rows * case["length"] * case["channels"] * (4 if case["state"] == "recurrent" else 2)
    return {"bytes": rows * (case["vocab"] * ESIZE[case["dtype"]] + 19) + states, "flops": 3 * rows * case["vocab"]}


def _run_beam(state):
    case = state["case"]
    logits, scores, ended, end = state["logits"], state["scores"], state["finished"], state["end"]
    dim = 1 if case["state"] == "recurrent" else 0
    if own:
        scores, parents, tokens, ended = _ops().beam_select(logits, scores, finished=ended, end_token=end)
        return [scores, parents, tokens, ended, *_ops().beam_reorder(parents, state["states"], dim=dim)]
    B, W, V = case["streams"], case["beams"], case["vocab"]
    x = logits.float()
    top = x.amax(1, keepdim=True)
    logz = top + (x - top).exp().sum(1, keepdim=True).log()
    total = scores.view(-1, 1) + (x - logz)
    total = torch.where(ended.view(-1, 1), float("-inf"), total)
    total[:, end] = torch.where(ended.view(-1), scores.view(-1), total[:, end])
    # the totals' order as whole numbers, the lower index first among equals
    bits = (total + 0.0).view(torch.int32).long().view(B, W * V)
    key = torch.where(bits < 0, (bits ^ 0x7FFFFFFF), bits)
    key = key * (1 << 31) + ((1 << 31) - 1 - torch.arange(W * V, device=key.device))
    at = (1 << 31) - 1 - (torch.topk(key, W, 1).values & ((1 << 31) - 1))
    best = total.view(B, W * V).gather(1, at)
    found = best > float("-inf")
    parents = torch.where(found, at // V, torch.arange(W, device=at.device)).int()
    tokens = torch.where(found, at % V, -1).int()
    was = ended.gather(1, parents.long())
    rows = (parents + W * torch.arange(B, device=at.device)[:, None]).view(-1)
    return [best, parents, tokens, was | (tokens == end), *[s.index_select(dim, rows) for s in state["states"]]]


def _beam_exact(case, x):
    B, W, V, end = case["streams"], case["beams"], case["vocab"], x["end"]
    scores, parents, tokens, ended = [], [], [], []
    slots = torch.arange(W, device="cuda")
    for b in range(B):
        rows = torch.log_softmax(x["logits"][b * W:(b + 1) * W].double(), 1) + x["scores"][b].double()[:, None]
        over = x["finished"][b]
        rows[over] = float("-inf")
        rows[over, end] = x["scores"][b].double()[over]
        value, order = torch.sort(rows.flatten(), descending=True, stable=True)
        value, order = value[:W], order[:W]
        alive = torch.isfinite(value)
        scores.append(value)
        parents.append(torch.where(alive, order.div(V, rounding_mode="floor"), slots))
        tokens.append(torch.where(alive, order.remainder(V), torch.full_like(order, -1)))
        ended.append(over[parents[-1]] | (tokens[-1] == end))
    p = torch.stack(parents)
    rows = (p + W * torch.arange(B, device="cuda")[:, None]).flatten()
    moved = [s[:, rows] if case["state"] == "recurrent" else s[rows] for s in x["states"]]
    return [torch.stack(scores), p.int(), torch.stack(tokens).int(), torch.stack(ended), *moved]
