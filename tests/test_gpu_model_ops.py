"""Rotary positions, norms around a block and beam search against plain
computations in 64 bits.

Tolerances: an output is rounded once to its type (half an ulp of the value, u =
2^-9 bfloat16, 2^-12 float16, 2^-25 float32; doubled below), after f32 arithmetic
whose error is stated beside each check."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


@pytest.fixture(scope="module")
def ops():
    from scriptrs_amd import ModelOps
    m = ModelOps()
    yield m
    m.close()


# ---- rotary ----------------------------------------------------------------------


def turned(x, positions, R, layout, freqs, magnitude=1.0, sign=1.0):
    import torch
    y = x.cpu().double().clone()
    angle = sign * positions.cpu().double()[:, None] * torch.tensor(freqs, dtype=torch.float64)
    c, s = magnitude * angle.cos()[:, None], magnitude * angle.sin()[:, None]
    first = slice(0, R // 2) if layout == "half" else slice(0, R, 2)
    second = slice(R // 2, R) if layout == "half" else slice(1, R, 2)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def close(got, want, dtype, slack):
    import torch
    err = (got.cpu().double() - want).abs()
    tol = U[dtype] * want.abs() + slack
    assert torch.isfinite(got).all() and (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,R", [(64, 64), (128, 96), (80, 80), (80, 40), (66, 30), (7, 2), (256, 256), (300, 64)])
def test_rotary(ops, dim, R, dtype, layout):
    import torch
    from scriptrs_amd import RotaryTable
    table = RotaryTable(R, layout=layout, base=10_000.0, magnitude=1.25)
    freqs = [10_000.0 ** (-2 * p / R) for p in range(R // 2)]
    g = torch.Generator(device="cuda").manual_seed(dim)
    for rows, heads, kv in ((1, 1, 0), (67, 5, 2), (3000, 2, 1)):
        x = torch.randn(rows, heads + 2 * kv, dim, device="cuda", generator=g).to(torch_dtype(dtype))
        q, k = x[:, :heads], x[:, heads:heads + kv] if kv else None
        pos = torch.randint(-100, 100_000, (rows,), device="cuda", generator=g, dtype=torch.int32)
        pos[0] = 2_147_483_647
        qo, ko = ops.rotary(table, pos, q, k)
        # values up to 5: angle off by 2e-7 rad, sine and cosine by 2e-7
        close(qo, turned(q, pos, R, layout, freqs, 1.25), dtype, 6e-6)
        if kv:
            close(ko, turned(k, pos, R, layout, freqs, 1.25), dtype, 6e-6)
            before = x.clone()
            q2, k2 = ops.rotary(table, pos, q, k, inplace=True)
            assert q2 is q and torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(x[:, heads + kv:], before[:, heads + kv:])


def test_rotary_inverse_is_the_gradient(ops):
    """The inverse undoes the turn, and is the gradient of it (by the formula and by differences)."""
    import torch
    from scriptrs_amd import RotaryTable
    g = torch.Generator(device="cuda").manual_seed(3)
    for layout in ("half", "interleaved"):
        table = RotaryTable(32, layout=layout)
        x, w = (torch.randn(50, 3, 40, device="cuda", generator=g) for _ in range(2))
        pos = torch.randint(0, 5000, (50,), device="cuda", generator=g, dtype=torch.int32)
        y, _ = ops.rotary(table, pos, x)
        back, _ = ops.rotary(table, pos, y, inverse=True)
        close(back, x.cpu().double(), "f32", 1e-5)
        grad, _ = ops.rotary(table, pos, w, inverse=True)
        xd = x.cpu().double().requires_grad_()
        freqs = [10_000.0 ** (-2 * p / 32) for p in range(16)]
        angle = pos.cpu().double()[:, None] * torch.tensor(freqs, dtype=torch.float64)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = (xd[..., :16], xd[..., 16:32]) if layout == "half" else (xd[..., 0:32:2], xd[..., 1:32:2])
        ya, yb = a * c - b * s, b * c + a * s
        yd = torch.cat([ya, yb], -1) if layout == "half" else torch.stack([ya, yb], -1).flatten(-2)
        (torch.cat([yd, xd[..., 32:]], -1) * w.cpu().double()).sum().backward()
        close(grad, xd.grad, "f32", 6e-6)
        # differences: the turn is linear, so a step of any size does
        d = torch.randn(x.shape, device="cuda", generator=g)
        diff = ((ops.rotary(table, pos, x + d)[0] - y).double() * w.double()).sum()
        want = (grad.double() * d.double()).sum()
        assert abs(float(diff - want)) <= 6e-6 * float((w.abs().double() * 4).sum())


@pytest.mark.parametrize("scaling", ["linear", "base", "parts"])
def test_rotary_scaling(ops, scaling):
    import torch
    from scriptrs_amd import RotaryTable
    R, factor, L, low, high = 64, 8.0, 4096, 1.0, 32.0
    base = 10_000.0 * (factor ** (R / (R - 2)) if scaling == "base" else 1.0)
    freqs = []
    for p in range(R // 2):
        f = base ** (-2 * p / R)
        if scaling == "linear":
            f /= factor
        if scaling == "parts":
            keep = min(1.0, max(0.0, (L * f / (2 * math.pi) - low) / (high - low)))
            f *= (1 - keep) / factor + keep
        freqs.append(f)
    table = RotaryTable(R, base=10_000.0, scaling=scaling, factor=factor, original_length=L, low=low, high=high)
    x = torch.randn(200, 2, R, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    pos = torch.arange(200, device="cuda", dtype=torch.int32) * 151
    close(ops.rotary(table, pos, x)[0], turned(x, pos, R, "half", freqs), "f32", 6e-6)


def test_rotary_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput, RotaryTable
    table = RotaryTable(32)
    x = torch.zeros(5, 2, 32, device="cuda")
    pos = torch.zeros(5, dtype=torch.int32, device="cuda")
    bad = [lambda: RotaryTable(31), lambda: RotaryTable(0), lambda: RotaryTable(258), lambda: RotaryTable(32, layout="x"),
           lambda: RotaryTable(32, base=0.5), lambda: RotaryTable(32, scaling="linear", factor=0.0),
           lambda: RotaryTable(32, scaling="parts", factor=2.0, original_length=10, low=2.0, high=1.0),
           lambda: RotaryTable(32, magnitude=float("inf")), lambda: RotaryTable(2, scaling="base", factor=2.0),
           lambda: ops.rotary(table, pos.long(), x), lambda: ops.rotary(table, pos[:4], x),
           lambda: ops.rotary(table, pos, x.double()), lambda: ops.rotary(table, pos, x[..., :16]),
           lambda: ops.rotary(table, pos, x, x.half()), lambda: ops.rotary(table, pos, x, x[:4]),
           lambda: ops.rotary(table, pos, x.cpu()), lambda: ops.rotary(table, pos, x.transpose(1, 2)),
           lambda: ops.rotary(table, pos, x[:, :1].expand(5, 2, 32), inplace=True),
           lambda: ops.rotary(table, pos, x, x[:, 1:], inplace=True)]
    for i, f in enumerate(bad):
        with pytest.raises(InvalidModelOutput):
            f()
            raise AssertionError(f"call {i} was not refused")
    assert ops.rotary(table, pos[:0], x[:0])[0].shape == (0, 2, 32)


# ---- norms around a block ----------------------------------------------------------


def normed(x, kind, w, b, eps):
    import torch
    if kind is None:
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * w.cpu().double()
    return x if b is None else x + b.cpu().double()


def norm_case(ops, rows, width, stream, dtype, post, pre, gate, act, seed=0, bias=True, view=False):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    pad = 3 if view else 0
    r = (normal(rows, width + pad) * 3 + 1).to(torch_dtype(stream))[:, pad:]
    y = normal(rows, width + pad).to(torch_dtype(dtype))[:, :width]
    gt = {None: None, "channel": normal(width), "rows": normal(rows, width)}[gate]
    gt = gt if gt is None else gt.to(torch_dtype(dtype))
    w = {n: 1 + 0.2 * normal(width) for n in ("post", "pre")}
    b = {n: normal(width) if k == "layer" and bias else None for n, k in (("post", post), ("pre", pre))}
    x, z = ops.residual_norm(r, y, scale=0.5, gate=gt, gate_activation=act, post=post,
                             post_weight=w["post"] if post else None, post_bias=b["post"], pre=pre,
                             pre_weight=w["pre"] if pre else None, pre_bias=b["pre"], eps=1e-5)
    h = normed(y.cpu().double(), post, w["post"], b["post"], 1e-5)
    if gt is not None:
        h = h * (torch.sigmoid(gt.cpu().double()) if act else gt.cpu().double())
    want = r.cpu().double() + 0.5 * h
    # f32 arithmetic on values up to about 40 (sums of a row in a fixed tree): 1e-5 of
    # a row's largest; a norm divides it by the row's deviation, which eps keeps above 3e-3
    big = want.abs().amax(1, keepdim=True) + h.abs().amax(1, keepdim=True)
    close(x, want, stream, 1e-5 * big)
    if pre is None:
        assert z is None
        return
    nz = normed(want, pre, w["pre"], b["pre"], 1e-5)
    dev = torch.sqrt(((want - (want.mean(1, keepdim=True) if pre == "layer" else 0)) ** 2).mean(1, keepdim=True) + 1e-5)
    close(z, nz, dtype, 3e-5 * big / dev + 1e-6)


@pytest.mark.parametrize("stream,dtype", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("width", [1, 2, 17, 64, 512, 520, 1000, 1024, 1032, 2048, 2055, 4096, 8191, 8200, 16384])
def test_residual_norm_widths(ops, width, stream, dtype):
    norm_case(ops, 9, width, stream, dtype, "layer", "rms", "rows", "sigmoid", seed=width)


@pytest.mark.parametrize("gate,act", [(None, None), ("channel", None), ("channel", "sigmoid"), ("rows", None)])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
def test_residual_norm_kinds(ops, post, pre, gate, act):
    for rows, width in ((1, 96), (67, 640)):
        norm_case(ops, rows, width, "f32", "bf16", post, pre, gate, act, bias=rows > 1)
        norm_case(ops, rows, width, "bf16", "bf16", post, pre, gate, act, view=True)


def test_residual_norm_in_place_and_extremes(ops):
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    r, y = (torch.randn(300, 1024, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.ones(1024, device="cuda")
    x, z = ops.residual_norm(r, y, pre="rms", pre_weight=w)
    r2, y2 = r.clone(), y.clone()
    x2, z2 = ops.residual_norm(r2, y2, pre="rms", pre_weight=w, out=r2, norm_out=y2)
    assert x2 is r2 and z2 is y2 and torch.equal(x2, x) and torch.equal(z2, z)
    # rows of zeros and of one value have no deviation; large offsets keep theirs
    r = torch.zeros(3, 1000, device="cuda")
    r[1] = 7.0
    r[2] = 1000.0 + torch.arange(1000, device="cuda") % 2
    _, z = ops.residual_norm(r, torch.zeros_like(r), pre="layer", pre_weight=w[:1000], eps=1e-5)
    assert (z[:2] == 0).all() and (z[2].abs() - 1).abs().max() < 1e-3


def test_residual_norm_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    bad = [lambda: ops.residual_norm(x, x[:3]), lambda: ops.residual_norm(x.bfloat16(), x), lambda: ops.residual_norm(x[0], x[0]),
           lambda: ops.residual_norm(x.double(), x.double()), lambda: ops.residual_norm(x, x, pre="rms"),
           lambda: ops.residual_norm(x, x, pre="rms", pre_weight=w, pre_bias=w), lambda: ops.residual_norm(x, x, pre="x", pre_weight=w),
           lambda: ops.residual_norm(x, x, pre="rms", pre_weight=w.half()), lambda: ops.residual_norm(x, x, gate=w.half()),
           lambda: ops.residual_norm(x, x, gate=w[:32]), lambda: ops.residual_norm(x, x, gate_activation="tanh"),
           lambda: ops.residual_norm(x.t(), x.t()), lambda: ops.residual_norm(x, x.cpu()),
           lambda: ops.residual_norm(x, x, eps=-1.0), lambda: ops.residual_norm(x, x, scale=float("nan")),
           lambda: ops.residual_norm(torch.zeros(1, 20000, device="cuda"), torch.zeros(1, 20000, device="cuda")),
           lambda: ops.residual_norm(x, x, out=torch.zeros(1, 64, device="cuda").expand(4, 64)),
           lambda: ops.residual_norm(x, x, pre="rms", pre_weight=w, out=x, norm_out=x)]
    for i, f in enumerate(bad):
        with pytest.raises(InvalidModelOutput):
            f()
            raise AssertionError(f"call {i} was not refused")
    assert ops.residual_norm(x[:0], x[:0])[0].shape == (0, 64)


# ---- beam search ---------------------------------------------------------------------


def selected(logits, scores, finished, end):
    """By the definition, in 64 bits on the host."""
    import torch
    B, W = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double()
    total = scores.cpu().double().view(-1, 1) + (x - torch.logsumexp(x, 1, keepdim=True))
    if finished is not None:
        f = finished.cpu().view(-1)
        total[f] = -math.inf
        total[f, end] = scores.cpu().double().view(-1)[f]
    total = torch.where(torch.isnan(total), -math.inf, total).view(B, W * V)
    value, at = torch.sort(total, stable=True, dim=1, descending=True)
    value, at = value[:, :W], at[:, :W]
    found = value > -math.inf
    place = torch.arange(W).expand(B, W)
    if at.shape[1] < W:
        value = torch.cat([value, torch.full((B, W - at.shape[1]), -math.inf, dtype=torch.float64)], 1)
    parents = torch.where(found, at // V, place[:, :at.shape[1]])
    tokens = torch.where(found, at % V, -1)
    ended = torch.gather(finished.cpu(), 1, parents) if finished is not None else torch.zeros_like(found)
    return value, parents.int(), tokens.int(), ended | (found & (tokens == end))


def beam_check(ops, logits, scores, finished=None, end=-1):
    import torch
    got = ops.beam_select(logits, scores, finished=finished, end_token=end)
    want = selected(logits, scores, finished, end)
    fin = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0]).cpu(), fin)
    # sums of exponentials in f32: 1e-6 of log, and the total's own rounding
    err = (got[0].cpu().double() - want[0])[fin].abs()
    assert (err <= 2e-6 + 4e-7 * want[0][fin].abs()).all(), float(err.max())
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a.cpu(), b), torch.nonzero(a.cpu() != b)[:4].tolist()
    return got


def grid_logits(g, rows, vocab, dtype):
    """Logits on a grid of 1/8 (ties abound): totals of a beam differ by 1/8 or are equal."""
    import torch
    return ((torch.randn(rows, vocab, device="cuda", generator=g) * 8).round() / 8).to(torch_dtype(dtype))


def apart_scores(logits, g):
    """Scores that put every beam's totals on a grid of 1/8 of its own offset, a multiple of 1/512 apart from the others'."""
    import torch
    import numpy as np
    rows = logits.shape[0]
    lz = torch.logsumexp(logits.cpu().double(), 1)
    rng = np.random.default_rng(int(torch.randint(0, 1 << 30, (1,), device="cuda", generator=g)))
    off = torch.from_numpy(rng.permutation(64)[:rows % 64 or 64] if rows <= 64 else
                           np.concatenate([rng.permutation(64) for _ in range(rows // 64 + 1)])[:rows]).double()
    return (lz + off / 512 - 8).float().cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("streams,beams,vocab", [(1, 1, 1), (2, 1, 50), (3, 4, 7), (2, 8, 1025), (2, 5, 4097), (1, 32, 33),
                                                 (2, 16, 9000), (1, 8, 40_000), (2, 3, 128_001)])
def test_beam_select(ops, streams, beams, vocab, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = grid_logits(g, streams * beams, vocab, dtype)
    # offsets of 1/512 within a stream keep beams apart (beams <= 64)
    scores = torch.cat([apart_scores(logits[b * beams:(b + 1) * beams], g) for b in range(streams)]).view(streams, beams)
    beam_check(ops, logits, scores)
    finished = torch.rand(streams, beams, device="cuda", generator=g) < 0.4
    scores = torch.where(finished, -3 - torch.arange(beams, device="cuda") / 512 - 1 / 1024, scores).contiguous()
    beam_check(ops, logits, scores, finished, end=vocab - 1)
    first = torch.full_like(scores, float("-inf"))
    first[:, 0] = 0.0
    beam_check(ops, logits, first, end=0)
    strided = torch.full((streams * beams, vocab + 3), float("nan"), dtype=logits.dtype, device="cuda")
    strided[:, 1:vocab + 1] = logits
    got = ops.beam_select(strided[:, 1:vocab + 1], first, end_token=0)
    for a, b in zip(got, ops.beam_select(logits, first, end_token=0)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("vocab", [40, 3000, 20_000])
def test_beam_ties_and_masked_tokens(ops, vocab):
    """Equal logits go to the lowest tokens and beams; tokens at -inf or the type's lowest value; whole rows
    hidden; NaN rows have no candidates."""
    import torch
    for beams in (1, 4, 16):
        logits = torch.zeros(2 * beams, vocab, device="cuda")
        scores = torch.zeros(2, beams, device="cuda")
        beam_check(ops, logits, scores)
        logits[:, vocab // 2:] = float("-inf")
        logits[::2, :3] = torch.finfo(torch.float32).min
        beam_check(ops, logits, scores, end=5)
        logits[:beams] = float("-inf")
        logits[:beams, 7] = 1.5
        got = beam_check(ops, logits, scores, end=5)
        assert (got[2][0] == 7).all()
        logits[:beams] = float("-inf")
        got = beam_check(ops, logits, scores)
        assert (got[2][0] == -1).all() and (got[1][0].cpu() == torch.arange(beams)).all()
        logits[beams:] = float("nan")
        if beams > 1:
            logits[beams + 1] = 0.25
            got = ops.beam_select(logits, scores)
            assert (got[1][1] == 1).all() and (got[2][1].cpu() == torch.arange(beams)).all()


@pytest.mark.parametrize("beams", [1, 3, 4, 8, 9, 32])
@pytest.mark.parametrize("shape,dim,dtype", [((2, -1, 640), 1, "f32"), ((-1, 7, 48), 0, "bf16"), ((-1, 3), 0, "bf16"),
                                             ((3, -1, 5), 1, "f32"), ((-1,), 0, "f16"), ((1, -1, 0), 1, "f32")])
def test_beam_reorder(ops, shape, dim, dtype, beams):
    import torch
    g = torch.Generator(device="cuda").manual_seed(beams)
    for streams in (1, 5):
        n = streams * beams
        parents = torch.randint(0, beams, (streams, beams), device="cuda", generator=g, dtype=torch.int32)
        full = [n if s == -1 else s for s in shape]
        states = [torch.randn(full, device="cuda", generator=g).to(torch_dtype(dtype)) for _ in range(11)]
        rows = (parents + beams * torch.arange(streams, device="cuda")[:, None]).view(-1)
        want = [s.index_select(dim, rows) for s in states]
        got = ops.beam_reorder(parents, states, dim=dim)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.beam_reorder(parents, states, dim=dim, out=states)
        assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_beam_reorder_ignores_parents_that_are_none(ops):
    import torch
    state = torch.arange(8.0, device="cuda").view(8, 1)
    parents = torch.tensor([[-1, 0, 99, 1], [3, 2, 1, 4]], dtype=torch.int32, device="cuda")
    got = ops.beam_reorder(parents, [state])[0]
    assert got.view(-1).tolist() == [0, 0, 2, 1, 7, 6, 5, 7]


def test_beam_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput
    logits, scores = torch.zeros(6, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    parents, state = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(6, 4, device="cuda")
    bad = [lambda: ops.beam_select(logits[:5], scores), lambda: ops.beam_select(logits, scores.double()),
           lambda: ops.beam_select(logits.double(), scores), lambda: ops.beam_select(logits, scores, end_token=10),
           lambda: ops.beam_select(logits, scores, finished=torch.zeros(2, 3, dtype=torch.bool, device="cuda")),
           lambda: ops.beam_select(logits, scores, finished=torch.zeros(2, 2, dtype=torch.bool, device="cuda"), end_token=1),
           lambda: ops.beam_select(logits.t(), scores), lambda: ops.beam_select(logits.cpu(), scores),
           lambda: ops.beam_select(torch.zeros(33, 4, device="cuda"), torch.zeros(1, 33, device="cuda")),
           lambda: ops.beam_select(logits[:, :0], scores),
           lambda: ops.beam_reorder(parents.long(), [state]), lambda: ops.beam_reorder(parents, [state[:5]]),
           lambda: ops.beam_reorder(parents, [state.t()], dim=1), lambda: ops.beam_reorder(parents, [state], out=[]),
           lambda: ops.beam_reorder(parents, [torch.zeros(12, 4, device="cuda")[:6]], out=[torch.zeros(6, 4, device="cuda").half()])]
    for i, f in enumerate(bad):
        with pytest.raises(InvalidModelOutput):
            f()
            raise AssertionError(f"call {i} was not refused")
    both = torch.zeros(9, 4, device="cuda")
    with pytest.raises(InvalidModelOutput):
        ops.beam_reorder(parents, [both[:6]], out=[both[3:]])


def test_captured(ops):
    """The operators of a decoder's step, captured once and replayed on new inputs."""
    import torch
    from scriptrs_amd import RotaryTable
    g = torch.Generator(device="cuda").manual_seed(12)
    table = RotaryTable(64)
    x = torch.randn(12, 2, 64, device="cuda", generator=g)
    pos = torch.arange(12, device="cuda", dtype=torch.int32)
    r, y, w = torch.randn(12, 128, device="cuda", generator=g), torch.randn(12, 128, device="cuda", generator=g), torch.ones(128, device="cuda")
    logits, scores = torch.randn(12, 20_000, device="cuda", generator=g), torch.randn(3, 4, device="cuda", generator=g)

    def step():
        q, _ = ops.rotary(table, pos, x)
        n = ops.residual_norm(r, y, pre="rms", pre_weight=w)
        s = ops.beam_select(logits, scores, end_token=3)
        return [q, *n, *s, *ops.beam_reorder(s[1], [r])]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(4):
        for t in (x, r, y, logits, scores):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def busy():
    """Holds the current stream for milliseconds, long after the host's next calls."""
    import torch
    torch.cuda._sleep(5_000_000)


def test_outputs_of_calls_on_another_stream(ops):
    """Memory that the current stream has freed and still reads is not the output of a call on another stream."""
    import torch
    side, n = torch.cuda.Stream(), 1 << 20
    x = torch.ones(1024, 1024, device="cuda")
    for _ in range(3):
        ops.residual_norm(x, x, stream=side)
        torch.cuda.synchronize()
        a, kept = torch.full((n,), 3.0, device="cuda").view(1024, 1024), torch.empty(n, device="cuda").view(1024, 1024)
        torch.cuda.synchronize()
        busy()
        kept.copy_(a)
        del a
        y, _ = ops.residual_norm(x, x, stream=side)
        torch.cuda.synchronize()
        assert (kept == 3).all() and (y == 2).all()


def test_inputs_of_calls_on_another_stream(ops):
    """An input that is freed after a call on another stream keeps its memory until the call has read it."""
    import torch
    side, x = torch.cuda.Stream(), torch.ones(1024, 1024, device="cuda")
    for _ in range(3):
        ops.residual_norm(x, x, stream=side)
        a = torch.full_like(x, 3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            busy()
        y, _ = ops.residual_norm(x, a, stream=side)
        del a
        junk = [torch.full_like(x, 9.0) for _ in range(4)]
        torch.cuda.synchronize()
        assert (y == 4).all()
        del junk


def test_outputs_of_another_stream_read_on_the_current_one(ops):
    """An output that is freed while the current stream reads it is not written by the other stream's next call."""
    import torch
    side, x = torch.cuda.Stream(), torch.ones(1024, 1024, device="cuda")
    for _ in range(3):
        y, _ = ops.residual_norm(x, x, stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        busy()
        kept = y * 1
        del y
        z, _ = ops.residual_norm(x, x, scale=6.0, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert (kept == 2).all() and (z == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,order", [((500, 3, 4, 64), (0, 2, 3)), ((500, 4, 3, 64), (0, 1, 3)), ((4, 500, 3, 64), (1, 0, 3)),
                                         ((4, 3, 500, 64), (2, 0, 3)), ((3, 4, 500, 64), (2, 1, 3))], ids=str)
def test_rotary_in_place_on_views_of_one_projection(ops, shape, order, dtype):
    """q and k interleaved by rows, by heads or head by head: turned where they lie, the third part untouched."""
    import torch
    from scriptrs_amd import RotaryTable
    x = torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(torch_dtype(dtype))
    part = next(i for i in range(4) if i not in order)

    def views(t):
        kept = [d for d in range(4) if d != part]
        return [t.select(part, i).permute([kept.index(d) for d in order]) for i in range(3)]
    q, k, v = views(x)
    assert q.shape == (500, 4, 64)
    pos = torch.arange(500, device="cuda", dtype=torch.int32)
    table, before = RotaryTable(64), v.clone()
    qo, ko = ops.rotary(table, pos, q, k)
    assert not torch.equal(qo, q)
    ops.rotary(table, pos, q, k, inplace=True)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(v, before)
