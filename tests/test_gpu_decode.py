"""A decoder's step over a paged cache (norms of heads with rotary positions, the cache's write and read, attention of
new tokens over it, steered logits) against plain computations in 64 bits.

Tolerances: U is a rounding's half step (eps / 2 of the type).  What is added to an output's own rounding is
stated beside each check."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TOP = {"e4m3": 448.0, "int8": 127.0}


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


@pytest.fixture(scope="module")
def ops():
    from scriptrs_amd import ModelOps
    m = ModelOps()
    yield m
    m.close()


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol):
    import torch
    got = got.cpu().double()
    assert got.shape == want.shape
    same = torch.isnan(got) & torch.isnan(want) | (got == want)
    err = torch.where(same, torch.zeros_like(got), (got - want).abs())
    assert (err <= tol).all(), (float((err - tol).max()), int((~(err <= tol)).sum()))


# ---- norms of heads and rotary positions -------------------------------------------


def normed_turned(x, weight, positions, R, layout, norm, eps, magnitude=1.0, base=10_000.0):
    import torch
    y = x.cpu().double()
    if norm == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.cpu().double()
    angle = positions.cpu().double()[:, None] * torch.tensor([base ** (-2 * p / R) for p in range(R // 2)], dtype=torch.float64)
    c, s = magnitude * angle.cos()[:, None], magnitude * angle.sin()[:, None]
    first = slice(0, R // 2) if layout == "half" else slice(0, R, 2)
    second = slice(R // 2, R) if layout == "half" else slice(1, R, 2)
    out = y.clone()
    out[..., first] = y[..., first] * c - y[..., second] * s
    out[..., second] = y[..., second] * c + y[..., first] * s
    return out


def close_heads(got, want, dtype):
    # f32 arithmetic: at most 22 roundings of a sum over a head, halved by the root but doubled by a mean taken
    # off that is up to twice the spread, sine and cosine (5 half steps), weight, product and turn: below 96 half steps of the
    # largest value
    within(got, want, U[dtype] * want.abs() + 96 * 2.0 ** -24 * float(want.abs().max()))


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,R", [(64, 64), (128, 96), (80, 80), (80, 40), (66, 30), (7, 2), (2, 2), (256, 256), (255, 2), (128, 128)])
def test_norm_rotary(ops, dim, R, dtype, layout, norm):
    import torch
    from scriptrs_amd import RotaryTable
    table = RotaryTable(R, layout=layout, magnitude=1.25)
    g = gen(dim)
    for rows, heads, kv in ((1, 1, 0), (67, 5, 2), (3, 33, 33), (5000, 2, 1)):
        x = (torch.randn(rows, heads + 2 * kv, dim, device="cuda", generator=g) + 0.3).to(torch_dtype(dtype))
        if dim == 2 and norm == "layer":
            x[..., 1] = x[..., 0] + 1.0  # (a spread that is not lost in the inputs' own steps)
        q, k = x[:, :heads], x[:, heads:heads + kv] if kv else None
        wq = 1 + 0.1 * torch.randn(dim, device="cuda", generator=g)
        wk = 1 + 0.1 * torch.randn(dim, device="cuda", generator=g) if kv == 2 else None
        pos = torch.randint(-100, 100_000, (rows,), device="cuda", generator=g, dtype=torch.int32)
        pos[0] = 2_147_483_647
        qo, ko = ops.norm_rotary(table, pos, q, k, norm=norm, q_weight=wq, k_weight=wk, eps=1e-3)
        close_heads(qo, normed_turned(q, wq, pos, R, layout, norm, 1e-3, 1.25), dtype)
        if kv:
            close_heads(ko, normed_turned(k, wk, pos, R, layout, norm, 1e-3, 1.25), dtype)
            before = x.clone()
            q2, k2 = ops.norm_rotary(table, pos, q, k, norm=norm, q_weight=wq, k_weight=wk, eps=1e-3, inplace=True)
            assert q2 is q and torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(x[:, heads + kv:], before[:, heads + kv:])


def test_norm_rotary_of_single_head_columns(ops):
    """One head: a workgroup's heads are rows, whose sines and cosines fill the table."""
    import torch
    from scriptrs_amd import RotaryTable
    for dim, R in ((32, 32), (256, 256), (4, 2)):
        table = RotaryTable(R)
        x = torch.randn(20_000, 1, dim, device="cuda", generator=gen(R)).bfloat16()
        pos = torch.arange(20_000, device="cuda", dtype=torch.int32)
        close_heads(ops.norm_rotary(table, pos, x)[0], normed_turned(x, None, pos, R, "half", "rms", 1e-5), "bf16")


def test_norm_rotary_views(ops):
    """Unaligned channels, heads over rows, one row for all."""
    import torch
    from scriptrs_amd import RotaryTable
    table = RotaryTable(64, layout="interleaved")
    pos = torch.arange(40, device="cuda", dtype=torch.int32)
    wide = torch.randn(40, 3, 70, device="cuda", generator=gen(1)).half()
    for x in (wide[..., 1:65], wide[..., 2:66], wide[..., 4:68], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :64],
              wide[:1, :, :64].expand(40, 3, 64)):
        got, _ = ops.norm_rotary(table, pos, x)
        close_heads(got, normed_turned(x, None, pos, 64, "interleaved", "rms", 1e-5), "f16")


def test_norm_rotary_values_that_are_not_finite(ops):
    """A head with one is NaN or as the formula has it; the others are as without it."""
    import torch
    from scriptrs_amd import RotaryTable
    table = RotaryTable(32)
    x = torch.randn(6, 4, 32, device="cuda", generator=gen(2))
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    want, _ = ops.norm_rotary(table, pos, x, norm="layer")
    y = x.clone()
    y[2, 1, 5], y[3, 0, 31] = float("nan"), float("inf")
    got, _ = ops.norm_rotary(table, pos, y, norm="layer")
    assert got[2, 1].isnan().all() and got[3, 0].isnan().any()
    got[2, 1], got[3, 0] = want[2, 1], want[3, 0]
    assert torch.equal(got, want)


def test_norm_rotary_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput, RotaryTable
    table, pos = RotaryTable(32), torch.zeros(5, dtype=torch.int32, device="cuda")
    x, w = torch.zeros(5, 2, 32, device="cuda"), torch.ones(32, device="cuda")
    bad = [lambda: ops.norm_rotary(table, pos, x, norm="none"), lambda: ops.norm_rotary(table, pos, x, eps=-1.0),
           lambda: ops.norm_rotary(table, pos, x, eps=float("nan")), lambda: ops.norm_rotary(table, pos, x, q_weight=w[:16]),
           lambda: ops.norm_rotary(table, pos, x, q_weight=w.half()), lambda: ops.norm_rotary(table, pos, x, k_weight=w),
           lambda: ops.norm_rotary(table, pos, x, q_weight=w.cpu()), lambda: ops.norm_rotary(table, pos.long(), x),
           lambda: ops.norm_rotary(table, pos[:4], x), lambda: ops.norm_rotary(table, pos, x[..., :16]),
           lambda: ops.norm_rotary(table, pos, x, x.half()), lambda: ops.norm_rotary(table, pos, x.double()),
           lambda: ops.norm_rotary(table, pos, torch.zeros(5, 2, 264, device="cuda")),
           lambda: ops.norm_rotary(table, pos, x[:, :1].expand(5, 2, 32), inplace=True),
           lambda: ops.norm_rotary(table, pos, x, x, inplace=True),
           lambda: ops.norm_rotary(table, pos, x, q_weight=x.view(-1)[:32], inplace=True)]
    for f in bad:
        with pytest.raises(InvalidModelOutput):
            f()
    q, k = ops.norm_rotary(table, pos[:0], x[:0])
    assert q.shape == (0, 2, 32) and k is None


# ---- the cache's write and read -------------------------------------------------------


def quantised(x, kind):
    """What rows of values come back as, in float32: from the definition, in 64 bits."""
    import torch
    x = x.cpu()
    if kind not in TOP:
        return x.to(torch_dtype(kind)).float()
    a = x.double().abs().amax(-1, keepdim=True).clamp(min=2.0 ** -96)
    y = x.double() * TOP[kind] / a
    step = torch.ones_like(y)
    if kind == "e4m3":
        step = torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)
    codes = (y / step).round() * step
    out = codes.float() * (a.float() / TOP[kind])
    return torch.where(torch.isfinite(x).all(-1, keepdim=True), out, torch.full_like(out, math.nan))


def paged(lengths, page, rng, spare=3, columns=None):
    """(pages, table): each sequence's pages, in any order."""
    import torch
    held = [-(-max(0, n) // page) for n in lengths]
    order = rng.permutation(sum(held) + spare).astype(np.int32)
    table = np.full((len(lengths), columns or max(1, max(held, default=1))), -1, np.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = order[at:at + n]
        at += n
    return len(order), torch.from_numpy(table).cuda()


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 16, 16), (3, 80, 32), (8, 128, 64), (2, 64, 1024), (5, 112, 16), (4, 32, 128)])
def test_cache_round_trip(ops, kv_heads, dim, page, dtype, kind):
    """New tokens of ragged sequences (none, one, many, past several pages) read back as the codes' definition
    has them, and nothing else of the cache is written."""
    import torch
    from scriptrs_amd import KvCache
    rng = np.random.RandomState(dim + page)
    lengths, new = [1, 0, 37, page, 5 * page + 1, 700], [1, 0, 37, 1, 2 * page + 3, 20]
    pages, table = paged(lengths, page, rng)
    cache = KvCache(pages, page, kv_heads, dim, dtype=kind)
    cache.data.fill_(0x5a)
    g = gen(dim)
    kv = torch.randn(sum(new), 2 * kv_heads, dim, device="cuda", generator=g).to(torch_dtype(dtype))
    kv[3, 0] = 0.0
    kv[5, :, 1:] *= 1e-3
    k, v = kv[:, :kv_heads], kv[:, kv_heads:]
    plan = ops.cache_plan(offsets_of(new), kv_heads, kv_heads, dim)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ops.cache_write(plan, cache, table, length, k, v)
    back = ops.cache_read(plan, cache, table, length, dtype=torch.float32)
    for got, x in zip(back, (k, v)):
        want = quantised(x, kind)
        if dtype == "f32" and kind in TOP:
            # (x M is rounded before it is divided: a value next to the middle of two codes may go to either)
            scale = x.cpu().abs().amax(-1, keepdim=True).clamp(min=2.0 ** -96).double() / TOP[kind]
            half = 0.5 * scale if kind == "int8" else torch.maximum(x.cpu().double().abs() * 2.0 ** -4, scale * 2.0 ** -10)
            within(got, x.cpu().double(), half * (1 + 2.0 ** -20) + 2.0 ** -22 * x.cpu().double().abs())
        else:
            assert torch.equal(got.cpu(), want)
    # the places of other tokens, from the layout that the header states
    size = 1 if kind in TOP else 2
    touched = np.zeros(tuple(cache.data.shape), bool)
    for s, (n, m) in enumerate(zip(lengths, new)):
        for token in range(n - m, n):
            p, slot = int(table[s, token // page]), token % page
            for part in range(2):
                at = (part * page + slot) * dim * size
                touched[p, :, at:at + dim * size] = True
                if kind in TOP:
                    at = 2 * page * dim + 4 * (part * page + slot)
                    touched[p, :, at:at + 4] = True
    assert (cache.data.cpu().numpy()[~touched] == 0x5a).all()
    for out in ("bf16", "f16"):
        o = [torch.empty(sum(new), kv_heads, dim + 8, device="cuda", dtype=torch_dtype(out))[..., :dim] for _ in range(2)]
        got = ops.cache_read(plan, cache, table, length, out=o)
        assert got[0] is o[0] and torch.equal(o[0], back[0].to(o[0].dtype)) and torch.equal(o[1], back[1].to(o[1].dtype))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_cache_codes_of_every_mantissa(ops, kind):
    """All 16-bit mantissas against all largest ones: quotients halfway between two codes go to the even one."""
    import torch
    from scriptrs_amd import KvCache
    for dtype, bits in ((torch.bfloat16, 7), (torch.float16, 10)):
        tops = torch.arange(2 ** bits, 2 ** (bits + 1), device="cuda").double() / 2 ** bits
        tops = tops[::max(1, len(tops) // 256)]
        x = torch.empty(len(tops) * 10, 1, 128, device="cuda", dtype=dtype)
        for e in range(10):
            part = (torch.arange(127, device="cuda").double() / 127 * (2 ** bits - 1)).round() / 2 ** bits + 1
            x[e::10, 0, 1:] = (part * 2.0 ** -e).to(dtype)
            x[e::10, 0, 0] = (2 * tops).to(dtype) * (1 if e % 2 else -1)
        rows = len(x)
        plan = ops.cache_plan([0, rows], 1, 1, 128)
        cache = KvCache(-(-rows // 64), 64, 1, 128, dtype=kind)
        table = torch.arange(cache.pages, device="cuda", dtype=torch.int32)[None]
        length = torch.tensor([rows], dtype=torch.int32, device="cuda")
        ops.cache_write(plan, cache, table, length, x, -x)
        k, v = ops.cache_read(plan, cache, table, length, dtype=torch.float32)
        assert torch.equal(k.cpu(), quantised(x, kind)) and torch.equal(v, -k)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_cache_rows_at_the_range_s_ends(ops, kind):
    import torch
    from scriptrs_amd import KvCache
    x = torch.randn(12, 2, 32, device="cuda", generator=gen(4))
    x[0] *= 3e38 / x[0].abs().amax(-1, keepdim=True)
    x[1] *= 2.0 ** -90
    x[2] *= 2.0 ** -120   # (below the least: as if 2^-96 were the largest)
    x[3] = 0.0
    x[4, 0, 7] = float("nan")
    x[5, 1, 31] = float("inf")
    x[6, 0, 0] = -float("inf")
    x[7, :, 3:] = 0.0
    x = x.bfloat16()
    plan = ops.cache_plan([0, 12], 2, 2, 32)
    cache = KvCache(1, 16, 2, 32, dtype=kind)
    table, length = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([12], dtype=torch.int32, device="cuda")
    ops.cache_write(plan, cache, table, length, x, x.flip(1))
    k, v = ops.cache_read(plan, cache, table, length, dtype=torch.float32)
    want = quantised(x, kind)
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(want)) and torch.equal(k.cpu().nan_to_num(), want.nan_to_num())
    assert torch.equal(v.nan_to_num(), k.flip(1).nan_to_num()) and int(torch.isnan(want).sum()) == 3 * 32


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_tokens_in_no_place(ops, kind):
    """Before the first token, past the table, in pages that are none of the cache's: not written, read as zeros."""
    import torch
    from scriptrs_amd import KvCache
    new, lengths = [40, 40, 40, 3, 2, 1], [25, 40, 100, 50, -7, 2_147_483_647]
    table = torch.full((6, 3), -1, dtype=torch.int32, device="cuda")
    table[0, :2] = torch.tensor([4, 0])
    table[1] = torch.tensor([1, 7, 2])                         # page 7 of 7
    table[2] = torch.tensor([5, 2_147_483_647, 6])             # (tokens 60 .. 99, the table ends at 48)
    cache = KvCache(7, 16, 2, 64, dtype=kind)
    cache.data.fill_(0x11)
    x = torch.randn(sum(new), 4, 64, device="cuda", generator=gen(5)).bfloat16()
    plan = ops.cache_plan(offsets_of(new), 2, 2, 64)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ops.cache_write(plan, cache, table, length, x[:, :2], x[:, 2:])
    k, v = ops.cache_read(plan, cache, table, length, dtype=torch.float32)
    there = torch.zeros(sum(new), dtype=torch.bool)
    there[15:40] = True                                        # sequence 0: tokens -15 .. 24
    there[40:56] = there[72:80] = True                         # sequence 1: tokens 0 .. 15 and 32 .. 39
    for got, want in ((k, quantised(x[:, :2], kind)), (v, quantised(x[:, 2:], kind))):
        assert torch.equal(got.cpu(), torch.where(there[:, None, None], want, torch.zeros_like(want)))
    for p in (3, 5, 6):
        assert (cache.data[p] == 0x11).all()


def test_cache_follows_its_lengths_in_a_graph(ops):
    """A captured step writes where the lengths say at each replay."""
    import torch
    from scriptrs_amd import KvCache
    new, page = 2, 16
    cache, other = (KvCache(12, page, 2, 64, dtype="int8") for _ in range(2))
    table = torch.tensor([[3, 1, 7, 0], [2, 11, 4, 5]], dtype=torch.int32, device="cuda")
    length = torch.tensor([2, 17], dtype=torch.int32, device="cuda")
    plan = ops.cache_plan([0, new, 2 * new], 4, 2, 64)
    kv = torch.zeros(2 * new, 4, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(2 * new, 4, 64, device="cuda", generator=gen(8)).bfloat16()
    ops.cache_write(plan, cache, table, length, kv[:, :2], kv[:, 2:])
    ops.cache_attention(plan, cache, table, length, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_write(plan, cache, table, length, kv[:, :2], kv[:, 2:])
        out = ops.cache_attention(plan, cache, table, length, q)
    cache.data.zero_()
    g = gen(9)
    for _ in range(20):
        kv.copy_(torch.randn(kv.shape, device="cuda", generator=g))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        ops.cache_write(plan, other, table, length, kv[:, :2], kv[:, 2:])
        assert torch.equal(cache.data, other.data)
        assert torch.equal(got, ops.cache_attention(plan, other, table, length, q))
        length += new


def test_cache_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput, KvCache, ModelOps
    for args in ((4, 8, 1, 64), (4, 48, 1, 64), (4, 2048, 1, 64), (4, 16, 1, 24), (4, 16, 1, 144), (4, 16, 0, 64), (-1, 16, 1, 64)):
        with pytest.raises(InvalidModelOutput):
            KvCache(*args)
    with pytest.raises(InvalidModelOutput):
        KvCache(4, 16, 1, 64, dtype="int4")
    with pytest.raises(InvalidModelOutput):
        KvCache(4, 16, 1, 64, data=torch.zeros(4, 1, 64, dtype=torch.uint8, device="cuda"))
    cache = KvCache(4, 16, 2, 64)
    plan = ops.cache_plan([0, 1, 3], 4, 2, 64)
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    inside = cache.data.view(torch.bfloat16).view(-1)[:3 * 128].view(3, 2, 64)
    closed = ops.cache_plan([0, 1], 4, 2, 64)
    closed.close()
    tall = ops.cache_plan([0, 65, 65], 4, 2, 64)
    tall_q = torch.zeros(65, 4, 64, device="cuda", dtype=torch.bfloat16)
    stranger = ModelOps()
    bad = [lambda: ops.cache_plan([1, 2], 4, 2, 64), lambda: ops.cache_plan([0, 2, 1], 4, 2, 64), lambda: ops.cache_plan([], 4, 2, 64),
           lambda: ops.cache_plan([0, 1], 3, 2, 64), lambda: ops.cache_plan([0, 1], 4, 2, 72), lambda: ops.cache_plan([0, 1 << 25], 4, 2, 64),
           lambda: ops.cache_write(plan, cache, table, n, k, k[:2]), lambda: ops.cache_write(plan, cache, table, n, k, k.half()),
           lambda: ops.cache_write(plan, cache, table, n, k[..., :32], k[..., :32]),
           lambda: ops.cache_write(plan, cache, table.long(), n, k, k), lambda: ops.cache_write(plan, cache, table[:1], n, k, k),
           lambda: ops.cache_write(plan, cache, table, n.long(), k, k), lambda: ops.cache_write(plan, cache, table, n[:1], k, k),
           lambda: ops.cache_write(plan, cache, table.t(), n, k, k), lambda: ops.cache_write(plan, cache, table.cpu(), n, k, k),
           lambda: ops.cache_write(plan, KvCache(4, 16, 1, 64), table, n, k, k), lambda: ops.cache_write(closed, cache, table[:1], n[:1], k, k),
           lambda: stranger.cache_write(plan, cache, table, n, k, k), lambda: ops.cache_write(plan, cache, table, n, inside, k),
           lambda: ops.cache_read(plan, cache, table, n, out=(k, k)), lambda: ops.cache_read(plan, cache, table, n, out=(inside, k)),
           lambda: ops.cache_read(plan, cache, table, n, dtype=torch.float64),
           lambda: ops.cache_read(plan, cache, table, n, out=(k[:1].expand(3, 2, 64), torch.empty_like(k))),
           lambda: ops.cache_attention(plan, cache, table, n, q.float()), lambda: ops.cache_attention(plan, cache, table, n, q.half()),
           lambda: ops.cache_attention(plan, cache, table, n, q[:, :2]), lambda: ops.cache_attention(plan, cache, table, n, q[:2]),
           lambda: ops.cache_attention(plan, cache, table, n, q, scale=0.0), lambda: ops.cache_attention(plan, cache, table, n, q, scale=math.inf),
           lambda: ops.cache_attention(plan, cache, table, n, q, out=q), lambda: ops.cache_attention(plan, cache, table, n, q, out=q[:2]),
           lambda: ops.cache_attention(plan, cache, table, n, q, tree=n),
           lambda: ops.cache_attention(plan, cache, table, n, q, tree=torch.zeros(2, dtype=torch.int64, device="cuda")),
           lambda: ops.cache_attention(tall, cache, table, n, tall_q, tree=torch.zeros(65, dtype=torch.int64, device="cuda"))]
    for f in bad:
        with pytest.raises(InvalidModelOutput):
            f()
    stranger.close()


# ---- attention of new tokens over the cache ---------------------------------------------


def attended(q, k, v, see, scale):
    """(out, sum of weight |v|) in 64 bits: q [rows, heads, dim], k, v [keys, kv_heads, dim], see [rows, keys]."""
    import torch
    H, K = q.shape[1], k.shape[1]
    out, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for h in range(H):
        keys, values = k[:, h // (H // K)].double(), v[:, h // (H // K)].double()
        for i in range(q.shape[0]):
            if see[i].any():
                w = torch.softmax(keys[see[i]] @ q[i, h].double() * scale, 0)
                out[i, h] = w @ values[see[i]]
                size[i, h] = w @ values[see[i]].abs()
    return out, size


def random_tree(m, rng):
    rows = []
    for i in range(m):
        parent = rng.randint(-1, i) if i else -1
        rows.append((rows[parent] if parent >= 0 else 0) | 1 << i)
    return rows


def signed(rows):
    import torch
    return torch.from_numpy(np.array([r % (1 << 64) for r in rows], np.uint64).astype(np.int64)).cuda()


def run_attention(ops, lengths, new, heads, kv_heads, dim, page, kind, dtype="bf16", tree=None, seed=0, columns=None,
                  spoil=None, scale=None, values=1.0):
    """Fills a cache, attends, and compares with 64 bits.  tree: masks of all rows, or None.  spoil(cache, table): changes
    pages' numbers and the like after the write; returns tokens [sequence][length] that are then in no place."""
    import torch
    from scriptrs_amd import KvCache
    rng = np.random.RandomState(seed)
    pages, table = paged(lengths, page, rng, columns=columns)
    cache = KvCache(pages, page, kv_heads, dim, dtype=kind)
    cache.data.fill_(0xff)  # (NaN in every type: what is not written is not looked at)
    g = gen(seed + 1)
    held = [max(0, n) for n in lengths]
    kv = torch.randn(sum(held), 2 * kv_heads, dim, device="cuda", generator=g)
    kv[:, kv_heads:] *= values
    kv = kv.to(torch_dtype(dtype))
    k, v = kv[:, :kv_heads], kv[:, kv_heads:]
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    everything = ops.cache_plan(offsets_of(held), kv_heads, kv_heads, dim)
    ops.cache_write(everything, cache, table, torch.tensor(held, dtype=torch.int32, device="cuda"), k, v)
    gone = spoil(cache, table) if spoil else [[] for _ in lengths]
    q = torch.randn(sum(new), heads, dim, device="cuda", generator=g).to(torch_dtype(dtype))
    plan = ops.cache_plan(offsets_of(new), heads, kv_heads, dim)
    got = ops.cache_attention(plan, cache, table, length, q, tree=None if tree is None else signed(tree), scale=scale)
    kq, vq = quantised(k, kind), quantised(v, kind)
    want, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    begins, rows = offsets_of(held), offsets_of(new)
    for s, (n, m) in enumerate(zip(held, new)):
        see = torch.zeros(m, n, dtype=torch.bool)
        for i in range(m):
            at = lengths[s] - m + i
            if at < 0:
                continue
            see[i, :max(0, lengths[s] - m)] = True
            for j in range(m):
                token = lengths[s] - m + j
                if token >= 0:
                    see[i, token] = (j <= i) if tree is None else bool(tree[rows[s] + i] >> j & 1)
        see[:, list(gone[s])] = False
        part = slice(rows[s], rows[s + 1])
        want[part], size[part] = attended(q[part].cpu(), kq[begins[s]:begins[s] + n], vq[begins[s]:begins[s] + n], see,
                                          scale or 1 / math.sqrt(dim))
    # a weight is rounded to 16 bits (bf16 over a cache in it, f16 elsewhere at most 2^-11 or as bf16), the output once; sums, exponentials
    # of scores below 64 and scales in f32: below 2^-13
    u = U[dtype]
    within(got, want, (2 * u + 2.0 ** -13) * size + 2.0 ** -24 * values)
    return got


KINDS = [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16"), ("int8", "bf16"), ("int8", "f16")]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 16, 16), (4, 4, 64, 16), (8, 2, 80, 32), (16, 4, 128, 64), (6, 2, 96, 128),
                                                     (16, 1, 112, 16), (32, 1, 48, 1024)])
def test_single_tokens(ops, heads, kv_heads, dim, page, kind, dtype):
    """One token over none before it up to several pages, ragged."""
    run_attention(ops, [1, 2, 15, 16, 17, 31, 33, 64, 127, 130, 517, 1031], [1] * 12, heads, kv_heads, dim, page, kind, dtype)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("m,heads,kv_heads", [(2, 4, 4), (5, 8, 2), (16, 8, 2), (64, 4, 1), (33, 6, 2)])
def test_trees(ops, m, heads, kv_heads, kind, dtype):
    rng = np.random.RandomState(m)
    new = [m, 1, 0, m, max(1, m // 2), m]
    lengths = [m, 40, 0, m + 1, 200, 700 + m]
    tree = sum((random_tree(x, rng) for x in new), [])
    tree[0] = 0                 # sees the context alone: here none
    tree[-1] |= 1 << 63         # (a bit past the last new token counts for nothing unless there are 64)
    if m == 64:
        tree[-1] = 1 << 63
    run_attention(ops, lengths, new, heads, kv_heads, 64, 16, kind, dtype, tree=tree)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("m", [2, 7, 100, 300])
def test_runs_of_tokens(ops, m, kind, dtype):
    run_attention(ops, [m, 300, m + 65, 3], [m, 1, m, 3], 4, 2, 64, 32, kind, dtype)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_sequences_shorter_than_their_new_tokens(ops, kind, dtype):
    """Tokens before the first are none: their rows see nothing, and none sees them; empty and negative lengths."""
    rng = np.random.RandomState(3)
    run_attention(ops, [3, 0, 1, -5, 40], [5, 4, 1, 2, 5], 4, 2, 64, 16, kind, dtype)
    run_attention(ops, [3, 0, 1, -5, 40], [5, 4, 1, 2, 5], 4, 2, 64, 16, kind, dtype,
                  tree=sum((random_tree(x, rng) for x in (5, 4, 1, 2, 5)), []))


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_pages_that_are_none(ops, kind, dtype):
    """Tokens in such pages and past the table are seen by nobody."""
    def spoil(cache, table):
        table[0, 1] = -1
        table[1, 0] = cache.pages
        table[1, 3] = 2_147_483_647
        table[2, :] = -3
        return [range(16, 32), list(range(16)) + list(range(48, 64)), range(70), [], []]
    run_attention(ops, [50, 100, 70, 20, 40], [1, 3, 2, 1, 1], 4, 2, 64, 16, kind, dtype, spoil=spoil)


def test_long_sequences_are_cut(ops):
    """More keys than one workgroup takes, of few and of many sequences."""
    run_attention(ops, [9000], [1], 4, 2, 64, 64, "e4m3")
    run_attention(ops, [5000, 1, 3333, 0], [2, 1, 2, 1], 2, 2, 128, 16, "int8")
    run_attention(ops, [4097, 2900], [16, 16], 4, 1, 64, 32, "bf16", tree=random_tree(16, np.random.RandomState(1)) * 2)


def test_long_runs_of_new_tokens(ops):
    """A prompt's second chunk: many tiles of 128 rows, whole and in shares."""
    run_attention(ops, [900], [600], 8, 2, 64, 32, "int8")
    run_attention(ops, [5000, 10], [40, 3], 8, 2, 128, 64, "e4m3", columns=400)
    run_attention(ops, [150] * 40, [140] * 40, 8, 8, 32, 16, "bf16", columns=1000)


def test_a_cache_keeps_its_memory():
    from scriptrs_amd import KvCache
    cache = KvCache(2, 16, 1, 16)
    with pytest.raises(AttributeError):
        cache.data = cache.data.clone()


def test_caches_past_4_gib(ops):
    """Pages whose places pass 32 bits."""
    import torch
    from scriptrs_amd import KvCache
    K, D, page, n = 8, 128, 64, 150
    for kind in ("bf16", "int8"):
        pages = (5 << 30) // (K * (2 * page * D * (2 if kind == "bf16" else 1)))
        cache = KvCache(pages, page, K, D, dtype=kind)
        assert cache.data.numel() > 1 << 32
        table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        kv = torch.randn(n, 2 * K, D, device="cuda", generator=gen(1)).bfloat16()
        whole = ops.cache_plan([0, n], K, K, D)
        ops.cache_write(whole, cache, table, length, kv[:, :K], kv[:, K:])
        k, v = ops.cache_read(whole, cache, table, length, dtype=torch.float32)
        kq, vq = quantised(kv[:, :K], kind), quantised(kv[:, K:], kind)
        assert torch.equal(k.cpu(), kq) and torch.equal(v.cpu(), vq)
        q = torch.randn(1, 2 * K, D, device="cuda", generator=gen(2)).bfloat16()
        got = ops.cache_attention(ops.cache_plan([0, 1], 2 * K, K, D), cache, table, length, q)
        want, size = attended(q.cpu(), kq, vq, torch.ones(1, n, dtype=torch.bool), D ** -0.5)
        within(got, want, (2 * U["bf16"] + 2.0 ** -13) * size)
        del cache


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_hidden_values_that_are_not_finite(ops, kind, dtype):
    """NaN and infinities of drafts that a row does not see reach nothing; those that it sees do."""
    import torch
    from scriptrs_amd import KvCache
    m, context, K, D = 6, 45, 2, 64
    rng = np.random.RandomState(5)
    tree = random_tree(m, rng)
    tree[5] = 1 << 5
    bad = 3
    tree = [t if i in (bad, 4) else t & ~(1 << bad) for i, t in enumerate(tree)]
    tree[4] |= 1 << bad
    cache = KvCache(8, 16, K, D, dtype=kind)
    table = torch.tensor([[1, 5, 2, 7]], dtype=torch.int32, device="cuda")
    length = torch.tensor([context + m], dtype=torch.int32, device="cuda")
    g = gen(6)
    kv = torch.randn(context + m, 2 * K, D, device="cuda", generator=g).to(torch_dtype(dtype))
    q = torch.randn(m, 4, D, device="cuda", generator=g).to(torch_dtype(dtype))
    whole, plan = ops.cache_plan([0, context + m], K, K, D), ops.cache_plan([0, m], 4, K, D)
    ops.cache_write(whole, cache, table, length, kv[:, :K], kv[:, K:])
    clean = ops.cache_attention(plan, cache, table, length, q, tree=signed(tree))
    for value in (math.nan, math.inf, -math.inf):
        spoiled = kv.clone()
        spoiled[context + bad, K:, 3] = value      # of V alone
        ops.cache_write(whole, cache, table, length, spoiled[:, :K], spoiled[:, K:])
        got = ops.cache_attention(plan, cache, table, length, q, tree=signed(tree))
        for i in range(m):
            if i in (bad, 4):
                if kind in TOP:
                    assert got[i].isnan().all()
                else:
                    assert not got[i, :, 3].isfinite().any() and (math.isnan(value) or torch.equal(got[i, :, 3], torch.full_like(got[i, :, 3], value)))
                    assert torch.equal(got[i, :, 4:], clean[i, :, 4:])
            else:
                assert torch.equal(got[i], clean[i]), i
        spoiled[context + bad, :K, 1] = value      # of K too
        ops.cache_write(whole, cache, table, length, spoiled[:, :K], spoiled[:, K:])
        got = ops.cache_attention(plan, cache, table, length, q, tree=signed(tree))
        for i in range(m):
            if i not in (bad, 4):
                assert torch.equal(got[i], clean[i]), i


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_rows_do_not_touch_each_other(ops, kind, dtype):
    """Queries that are not finite, far larger or far smaller than others leave the others' results as they are."""
    import torch
    from scriptrs_amd import KvCache
    K, D = 2, 64
    for m in (2, 20):
        n = 150 + m
        cache = KvCache(11, 16, K, D, dtype=kind)
        table, length = torch.arange(11, device="cuda", dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32, device="cuda")
        kv = torch.randn(n, 2 * K, D, device="cuda", generator=gen(m)).to(torch_dtype(dtype))
        ops.cache_write(ops.cache_plan([0, n], K, K, D), cache, table, length, kv[:, :K], kv[:, K:])
        plan = ops.cache_plan([0, m], 4, K, D)
        q = torch.randn(m, 4, D, device="cuda", generator=gen(m + 1)).to(torch_dtype(dtype))
        want = ops.cache_attention(plan, cache, table, length, q)
        for value in (math.nan, math.inf, 60000.0 if dtype == "f16" else 3e38, 1e-7 if dtype == "f16" else 1e-38):
            other = q.clone()
            other[1, 2] = value
            got = ops.cache_attention(plan, cache, table, length, other)
            keep = torch.ones(m, 4, dtype=torch.bool, device="cuda")
            keep[1, 2] = False
            assert torch.equal(got[keep], want[keep]), (m, value)
            if abs(value) < 1e-3:  # (all scores alike)
                mean = quantised(kv[:150 + 2, K:], kind).double().mean(0)[1]
                size = quantised(kv[:150 + 2, K:], kind).double().abs().mean(0)[1]
                within(got[1, 2], mean, (2 * U[dtype] + 2.0 ** -13) * size)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_scores_and_values_far_from_one(ops, kind, dtype):
    run_attention(ops, [200, 700], [1, 2], 4, 2, 64, 32, kind, dtype, scale=1e-6)
    run_attention(ops, [200, 700], [1, 2], 4, 2, 64, 32, kind, dtype, values=2e-4)
    run_attention(ops, [200, 700], [1, 2], 4, 2, 64, 32, kind, dtype, values=500.0)
    if dtype == "bf16":
        run_attention(ops, [200, 700], [1, 2], 4, 2, 64, 32, kind, dtype, values=1e30)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_values_of_very_different_scales(ops, kind, dtype):
    """The largest values are the last ones: sums of small ones before them lose nothing that counts."""
    import torch
    from scriptrs_amd import KvCache
    n, K, D = 600, 2, 64
    kv = torch.randn(n, 2 * K, D, device="cuda", generator=gen(7))
    size = torch.logspace(-3, 3, n, device="cuda")
    kv[:, K:] *= size[:, None, None]
    kv = kv.to(torch_dtype(dtype))
    q = torch.randn(1, 4, D, device="cuda", generator=gen(8)).to(torch_dtype(dtype))
    for order in (torch.arange(n), torch.arange(n - 1, -1, -1), torch.randperm(n, generator=torch.Generator().manual_seed(1))):
        x = kv[order.cuda()]
        cache = KvCache(10, 64, K, D, dtype=kind)
        table, length = torch.arange(10, device="cuda", dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32, device="cuda")
        ops.cache_write(ops.cache_plan([0, n], K, K, D), cache, table, length, x[:, :K], x[:, K:])
        got = ops.cache_attention(ops.cache_plan([0, 1], 4, K, D), cache, table, length, q)
        want, weight = attended(q.cpu(), quantised(x[:, :K], kind), quantised(x[:, K:], kind), torch.ones(1, n, dtype=torch.bool), D ** -0.5)
        within(got, want, (2 * U[dtype] + 2.0 ** -13) * weight)


def test_large_scores_and_ties(ops):
    """One key far above the rest, and all alike."""
    import torch
    from scriptrs_amd import KvCache
    n, D = 100, 64
    k = torch.zeros(n, 1, D, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n, 1, D, device="cuda", generator=gen(9)).bfloat16()
    q = torch.ones(1, 1, D, device="cuda", dtype=torch.bfloat16)
    table, length = torch.arange(7, device="cuda", dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    whole, one = ops.cache_plan([0, n], 1, 1, D), ops.cache_plan([0, 1], 1, 1, D)
    for kind in ("bf16", "int8"):
        cache = KvCache(7, 16, 1, D, dtype=kind)
        ops.cache_write(whole, cache, table, length, k, v)
        got = ops.cache_attention(one, cache, table, length, q)
        values = quantised(v, kind).double()
        within(got, values.mean(0, keepdim=True), (2 * U["bf16"] + 2.0 ** -13) * values.abs().mean(0, keepdim=True))
        k2 = k.clone()
        k2[77] = 1000.0
        ops.cache_write(whole, cache, table, length, k2, v)
        got = ops.cache_attention(one, cache, table, length, q)
        within(got, values[77:78], 2 * U["bf16"] * values[77:78].abs())


def test_attention_rows_past_the_last_and_views(ops):
    import torch
    from scriptrs_amd import KvCache
    cache = KvCache(6, 16, 2, 64, dtype="int8")
    table, length = torch.arange(6, device="cuda", dtype=torch.int32)[None], torch.tensor([90], dtype=torch.int32, device="cuda")
    kv = torch.randn(90, 4, 64, device="cuda", generator=gen(1)).bfloat16()
    ops.cache_write(ops.cache_plan([0, 90], 2, 2, 64), cache, table, length, kv[:, :2], kv[:, 2:])
    plan = ops.cache_plan([0, 3], 4, 2, 64)
    wide = torch.randn(5, 8, 80, device="cuda", generator=gen(2)).bfloat16()
    q = wide[:, ::2, 8:72]
    want = ops.cache_attention(plan, cache, table, length, q[:3].contiguous())
    got = ops.cache_attention(plan, cache, table, length, q)
    assert torch.equal(got[:3], want) and not got[3:].any()
    out = torch.full((5, 4, 72), 7.0, device="cuda", dtype=torch.bfloat16)
    assert ops.cache_attention(plan, cache, table, length, q, out=out[..., :64]).shape == (5, 4, 64)
    assert torch.equal(out[:3, :, :64], want) and not out[3:, :, :64].any() and (out[..., 64:] == 7.0).all()
    wide_table = torch.full((1, 20), -1, dtype=torch.int32, device="cuda")
    wide_table[:, 4:10] = table
    assert torch.equal(ops.cache_attention(plan, cache, wide_table[:, 4:], length, q[:3]), want)
    none = ops.cache_plan([0, 0], 4, 2, 64)
    assert not ops.cache_attention(none, cache, table, length, q).any()
    assert ops.cache_attention(none, cache, table, length, q[:0]).shape == (0, 4, 64)


def test_calls_on_another_stream(ops):
    import torch
    from scriptrs_amd import KvCache
    side = torch.cuda.Stream()
    for _ in range(5):
        cache = KvCache(40, 16, 2, 64, dtype="e4m3")
        table, length = torch.arange(40, device="cuda", dtype=torch.int32)[None], torch.tensor([600], dtype=torch.int32, device="cuda")
        kv = torch.randn(600, 4, 64, device="cuda", generator=gen(1)).bfloat16()
        q = torch.randn(2, 4, 64, device="cuda", generator=gen(2)).bfloat16()
        logits = torch.randn(8, 5000, device="cuda", generator=gen(3))
        whole, plan = ops.cache_plan([0, 600], 2, 2, 64), ops.cache_plan([0, 2], 4, 2, 64)
        side.wait_stream(torch.cuda.current_stream())
        ops.cache_write(whole, cache, table, length, kv[:, :2], kv[:, 2:], stream=side)
        out = ops.cache_attention(plan, cache, table, length, q, stream=side)
        k, v = ops.cache_read(whole, cache, table, length, stream=side)
        z = ops.adjust_logits(logits, bias=torch.ones(5000, device="cuda"), stream=side)
        del q
        torch.empty(1 << 20, device="cuda").fill_(3.0)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(k.cpu().float(), quantised(kv[:, :2], "e4m3").bfloat16().float())
        q = torch.randn(2, 4, 64, device="cuda", generator=gen(2)).bfloat16()
        assert torch.equal(out, ops.cache_attention(plan, cache, table, length, q))
        assert torch.equal(z, logits + 1.0)


# ---- steering of logits ---------------------------------------------------------------------


def steered(z, history, lengths, repetition, presence, frequency, bias, allowed, states):
    import torch
    rows, vocab = z.shape
    z = z.cpu().double().clone()
    for r in range(rows):
        if history is not None:
            said = history[r].cpu() if lengths is None else history[r, :max(0, int(lengths[r]))].cpu()
            for t, c in zip(*torch.unique(said, return_counts=True)):
                t = int(t)
                if 0 <= t < vocab:
                    rep, pre, fre = (float(x[r]) if isinstance(x, torch.Tensor) else float(np.float32(x)) for x in (repetition, presence, frequency))
                    z[r, t] = (z[r, t] / rep if z[r, t] > 0 else z[r, t] * rep) - pre - fre * int(c)
        if bias is not None:
            z[r] += (bias if bias.dim() == 1 else bias[r]).cpu().double()
        if allowed is not None:
            state = int(states[r]) if states is not None else r
            if 0 <= state < len(allowed):
                words = allowed[state].cpu().numpy().astype(np.uint32)
                bits = torch.from_numpy((words[:, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(-1)[:vocab].astype(bool))
                z[r, ~bits] = -math.inf
    return z


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 4096, 9001, 40_003])
@pytest.mark.parametrize("what", ["history", "bias", "mask", "all", "none"])
def test_adjust_logits(ops, what, vocab, dtype):
    import torch
    g = gen(vocab)
    for rows in (1, 7):
        logits = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(torch_dtype(dtype))
        args = dict(history=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None, states=None)
        if what in ("history", "all"):
            args["history"] = torch.randint(-2, min(vocab + 2, 60), (rows, 300), device="cuda", generator=g).int()
            args["history"][:, 250:] = torch.randint(0, vocab, (rows, 50), device="cuda", generator=g).int()
            args["repetition"], args["presence"], args["frequency"] = 1.3, 0.25, 0.0625
        if what == "all":
            args["lengths"] = torch.randint(0, 301, (rows,), device="cuda", generator=g).int()
            args["lengths"][0], args["lengths"][-1] = 300, 1000  # (more than there are: all)
            args["repetition"] = 1 + torch.rand(rows, device="cuda", generator=g)
            args["frequency"] = torch.rand(rows, device="cuda", generator=g) / 8
        if what in ("bias", "all"):
            args["bias"] = torch.randn(*((vocab,) if what == "all" else (rows, vocab)), device="cuda", generator=g)
        if what in ("mask", "all"):
            masks = rows if what == "mask" else 3
            args["allowed"] = torch.randint(-(1 << 31), 1 << 31, (masks, (vocab + 31) // 32), device="cuda", generator=g).int()
            if what == "all":
                args["states"] = torch.randint(-1, 5, (rows,), device="cuda", generator=g).int()
        want = steered(logits, **args)
        got = ops.adjust_logits(logits, **args)
        assert got.dtype == logits.dtype
        # f32: up to 6 roundings of values below 64, and the output's own
        finite = torch.where(torch.isfinite(want), want.abs(), torch.zeros_like(want))
        within(got, want, U[dtype] * finite + 6 * 2.0 ** -24 * 64)
        again = logits.clone()
        assert ops.adjust_logits(again, **args, out=again) is again and torch.equal(again, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_of_other_rows(ops, dtype):
    """Rows within larger ones, at every alignment, into an output that lies alike or not."""
    import torch
    vocab = 2500
    wide = torch.randn(5, vocab + 37, device="cuda", generator=gen(1)).to(torch_dtype(dtype))
    history = torch.randint(0, vocab, (5, 64), device="cuda", generator=gen(2)).int()
    allowed = torch.randint(-(1 << 31), 1 << 31, (5, 90), device="cuda", generator=gen(3)).int()
    for at in (0, 1, 2, 3, 5, 8, 16, 37):
        x = wide[:, at:at + vocab]
        want = ops.adjust_logits(x.contiguous(), history=history, frequency=0.5, allowed=allowed)
        for other in (at, 0, 7):
            out = torch.full_like(wide, 9.0)
            ops.adjust_logits(x, history=history, frequency=0.5, allowed=allowed, out=out[:, other:other + vocab])
            assert torch.equal(out[:, other:other + vocab], want)
            assert (out[:, :other] == 9.0).all() and (out[:, other + vocab:] == 9.0).all()
    one = wide[:1, :vocab].expand(5, vocab)  # (one row for all)
    assert torch.equal(ops.adjust_logits(one, history=history, presence=1.0),
                       ops.adjust_logits(one.contiguous(), history=history, presence=1.0))


def test_logits_that_are_not_finite(ops):
    import torch
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0, math.nan, -2.0, 0.0, 3.0]], device="cuda")
    history = torch.tensor([[0, 1, 2, 5, 6]], dtype=torch.int32, device="cuda")
    allowed = torch.tensor([[0b11101111]], dtype=torch.int32, device="cuda")
    got = ops.adjust_logits(x, history=history, repetition=2.0, allowed=allowed)[0].tolist()
    assert got[:2] == [math.inf, -math.inf] and math.isnan(got[2]) and got[3:] == [1.0, -math.inf, -4.0, 0.0, 3.0]


def test_a_mask_of_nothing_leaves_no_candidate(ops):
    """A grammar's dead end: all -inf, which beam search takes as no candidate."""
    import torch
    logits = torch.randn(4, 1025, device="cuda", generator=gen(1))
    allowed = torch.zeros(1, 33, dtype=torch.int32, device="cuda")
    states = torch.tensor([0, -1, 0, -1], dtype=torch.int32, device="cuda")
    z = ops.adjust_logits(logits, allowed=allowed, states=states)
    assert torch.isinf(z[::2]).all() and torch.equal(z[1::2], logits[1::2])
    scores, parents, tokens, _ = ops.beam_select(z, torch.zeros(2, 2, device="cuda"))
    assert (parents == 1).all() and (tokens >= 0).all()


def test_adjust_logits_in_a_graph(ops):
    import torch
    x = torch.randn(6, 9001, device="cuda", generator=gen(1)).bfloat16()
    history = torch.zeros(6, 100, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(6, dtype=torch.int32, device="cuda")
    ops.adjust_logits(x, history=history, lengths=lengths, repetition=1.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adjust_logits(x, history=history, lengths=lengths, repetition=1.5)
    for step in range(5):
        history[:, step] = torch.randint(0, 9001, (6,), device="cuda", generator=gen(step)).int()
        lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.adjust_logits(x, history=history, lengths=lengths, repetition=1.5))


def test_adjust_logits_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput
    x = torch.zeros(4, 100, device="cuda")
    h = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    masks = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    big = torch.zeros(8, 100, device="cuda")
    bad = [lambda: ops.adjust_logits(x[0]), lambda: ops.adjust_logits(x.double()), lambda: ops.adjust_logits(x.cpu()),
           lambda: ops.adjust_logits(x.t()), lambda: ops.adjust_logits(x, history=h.long()), lambda: ops.adjust_logits(x, history=h[:3]),
           lambda: ops.adjust_logits(x, lengths=n), lambda: ops.adjust_logits(x, history=h, lengths=n[:3]),
           lambda: ops.adjust_logits(x, history=h, lengths=n.long()), lambda: ops.adjust_logits(x, history=h, repetition=0.0),
           lambda: ops.adjust_logits(x, history=h, repetition=-1.0), lambda: ops.adjust_logits(x, history=h, repetition=math.nan),
           lambda: ops.adjust_logits(x, history=h, presence=math.inf), lambda: ops.adjust_logits(x, history=h, repetition=n),
           lambda: ops.adjust_logits(x, bias=x[0, :50]), lambda: ops.adjust_logits(x, bias=x[:2]), lambda: ops.adjust_logits(x, bias=x.half()),
           lambda: ops.adjust_logits(x, allowed=masks[:, :3]), lambda: ops.adjust_logits(x, allowed=masks[:3]),
           lambda: ops.adjust_logits(x, states=n), lambda: ops.adjust_logits(x, allowed=masks, states=n.long()),
           lambda: ops.adjust_logits(x, out=x.half()), lambda: ops.adjust_logits(big[:4], out=big[1:5]),
           lambda: ops.adjust_logits(x, out=x[:1].expand(4, 100)), lambda: ops.adjust_logits(x, bias=x, out=x)]
    for f in bad:
        with pytest.raises(InvalidModelOutput):
            f()
    assert ops.adjust_logits(x[:0]).shape == (0, 100)
    assert torch.equal(ops.adjust_logits(x, history=h[:, :0], lengths=n, repetition=2.0), x)
    assert torch.equal(ops.adjust_logits(x, allowed=masks[:0], states=n), x)
