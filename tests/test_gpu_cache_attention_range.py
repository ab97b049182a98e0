"""Attention over a paged cache at the ends of what its types hold, against 64 bits: value scales far apart, the
largest values, scores far from one and past f32."""
import math

import pytest

pytestmark = pytest.mark.gpu

from test_gpu_decode import KINDS, TOP, U, attended, gen, ops, quantised, torch_dtype, within  # noqa: E402, F401

CODED = [x for x in KINDS if x[0] in TOP]


def filled(ops, k, v, kind, page=16):  # noqa: F811
    """A cache of one sequence's k, v [tokens, kv_heads, dim], its page table and length."""
    import torch
    from scriptrs_amd import KvCache
    n, K, D = k.shape
    cache = KvCache(-(-n // page), page, K, D, dtype=kind)
    table = torch.arange(cache.pages, device="cuda", dtype=torch.int32).flip(0)[None].contiguous()
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    ops.cache_write(ops.cache_plan([0, n], K, K, D), cache, table, length, k, v)
    return cache, table, length


def attend(ops, q, held, K, scale=None, tree=None):  # noqa: F811
    rows, H, D = q.shape
    return ops.cache_attention(ops.cache_plan([0, rows], H, K, D), *held, q, tree=tree, scale=scale)


def chain(rows, n):
    """What each of the last `rows` of n tokens sees."""
    import torch
    return torch.arange(n)[None] <= torch.arange(n - rows, n)[:, None]


@pytest.mark.parametrize("kind,dtype", CODED)
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("ratio", [2.0 ** 20, 2.0 ** 26, 2.0 ** 30, 2.0 ** 60])
def test_a_large_value_of_next_to_no_weight(ops, ratio, rising, kind, dtype):  # noqa: F811
    """A token that a row sees with a weight of e^-60 of the rest, and values far above theirs: what the others' weights add up
    to keeps its bits, wherever the token is.  rising: the others' scores rise by 80 on the way, so that the first of them weigh as
    little."""
    import torch
    n, D = 256, 64
    g = gen(3)
    q = torch.randint(0, 2, (1, 2, D), device="cuda", generator=g).mul_(2).sub_(1).to(torch_dtype(dtype))
    q[0, 1] = q[0, 0]
    k = torch.randn(n, 1, D, device="cuda", generator=g)
    if rising:
        k += q[:, :1].float() * (torch.arange(n, device="cuda") * (80.0 / n / math.sqrt(D)))[:, None, None]
    v = torch.randn(n, 1, D, device="cuda", generator=g)
    for at in (0, 1, 40, 250, n - 1):
        far, large = k.clone(), v.clone()
        far[at, 0] = -60.0 / math.sqrt(D) * q[0, 0].float()
        large[at] *= ratio
        got = attend(ops, q, filled(ops, far, large, kind), 1)
        want, size = attended(q.cpu(), quantised(far, kind), quantised(large, kind), torch.ones(1, n, dtype=torch.bool), D ** -0.5)
        assert size.max() < 8
        # (two roundings to 16 bits, and f32's)
        within(got, want, (2 * U[dtype] + 2.0 ** -13) * size)


@pytest.mark.parametrize("kind", ["bf16", *sorted(TOP)])
@pytest.mark.parametrize("n,rows", [(1000, 1), (1000, 3), (700, 40), (20_000, 2)])
def test_the_largest_values(ops, n, rows, kind):  # noqa: F811
    """Means of values up to the largest of bf16 are no larger than they are, however many: no sum on the way is infinite."""
    import torch
    D = 64
    g = gen(4)
    v = ((0.5 + 0.5 * torch.rand(n, 2, D, device="cuda", generator=g)) * 3.3e38).bfloat16()
    v[..., ::2] *= -1
    q = (0.1 * torch.randn(rows, 4, D, device="cuda", generator=g)).bfloat16()
    k = torch.randn(n, 2, D, device="cuda", generator=g).bfloat16()
    got = attend(ops, q, filled(ops, k, v, kind), 2)
    want, size = attended(q.cpu(), quantised(k, kind), quantised(v, kind), chain(rows, n), D ** -0.5)
    within(got, want, (2 * U["bf16"] + 2.0 ** -13) * size)


@pytest.mark.parametrize("kind", ["bf16", *sorted(TOP)])
def test_small_values(ops, kind):  # noqa: F811
    """Values down to 2^-90 keep their bits, alone and behind large weights."""
    import torch
    n, D = 700, 64
    g = gen(7)
    k, v = torch.randn(n, 2, D, device="cuda", generator=g).bfloat16(), torch.randn(n, 2, D, device="cuda", generator=g) * 2.0 ** -90
    v = (v.sign() * v.abs().clamp(min=2.0 ** -94)).bfloat16()
    for gain in (0.1, 8.0):
        q = (gain * torch.randn(3, 4, D, device="cuda", generator=g)).bfloat16()
        got = attend(ops, q, filled(ops, k, v, kind), 2)
        want, size = attended(q.cpu(), quantised(k, kind), quantised(v, kind), chain(3, n), D ** -0.5)
        # (gain 8: scores of up to 40, whose f32 error is 2^-24 of the sum of 64 products' magnitudes)
        within(got, want, (2 * U["bf16"] + 2.0 ** -13) * size)


@pytest.mark.parametrize("kind", ["bf16", *sorted(TOP)])
def test_the_largest_values_of_many_sequences(ops, kind):  # noqa: F811
    """As above, each workgroup over all of a sequence's 4,000 tokens."""
    import torch
    n, seqs, D = 4000, 300, 64
    g = gen(8)
    k, v = torch.randn(n, 1, D, device="cuda", generator=g).bfloat16(), torch.full((n, 1, D), 3e38, device="cuda").bfloat16()
    cache, table, length = filled(ops, k, v, kind)
    q = (0.1 * torch.randn(seqs, 2, D, device="cuda", generator=g)).bfloat16()
    plan = ops.cache_plan(list(range(seqs + 1)), 2, 1, D)
    got = ops.cache_attention(plan, cache, table.expand(seqs, -1), length.expand(seqs).contiguous(), q)
    want = quantised(v[:1], kind).double().expand(seqs, 2, D)
    within(got, want, (2 * U["bf16"] + 2.0 ** -13) * want.abs())


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_scores_past_f32(ops, kind, dtype):  # noqa: F811
    """A row whose scores are infinite in f32 is NaN, and not zeros as of a row that sees nothing; others keep theirs.  bf16: queries of
    1e36 and keys of 1e4, whose 64 products of either sign add up to 1e40; f16: 6e4 and 1e4 make 1e9, and the scale 1e39."""
    import torch
    n, D = 200, 64
    g = gen(5)
    kv = torch.randn(n, 2, D, device="cuda", generator=g)
    kv[:, 0] *= 1e4
    kv = kv.to(torch_dtype(dtype))
    held = filled(ops, kv[:, :1], kv[:, 1:], kind)
    scale = 1e30 if dtype == "f16" else None
    for m in (2, 20):
        q = torch.randn(m, 2, D, device="cuda", generator=g).to(torch_dtype(dtype))
        want = attend(ops, q, held, 1, scale=scale)
        large = q.clone()
        large[1, 1] = 60000.0 if dtype == "f16" else 1e36
        got = attend(ops, large, held, 1, scale=scale)
        keep = torch.ones(m, 2, dtype=torch.bool, device="cuda")
        keep[1, 1] = False
        assert torch.equal(got[keep], want[keep])
        assert got[1, 1].isnan().all()
        if kind in TOP:  # (codes' products stay in range: a scale that brings their sum back does)
            assert attend(ops, large, held, 1, scale=1e-9 if dtype == "bf16" else 1.0)[1, 1].isfinite().all()


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("scale", [2.0 ** 20, 1e25, 1e30])
def test_scores_far_past_one(ops, scale, kind, dtype):  # noqa: F811
    """Whole numbers as keys and queries, which every type holds (the largest magnitude is the largest code): scores are exact up to the
    scale, differ by a scale at least, and so a row is the mean of its best keys' values."""
    import torch
    n, D = 300, 64
    rng = torch.Generator().manual_seed(6)
    k = torch.randint(-4, 5, (n, 1, D), generator=rng).float() * 16
    k[..., 0] = TOP.get(kind, 448.0)
    if kind == "int8":
        k[..., 1:] /= 8
    k[200:220] = k[30:50]  # (ties)
    v = torch.randn(n, 1, D, generator=rng)
    for m in (1, 20):
        q = torch.randint(-2, 3, (m, 2, D), generator=rng).to(torch_dtype(dtype))
        held = filled(ops, k.cuda(), v.cuda(), kind)
        got = attend(ops, q.cuda(), held, 1, scale=scale)
        kq, vq, see = quantised(k, kind), quantised(v, kind).double(), chain(m, n)
        assert torch.equal(kq, k)
        want, size = torch.zeros(m, 2, D, dtype=torch.float64), torch.zeros(m, 2, D, dtype=torch.float64)
        for i in range(m):
            for h in range(2):
                s = torch.where(see[i], k[:, 0].double() @ q[i, h].double(), torch.tensor(-math.inf, dtype=torch.float64))
                best = vq[s == s.max(), 0]
                want[i, h], size[i, h] = best.mean(0), best.abs().mean(0)
        within(got, want, (2 * U[dtype] + 2.0 ** -13) * size)


@pytest.mark.parametrize("kind", sorted(TOP))
def test_scores_of_large_queries_and_few_channels(ops, kind):  # noqa: F811
    """Keys of one channel, queries that are all large: a score has the bits of its one product, whatever the channels without a
    part in it.  Scores of 1,000 that differ by a few: 3 roundings of f32 (product, key's scale, scale of the logarithm) of 1,445 each."""
    import torch
    n, D = 6, 128
    rng = torch.Generator().manual_seed(9)
    k, v = torch.zeros(n, 1, D), torch.randn(n, 1, D, generator=rng)
    k[torch.arange(n), 0, torch.arange(n) * 20 + 3] = 1.0
    for m in (1, 20):
        q = 1000 + 0.5 * torch.randint(0, 6, (m, 2, D), generator=rng)
        held = filled(ops, k.cuda(), v.cuda(), kind)
        got = ops.cache_attention(ops.cache_plan([0, m], 2, 1, D), held[0], held[1], held[2], q.half().cuda(),
                                  tree=torch.full((m,), (1 << m) - 1 if m > 1 else 1, dtype=torch.int64, device="cuda"), scale=1.0)
        see = torch.ones(m, n, dtype=torch.bool)
        if m > n:  # (new tokens before the first are none, and see nothing)
            see[:m - n] = False
        want, size = attended(q, k, quantised(v, kind), see, 1.0)
        within(got, want, (2 * U["f16"] + 2.0 ** -13 + 2 * 3 * 2.0 ** -24 * 1445) * size)


@pytest.mark.parametrize("kind", ["bf16", *sorted(TOP)])
@pytest.mark.parametrize("large", [1e13, 1e30])
def test_queries_of_very_different_channels(ops, large, kind):  # noqa: F811
    """A channel of the queries far above the others, where all keys are zero, takes nothing from the others' part in the scores."""
    import torch
    n, D = 150, 64
    g = gen(10)
    k, v = (torch.randn(n, 1, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    k[..., 5] = 0.0
    held = filled(ops, k, v, kind)
    for m in (1, 20):
        q = torch.randn(m, 2, D, device="cuda", generator=g).bfloat16()
        want = attend(ops, q, held, 1)
        q[..., 5] = large
        got = attend(ops, q, held, 1)
        assert torch.equal(got, want)
        exact, size = attended(q.cpu(), quantised(k, kind), quantised(v, kind), chain(m, n), D ** -0.5)
        within(got, exact, (2 * U["bf16"] + 2.0 ** -13) * size)
