"""The packed attention's tiles of 128 and 256 rows against a plain computation in 64 bits.

Small calls go through tiles of 16 rows as a whole, so each case here is joined by short sequences enough
that it does not.  The tolerance is the one of the small cases: an ulp of the output's type for
its own rounding, another of the weights times |v| for the weights' rounding, and 1e-4 of the weights
times |v| for the f32 scores and exponentials (scores of up to about 30)."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TYPES = {"bf16": "bfloat16", "f16": "float16"}


@pytest.fixture(scope="module")
def ops():
    from scriptrs_amd import ModelOps
    m = ModelOps()
    yield m
    m.close()


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def plain(q, k, v, qo, ko, left, right, mask, scale):
    """(result, sum of weights times |v|) in 64 bits; hidden keys are left out, not multiplied by zero."""
    import torch
    H, K = q.shape[1], k.shape[1]
    out, mag = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for s in range(len(qo) - 1):
        lq, lk = qo[s + 1] - qo[s], ko[s + 1] - ko[s]
        if lq == 0 or lk == 0:
            continue
        i = torch.arange(lq, device=q.device)[:, None] + lk - lq
        j = torch.arange(lk, device=q.device)[None, :]
        see = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        if left >= 0:
            see &= j >= i - left
        if right >= 0:
            see &= j <= i + right
        if mask is not None:
            see &= mask[ko[s]:ko[s + 1]][None, :]
        seen = see.any(0)[:, None]
        for h in range(H):
            kk, vv = (t[ko[s]:ko[s + 1], h * K // H].double() for t in (k, v))
            x = q[qo[s]:qo[s + 1], h].double() @ torch.where(seen, kk, 0.0).T * scale
            x = torch.where(see, x, -math.inf)
            top = x.amax(1, keepdim=True)
            p = torch.where(see, (x - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            finite = torch.isfinite(vv)
            r = p @ torch.where(finite, vv, 0.0)
            if not bool((finite | ~seen).all()):
                # what is not finite reaches exactly the queries that see it
                up, down, none = ((see.double() @ m.double()) > 0
                                  for m in (vv == math.inf, vv == -math.inf, torch.isnan(vv)))
                r = torch.where(up, math.inf, r)
                r = torch.where(down, -math.inf, r)
                r = torch.where(none | (up & down), math.nan, r)
            out[qo[s]:qo[s + 1], h] = r
            mag[qo[s]:qo[s + 1], h] = p @ torch.where(finite, vv, 0.0).abs()
    return out, mag


FILL = [17, 33, 5, 48] * 24  # 240 tiles of 16 rows a kv head, group of 1


def tensors(lq, lk, heads, kv_heads, dim, dtype, seed):
    import torch
    t = getattr(torch, TYPES[dtype])
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(sum(lq) + sum(FILL), heads, dim, device="cuda", generator=g).to(t)
    k, v = (torch.randn(sum(lk) + sum(FILL), kv_heads, dim, device="cuda", generator=g).to(t) for _ in range(2))
    return q, k, v


def check(ops, lq, lk, heads, kv_heads, dim, dtype="bf16", left=-1, right=-1, mask=None, seed=0, qkv=None):
    import torch
    q, k, v = tensors(lq, lk, heads, kv_heads, dim, dtype, seed) if qkv is None else qkv
    qo, ko = offsets(lq + FILL), offsets(lk + FILL)
    plan = ops.attention_plan(qo, ko, heads, kv_heads, dim, left=left, right=right)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    ops.attention(plan, q, k, v, key_mask=mask, out=out)
    want, mag = plain(q, k, v, qo, ko, left, right, mask, 1 / math.sqrt(dim))
    got = out.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    err = (got - want).abs()
    tol = U[dtype] * (want.abs() + mag) + 1e-4 * mag + 2.0 ** -24
    bad = ok & (err > tol)
    assert not bad.any(), (int(bad.sum()), float((err - tol)[ok].max()), torch.nonzero(bad)[:4].tolist())
    return out


WINDOWS = [(-1, -1), (-1, 0), (400, 300), (63, 64), (0, 0), (-1, 5), (450, -1)]
HEADS = [(4, 2), (2, 2), (8, 2), (6, 2)]


@pytest.mark.parametrize("window", WINDOWS, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dim", [40, 64, 80, 96, 104, 128])
def test_long_and_short_sequences(ops, dim, heads, window):
    check(ops, [701, 1, 0, 130, 512], [701, 1, 0, 130, 512], *heads, dim, left=window[0], right=window[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [127, 128, 129, 255, 256, 257, 511, 575, 577, 640, 1100])
def test_lengths_around_the_tiles(ops, n, dtype):
    for dim in (64, 128):
        for right in (-1, 0):
            check(ops, [n], [n], 2, 2, dim, dtype=dtype, right=right)


@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (300, 200)], ids=str)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lq,lk", [([600, 30], [2500, 7]), ([700], [90]), ([520, 64], [0, 4000]), ([16, 2], [1500, 3000])], ids=str)
def test_fewer_or_more_queries_than_keys(ops, lq, lk, dim, window):
    """Cut keys in every form, and rows before the first key (which see nothing and are zero)."""
    check(ops, lq, lk, 4, 2, dim, left=window[0], right=window[1])


def test_one_long_sequence_is_cut(ops):
    """Few tiles over many keys: pieces of the 128- and the 256-row tiles are joined."""
    import torch
    for dim, lq, lk in ((64, 200, 9000), (128, 200, 9000), (128, 560, 9000)):
        g = torch.Generator(device="cuda").manual_seed(dim)
        q = torch.randn(lq, 4, dim, device="cuda", generator=g).bfloat16()
        k, v = (torch.randn(lk, 2, dim, device="cuda", generator=g).bfloat16() for _ in range(2))
        for left, right in ((-1, -1), (-1, 0), (5000, 0)):
            out = ops.attention(ops.attention_plan([0, lq], [0, lk], 4, 2, dim, left=left, right=right), q, k, v).double()
            want, mag = plain(q, k, v, [0, lq], [0, lk], left, right, None, 1 / math.sqrt(dim))
            assert ((out - want).abs() <= U["bf16"] * (want.abs() + mag) + 1e-4 * mag + 2.0 ** -24).all(), (dim, left, right)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (350, 250)], ids=str)
def test_key_mask(ops, window, dim, dtype):
    """Hidden keys (a whole sequence, whole steps, the first and last of others) hold NaN and infinities."""
    import torch
    lengths = [700, 200, 577]
    q, k, v = tensors(lengths, lengths, 4, 2, dim, dtype, 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    mask = torch.rand(len(k), device="cuda", generator=g) < 0.6
    mask[:150] = False
    mask[256:330] = False
    mask[690:700] = False
    mask[700:900] = False
    k[~mask] = float("nan")
    v[~mask] = float("inf")
    out = check(ops, lengths, lengths, 4, 2, dim, dtype=dtype, left=window[0], right=window[1], mask=mask, qkv=(q, k, v))
    assert not out[700:900].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window", [(-1, 0), (300, 200), (-1, -1)], ids=str)
def test_values_that_are_not_finite(ops, window, bad, dim):
    """A value that is not finite reaches the queries that see its key and no others, masked or not."""
    import torch
    lengths = [700, 520]
    q, k, v = tensors(lengths, lengths, 4, 2, dim, "bf16", 6)
    v[699, 0, 5] = bad
    v[698, 0, dim - 1] = -bad
    v[350, 1, 40] = bad
    v[700, 1, 7] = bad
    check(ops, lengths, lengths, 4, 2, dim, left=window[0], right=window[1], qkv=(q, k, v))
    mask = torch.ones(len(k), dtype=torch.bool, device="cuda")
    mask[350] = mask[10] = False
    k[10] = bad
    check(ops, lengths, lengths, 4, 2, dim, left=window[0], right=window[1], mask=mask, qkv=(q, k, v))


@pytest.mark.parametrize("dim", [64, 128])
def test_keys_that_are_not_numbers(ops, dim):
    """A NaN key makes the whole row of each query that sees it NaN, and nothing else."""
    lengths = [700, 520]
    q, k, v = tensors(lengths, lengths, 4, 2, dim, "bf16", 8)
    k[500, 0, 3] = float("nan")
    k[700 + 519, 1, 0] = float("nan")
    check(ops, lengths, lengths, 4, 2, dim, right=0, qkv=(q, k, v))
    check(ops, lengths, lengths, 4, 2, dim, left=200, right=100, qkv=(q, k, v))


@pytest.mark.parametrize("dim", [64, 128])
def test_rising_scores(ops, dim):
    """Scores of up to a few hundred, rising along the keys: the reference exponent moves often."""
    import torch
    lengths = [700, 577]
    q, k, v = tensors(lengths, lengths, 4, 2, dim, "bf16", 9)
    k = (k * torch.linspace(0.01, 12, len(k), device="cuda")[:, None, None]).bfloat16()
    qo = offsets(lengths + FILL)
    for right in (-1, 0):
        out = ops.attention(ops.attention_plan(qo, qo, 4, 2, dim, right=right), q, k, v).double()
        want, mag = plain(q, k, v, qo, qo, -1, right, None, 1 / math.sqrt(dim))
        # (scores of up to 500: their f32 error of 500 * 2^-22 in the exponent)
        assert ((out - want).abs() <= U["bf16"] * (want.abs() + mag) + 1e-3 * mag.clamp(min=0.1)).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_views_orders_and_streams(ops, dim):
    """Views of a joint projection, head-major tensors and another stream give the same bits."""
    import torch
    lengths = [700, 33] + FILL
    o = offsets(lengths)
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(o[-1], 8, dim, device="cuda", generator=g).bfloat16()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    plan = ops.attention_plan(o, o, 4, 2, dim, right=0)
    want = ops.attention(plan, q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(ops.attention(plan, q, k, v), want)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    out = torch.empty(4, o[-1], dim, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(ops.attention(plan, *hm, out=out), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention(plan, q, k, v)
    side.synchronize()
    assert torch.equal(other, want)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_far_apart(ops, dim):
    """Keys and queries more than 2^32 bytes from the tensors' start, in the large tiles."""
    import torch
    n, stride = 800 + sum(FILL), (1 << 32) // (2 * 640)
    stride -= stride % 8
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free GPU memory")
    g = torch.Generator(device="cuda").manual_seed(12)
    store = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((n, 2, dim), (stride, dim, 1))
    far.copy_(torch.randn(n, 2, dim, device="cuda", generator=g))
    near = far.contiguous()
    o = offsets(FILL + [800])
    for right in (-1, 0):
        plan = ops.attention_plan(o, o, 2, 2, dim, right=right)
        assert torch.equal(ops.attention(plan, far, far, far), ops.attention(plan, near, near, near))


def test_captured(ops):
    """A captured call of all three forms and their joins replays on new inputs."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(13)
    lq, lk = [1, 700, 2, 90] + FILL, [4000, 700, 70, 6000] + FILL
    plan = ops.attention_plan(offsets(lq), offsets(lk), 4, 2, 128)
    q = torch.randn(sum(lq), 4, 128, device="cuda", generator=g).bfloat16()
    k = torch.randn(sum(lk), 2, 128, device="cuda", generator=g).bfloat16()
    mask = torch.ones(sum(lk), dtype=torch.bool, device="cuda")
    out = torch.empty_like(q)
    ops.attention(plan, q, k, k, key_mask=mask, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention(plan, q, k, k, key_mask=mask, out=out)
    for _ in range(4):
        q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        k.copy_(torch.randn(k.shape, device="cuda", generator=g))
        mask.copy_(torch.rand(mask.shape, device="cuda", generator=g) < 0.7)
        want = ops.attention(plan, q, k, k, key_mask=mask)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dim,lengths", [(64, [33]), (128, [33]), (64, FILL), (128, FILL + [600])], ids=["few64", "few128", "rows", "tall"])
def test_scores_near_the_lowest(ops, dim, lengths):
    """All of a row's scores far below zero (down to -1e38): the highest still takes the whole weight."""
    import torch
    o = offsets(lengths)
    g = torch.Generator(device="cuda").manual_seed(14)
    q = torch.full((o[-1], 2, dim), 1e17, device="cuda").bfloat16()
    # key j of a sequence scores about -(j + 1) 1e34 x dim, up to the 40th
    place = torch.cat([torch.arange(n, device="cuda") for n in lengths]).clamp(max=40)
    k = (-(place + 1.0) * 1e17)[:, None, None].expand(-1, 2, dim).bfloat16()
    v = torch.randn(o[-1], 2, dim, device="cuda", generator=g).bfloat16()
    out = ops.attention(ops.attention_plan(o, o, 2, 2, dim), q, k, v, scale=1.0)
    first = torch.tensor(o[:-1], device="cuda").repeat_interleave(torch.tensor(lengths, device="cuda"))
    assert torch.equal(out, v[first])
