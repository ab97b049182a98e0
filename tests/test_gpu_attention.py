"""Attention over packed sequences against a plain computation in 64 bits.

The tolerance is the kernel's rounding, element by element: the output's own
rounding (half an ulp, u |o|, u = 2^-9 for bfloat16 and 2^-12 for float16,
doubled where it may round either way at a boundary), the weights' rounding to
the inputs' type before the product with v (u of each term: u sum p |v|), and
the f32 scores and exponentials (scores of up to about 30 with a relative error
below 2^-20: 1e-4 of each term)."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


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
    H, K, D = q.shape[1], k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    for s in range(len(qo) - 1):
        lq, lk = qo[s + 1] - qo[s], ko[s + 1] - ko[s]
        if lq == 0 or lk == 0:
            continue
        i = torch.arange(lq)[:, None] + lk - lq
        j = torch.arange(lk)[None, :]
        see = torch.ones(lq, lk, dtype=torch.bool)
        if left >= 0:
            see &= j >= i - left
        if right >= 0:
            see &= j <= i + right
        if mask is not None:
            see &= mask.cpu()[ko[s]:ko[s + 1]][None, :]
        for h in range(H):
            kk, vv = k[ko[s]:ko[s + 1], h * K // H], v[ko[s]:ko[s + 1], h * K // H]
            x = q[qo[s]:qo[s + 1], h] @ torch.where(see.any(0)[:, None], kk, 0.0).T * scale
            x = torch.where(see, x, -math.inf)
            top = x.amax(1, keepdim=True)
            p = torch.where(see, (x - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            finite = torch.isfinite(vv)
            r = p @ torch.where(finite, vv, 0.0)
            # what is not finite reaches exactly the queries that see it
            for a, b in torch.nonzero(~finite).tolist():
                r[see[:, a], b] += vv[a, b]
            out[qo[s]:qo[s + 1], h] = r
            mag[qo[s]:qo[s + 1], h] = p @ torch.where(finite, vv, 0.0).abs()
    return out, mag


def check(ops, lq, lk, heads, kv_heads, dim, dtype="bf16", left=-1, right=-1, mask=None, seed=0, spread=1.0, q=None,
          k=None, v=None, scale=None):
    import torch
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    qo, ko = offsets(lq), offsets(lk)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if q is None:
        q = (torch.randn(qo[-1], heads, dim, device="cuda", generator=g) * spread).to(t)
        k, v = (torch.randn(ko[-1], kv_heads, dim, device="cuda", generator=g).to(t) for _ in range(2))
    plan = ops.attention_plan(qo, ko, heads, kv_heads, dim, left=left, right=right)
    out = torch.full(q.shape, float("nan"), dtype=t, device="cuda")
    ops.attention(plan, q, k, v, key_mask=mask, scale=scale, out=out)
    want, mag = plain(q, k, v, qo, ko, left, right, mask, 1 / math.sqrt(dim) if scale is None else scale)
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    err = (got - want).abs()
    tol = U[dtype] * (want.abs() + mag) + 1e-4 * mag + 2.0 ** -24
    bad = ok & (err > tol)
    assert not bad.any(), (int(bad.sum()), float((err - tol)[ok].max()), torch.nonzero(bad)[:4].tolist())
    return out


LENGTHS = [[1], [63], [64], [65], [129], [0, 1, 0, 17, 128, 0], [200, 3, 77, 1, 131]]


@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (20, 5), (0, 0), (-1, 3), (7, -1)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_self_attention(ops, lengths, window):
    check(ops, lengths, lengths, 4, 2, 64, left=window[0], right=window[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 24, 32, 40, 64, 72, 80, 96, 104, 120, 128])
def test_head_dims(ops, dim, dtype):
    check(ops, [70, 5], [70, 5], 2, 1, dim, dtype=dtype)
    check(ops, [1, 3], [300, 5], 2, 1, dim, dtype=dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (8, 8), (32, 2), (71, 71)])
def test_grouped_heads(ops, heads, kv_heads):
    check(ops, [33, 2], [33, 90], heads, kv_heads, 64)
    check(ops, [150], [150], heads, kv_heads, 64, right=0)


@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (30, 2)])
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [1, 700, 33]), ([4, 0, 2], [513, 9, 0]), ([40, 3], [17, 2]),
                                   ([100, 20], [700, 19]), ([1], [5000]), ([130], [2100])], ids=str)
def test_fewer_or_more_queries_than_keys(ops, lq, lk, window):
    """Single tokens, cut keys, queries before the first key (rows that see nothing are zero)."""
    check(ops, lq, lk, 4, 2, 128, left=window[0], right=window[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lq,lk", [([90, 300], [90, 300]), ([2, 1], [700, 64]), ([1], [4000])], ids=str)
def test_key_mask(ops, lq, lk, dtype):
    """Hidden keys (a whole sequence among them) hold NaN and infinities."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    n = sum(lk)
    mask = torch.rand(n, device="cuda", generator=g) < 0.6
    mask[:lk[0]] &= torch.arange(lk[0], device="cuda") % 128 >= 70
    if len(lk) > 1:
        mask[lk[0]:] = mask[lk[0]:] if dtype == "bf16" else False
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    q = torch.randn(sum(lq), 4, 80, device="cuda", generator=g).to(t)
    k, v = (torch.randn(n, 2, 80, device="cuda", generator=g).to(t) for _ in range(2))
    for x, bad in ((k, float("nan")), (v, float("inf"))):
        x[~mask] = bad
    check(ops, lq, lk, 4, 2, 80, dtype=dtype, mask=mask, q=q, k=k, v=v)
    check(ops, lq, lk, 4, 2, 80, dtype=dtype, mask=mask, left=100, right=0, q=q, k=k, v=v)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lq,lk,left,right", [([200], [200], -1, 0), ([200], [200], 40, 3), ([3], [300], -1, 0),
                                              ([3, 9], [300, 40], 20, 0)])
def test_values_outside_a_window_reach_nothing(ops, lq, lk, left, right, bad, dtype):
    """A value that is not finite reaches the queries that see its key and no others."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    q = torch.randn(sum(lq), 2, 64, device="cuda", generator=g).to(t)
    k, v = (torch.randn(sum(lk), 1, 64, device="cuda", generator=g).to(t) for _ in range(2))
    v[lk[0] - 1, 0, 5] = bad
    v[lk[0] - 2, 0, 63] = -bad
    v[lk[0] // 2, 0, 40] = bad
    check(ops, lq, lk, 2, 1, 64, dtype=dtype, left=left, right=right, q=q, k=k, v=v)


def test_neighbours_and_rows_past_the_end_reach_nothing(ops):
    """NaN in the sequences around, in the rows after the last and between the heads."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(7)
    lengths = [70, 50, 9]
    big = torch.full((200, 3, 96), float("nan"), dtype=torch.bfloat16, device="cuda")
    for a, b in ((0, 70), (120, 129)):
        big[a:b, :2, :64] = torch.randn(b - a, 2, 64, device="cuda", generator=g).bfloat16()
    x = big[:129, :2, :64]
    o = offsets(lengths)
    out = ops.attention(ops.attention_plan(o, o, 2, 2, 64), x, x, x)
    assert torch.isnan(out[70:120]).all() and torch.isfinite(out[:70]).all() and torch.isfinite(out[120:]).all()
    few = ops.attention(ops.attention_plan([0, 1, 2, 3], o, 2, 2, 64), x[[0, 1, 2]], x, x)
    assert torch.isfinite(few[0]).all() and torch.isnan(few[1]).all() and torch.isfinite(few[2]).all()


def test_large_scores_and_rising_maximum(ops):
    """Scores up to several hundred, rising along the keys: the reference exponent moves often."""
    import torch
    for lq, lk in (([64], [700]), ([1], [3000])):
        g = torch.Generator(device="cuda").manual_seed(8)
        q = torch.randn(sum(lq), 2, 64, device="cuda", generator=g).bfloat16()
        k, v = (torch.randn(sum(lk), 2, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
        k = (k * torch.linspace(0.01, 8, sum(lk), device="cuda")[:, None, None]).bfloat16()
        out = ops.attention(ops.attention_plan(offsets(lq), offsets(lk), 2, 2, 64), q, k, v, scale=1.0)
        want, mag = plain(q, k, v, offsets(lq), offsets(lk), -1, -1, None, 1.0)
        # (scores of up to 500: their f32 error of 500 * 2^-22 in the exponent)
        assert ((out.cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + mag) + 1e-3 * mag.clamp(min=0.1)).all()


def test_strided_views_and_streams(ops):
    """Views of a joint projection, head-major tensors, a stream other than the current one."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(9)
    lengths = [37, 150, 1]
    o = offsets(lengths)
    x = torch.randn(o[-1], 4 + 2 * 2, 64, device="cuda", generator=g).bfloat16()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    want = check(ops, lengths, lengths, 4, 2, 64, right=0, q=q, k=k, v=v)
    plan = ops.attention_plan(o, o, 4, 2, 64, right=0)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    out = torch.empty(4, o[-1], 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(ops.attention(plan, *hm, out=out), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention(plan, q, k, v)
    side.synchronize()
    assert torch.equal(other, want)


def test_rows_far_apart(ops):
    """Keys more than 2^32 bytes from the tensor's start."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(10)
    n, stride = 1300, 1 << 22
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free GPU memory")
    store = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((n, 2, 64), (stride, 64, 1))
    far.copy_(torch.randn(n, 2, 64, device="cuda", generator=g))
    near = far.contiguous()
    for lq, lk, right in (([100, 1200], [100, 1200], 0), ([1, 2], [100, 1200], -1)):
        plan = ops.attention_plan(offsets(lq), offsets(lk), 2, 2, 64, right=right)
        q = near[:sum(lq)]
        assert torch.equal(ops.attention(plan, q, far, far), ops.attention(plan, q, near, near))


def test_captured(ops):
    """A captured call replays on new inputs."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    lq, lk = [1, 130, 2], [4000, 130, 70]
    plan = ops.attention_plan(offsets(lq), offsets(lk), 4, 2, 64)
    q = torch.randn(sum(lq), 4, 64, device="cuda", generator=g).bfloat16()
    k = torch.randn(sum(lk), 2, 64, device="cuda", generator=g).bfloat16()
    out = torch.empty_like(q)
    ops.attention(plan, q, k, k, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention(plan, q, k, k, out=out)
    for _ in range(4):
        q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        k.copy_(torch.randn(k.shape, device="cuda", generator=g))
        want = ops.attention(plan, q, k, k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_plans_reuse_memory_in_order(ops):
    """Plans made and freed while earlier calls are queued, on one stream and on two."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(3000, 2, 64, device="cuda", generator=g).bfloat16()
    cases, wants = [[i * 37 % 400 + 1 for i in range(j, j + 5)] for j in range(12)], []
    for lengths in cases:
        o = offsets(lengths)
        wants.append(ops.attention(ops.attention_plan(o, o, 2, 2, 64), x[:o[-1]], x[:o[-1]], x[:o[-1]]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for i, lengths in enumerate(cases):
        with torch.cuda.stream(side if i % 3 == 2 else torch.cuda.current_stream()):
            o = offsets(lengths)
            plan = ops.attention_plan(o, o, 2, 2, 64)
            got.append(ops.attention(plan, x[:o[-1]], x[:o[-1]], x[:o[-1]]))
            plan.close()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, wants))


def test_refusals(ops):
    import torch
    from scriptrs_amd import InvalidModelOutput, ModelOps
    o = [0, 10]
    x = torch.zeros(10, 2, 64, dtype=torch.bfloat16, device="cuda")
    plan = ops.attention_plan(o, o, 2, 2, 64)
    bad = [
        lambda: ops.attention(plan, x.float(), x, x),
        lambda: ops.attention(plan, x, x.half(), x),
        lambda: ops.attention(plan, x[:9], x, x),
        lambda: ops.attention(plan, x, x[:9], x),
        lambda: ops.attention(plan, x[:, :1], x, x),
        lambda: ops.attention(plan, x.cpu(), x, x),
        lambda: ops.attention(plan, x, x, x, out=x),
        lambda: ops.attention(plan, x, x, x, scale=0.0),
        lambda: ops.attention(plan, x, x, x, scale=float("nan")),
        lambda: ops.attention(plan, x, x, x, key_mask=torch.ones(9, dtype=torch.bool, device="cuda")),
        lambda: ops.attention(plan, x, x, x, key_mask=torch.ones(10, device="cuda")),
        # data or strides off 16 bytes
        lambda: ops.attention(plan, torch.zeros(10, 2, 72, dtype=torch.bfloat16, device="cuda")[..., 4:68], x, x),
        lambda: ops.attention(plan, torch.zeros(10, 2, 65, dtype=torch.bfloat16, device="cuda")[..., :64], x, x),
        lambda: ops.attention(plan, x.transpose(1, 2).contiguous().transpose(1, 2), x, x),
        lambda: ops.attention(plan, x, x, x, out=torch.zeros(10, 1, 64, dtype=torch.bfloat16, device="cuda").expand(10, 2, 64)),
        lambda: ops.attention_plan(o, [0, 5, 10], 2, 2, 64),
        lambda: ops.attention_plan(o, o, 3, 2, 64),
        lambda: ops.attention_plan(o, o, 2, 2, 60),
        lambda: ops.attention_plan(o, o, 2, 2, 136),
        lambda: ops.attention_plan([0, -1], o, 2, 2, 64),
        lambda: ops.attention_plan([-1, 3], o, 2, 2, 64),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(InvalidModelOutput):
            f()
            raise AssertionError(f"call {i} was not refused")
    other = ModelOps()
    with pytest.raises(InvalidModelOutput):
        other.attention(plan, x, x, x)
    other.close()
    plan.close()
    with pytest.raises(InvalidModelOutput):
        ops.attention(plan, x, x, x)
    empty = ops.attention_plan([0], [0], 2, 2, 64)
    assert ops.attention(empty, x[:0], x[:0], x[:0]).shape == (0, 2, 64)


@pytest.mark.parametrize("own_stream", [False, True])
def test_rows_of_no_sequence_are_zero(ops, own_stream):
    """Rows before the first sequence and past the last, on the call's stream; a refused call writes nothing."""
    import torch
    from scriptrs_amd.frontend import InvalidModelOutput
    g = torch.Generator(device="cuda").manual_seed(15)
    q, k, v = (torch.randn(40, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    out = torch.full_like(q, 7.0)
    stream = torch.cuda.Stream() if own_stream else None
    torch.cuda.synchronize()
    plan = ops.attention_plan([3, 20, 33], [5, 20, 40], 2, 2, 64, stream=stream)
    with pytest.raises(InvalidModelOutput):
        ops.attention(plan, q, k, v, scale=-1.0, stream=stream, out=out)
    torch.cuda.synchronize()
    assert torch.all(out == 7.0)
    assert ops.attention(plan, q, k, v, stream=stream, out=out) is out
    torch.cuda.synchronize()
    assert not out[:3].any() and not out[33:].any()
    cut = ops.attention_plan([0, 17, 30], [0, 15, 35], 2, 2, 64)
    assert torch.equal(out[3:33], ops.attention(cut, q[3:33], k[5:], v[5:]))
    none = ops.attention_plan([5], [5], 2, 2, 64)
    assert not ops.attention(none, q, k, v).any()


@pytest.mark.parametrize("dim", [64, 128])
def test_no_keys_at_all(ops, dim):
    """Without a key nothing of k and v is read, whatever their stride (C callers: null, stride 0)."""
    import ctypes

    import torch
    from scriptrs_amd import _lib
    o = offsets([200] * 50)
    plan = ops.attention_plan(o, [0] * 51, 8, 8, dim)
    q = torch.randn(o[-1], 8, dim, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    rows, none = 8 * dim, _lib.SfeHeads(None, 0, 0)
    args = [ctypes.byref(h) for h in (_lib.SfeHeads(q.data_ptr(), rows, dim), none, none)]
    to = _lib.SfeHeads(out.data_ptr(), rows, dim)
    rc = _lib.lib().sfe_attention(plan._handle, _lib.SFE_BF16, *args, None, 0.125, ctypes.byref(to),
                                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == _lib.SFE_OK, _lib.last_error()
    assert not out.any()


def test_plans_end_with_their_context():
    """After close() a plan's calls are refused, on the same operators opened again too; other plans are not touched."""
    import torch
    from scriptrs_amd import InvalidModelOutput, ModelOps
    own = ModelOps()
    x = torch.randn(200, 2, 64, device="cuda").bfloat16()
    plan, kept = (own.attention_plan([0, 80, 200], [0, 80, 200], 2, 2, 64) for _ in range(2))
    want = own.attention(plan, x, x, x)
    own.close()
    with pytest.raises(InvalidModelOutput, match="destroyed"):
        own.attention(plan, x, x, x)
    again = own.attention_plan([0, 80, 200], [0, 80, 200], 2, 2, 64)
    with pytest.raises(InvalidModelOutput, match="destroyed"):
        own.attention(plan, x, x, x)
    plan.close()
    assert torch.equal(own.attention(again, x, x, x), want)
    again.close()
    own.close()
    del kept


@pytest.mark.parametrize("heads,dim,dtype", [(1, 8, "f16"), (2, 64, "bf16"), (5, 104, "bf16")])
def test_rows_of_no_sequence_in_the_contexts_order(heads, dim, dtype):
    """Zeroed within the call: an operator queued after it on another stream reads zeros."""
    import torch
    from scriptrs_amd import ModelOps
    own = ModelOps()
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    first, last, rows = 700, 900, 30_000
    plan = own.attention_plan([first, last], [0, 50], heads, heads, dim)
    q = torch.randn(rows, heads, dim, device="cuda").to(t)
    k = torch.randn(50, heads, dim, device="cuda").to(t)
    out = torch.empty(rows, heads, dim + 8, dtype=t, device="cuda")
    block = torch.zeros(rows, heads * (dim + 8), dtype=t, device="cuda")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    want = own.attention(plan, q, k, k)
    for stream in (a, b):  # (the context's first calls on other streams wait on the host)
        own.residual_norm(block, block, stream=stream)
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        own.attention(plan, q, k, k, stream=a, out=out[..., :dim])
        read, _ = own.residual_norm(block, out.view(rows, -1), stream=b)
        torch.cuda.synchronize()
        read = read.view(out.shape)
        assert (read[..., dim:] == 7).all() and torch.equal(read[..., :dim], want)
        assert not read[:first, :, :dim].any() and not read[last:, :, :dim].any() and read[first:last, :, :dim].all(-1).all()
    plan.close()
    own.close()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lq,lk,heads", [([1], [10], 2), ([3, 1], [33, 90], 2), ([1], [2100], 2), ([126], [126], 2),
                                         ([40] * 40, [40] * 40, 8), ([700, 5], [700, 5], 8)], ids=str)
def test_one_value_for_all_keys(ops, lq, lk, heads, bad):
    """A value row broadcast over the keys (stride 0), and rows that overlap each other: what is not finite arrives as it
    is, though the rows past a step's last key read as values too."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(16)
    for dim in (64, 128):
        q = torch.randn(sum(lq), heads, dim, device="cuda", generator=g).bfloat16()
        k = torch.randn(sum(lk), heads, dim, device="cuda", generator=g).bfloat16()
        row = torch.randn(1, heads, dim, device="cuda", generator=g).bfloat16()
        row[0, 0, 5] = bad
        check(ops, lq, lk, heads, heads, dim, q=q, k=k, v=row.expand(sum(lk), heads, dim))
        # rows 8 channels apart of one line of numbers, the last 8 of them not finite: only the last key's row holds them
        line = torch.randn(8 * (sum(lk) - 1) + dim, device="cuda", generator=g).bfloat16()
        line[-8:] = bad
        check(ops, lq, lk, heads, 1, dim, q=q, k=k[:, :1], v=line.as_strided((sum(lk), 1, dim), (8, dim, 1)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk,heads", [([1], [10], 2), ([3, 1], [33, 900], 2), ([1], [5000], 2), ([126], [126], 2),
                                         ([40] * 40, [40] * 40, 8), ([700, 5], [700, 5], 8), ([2100], [2100], 8)], ids=str)
def test_large_values(ops, lq, lk, heads, dim):
    """Values of 1e36: a mean of them is no larger than they are, and so are the sums on the way to it (below 1e36 times
    a few hundred keys of weight up to 1)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(17)
    q, k, v = (torch.randn(n, heads, dim, device="cuda", generator=g).bfloat16() for n in (sum(lq), sum(lk), sum(lk)))
    small = check(ops, lq, lk, heads, heads, dim, q=q, k=k, v=v)
    big = 2.0 ** 120  # 1.3e36; a power of 2: the same bits but for the exponent
    plan = ops.attention_plan(offsets(lq), offsets(lk), heads, heads, dim)
    out = ops.attention(plan, q, k, (v.float() * big).bfloat16())
    assert torch.isfinite(out).all() and torch.equal(out.float() / big, small.float())
