"""A step of beam search over the range of its logits: rows far from zero, rows wholly at the type's lowest value, rows
near its highest.

total = score + log softmax(logits): with the row's maximum m taken off first, ((x - m) - log sum exp(x - m)) does not
depend on where the row lies.  The logits here lie on a grid that keeps x - m exact in f32, so the error is that of the
logarithm (1e-6, sums of exponentials in f32) and of the total's own rounding; the tolerance is twice each:
2e-6 + 4e-7 of the total."""
import math

import pytest

pytestmark = pytest.mark.gpu

VOCABS = [40, 1025, 2048, 3000, 20_000, 128_000]


@pytest.fixture(scope="module")
def ops():
    from scriptrs_amd import ModelOps
    m = ModelOps()
    yield m
    m.close()


def check(ops, logits, scores, end=-1):
    """Against 64 bits; log softmax with the maximum taken off first."""
    import torch
    B, W = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double()
    x = x - x.amax(1, keepdim=True)
    total = (scores.cpu().double().view(-1, 1) + (x - x.exp().sum(1, keepdim=True).log())).view(B, W * V)
    value, at = torch.sort(total, stable=True, dim=1, descending=True)
    value, at = value[:, :W], at[:, :W]
    got = ops.beam_select(logits, scores, end_token=end)
    err = (got[0].cpu().double() - value).abs()
    assert (err <= 2e-6 + 4e-7 * value.abs()).all(), float(err.max())
    assert torch.equal(got[1].cpu(), (at // V).int()) and torch.equal(got[2].cpu(), (at % V).int())


def rows_apart(streams, beams):
    """Scores a multiple of 1/512 apart within a stream."""
    import torch
    return (-3 - torch.arange(beams, device="cuda") / 512).repeat(streams, 1).contiguous()


@pytest.mark.parametrize("offset", [1e4, -1e4, 65_536.0, 1e6, -1e6])
@pytest.mark.parametrize("vocab", VOCABS)
def test_rows_far_from_zero(ops, vocab, offset):
    """Every beam's row is the same but for its order and its place: at 0 and at multiples of the offset."""
    import torch
    for streams, beams in ((1, 1), (2, 5), (1, 16)):
        g = torch.Generator(device="cuda").manual_seed(vocab + beams)
        row = (torch.randn(vocab, device="cuda", generator=g) * 8).round() / 8
        logits = torch.stack([row.roll(7 * w) + offset * (w % 3) / 2 for w in range(streams * beams)])
        check(ops, logits, rows_apart(streams, beams))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_rows_at_the_types_ends(ops, vocab, dtype):
    """A row wholly at the lowest value is even (log 1 / V each); where some tokens are at the highest, they share it."""
    import torch
    t = getattr(torch, dtype)
    low, high = torch.finfo(t).min, torch.finfo(t).max
    for streams, beams in ((2, 1), (1, 4), (1, 16)):
        scores = rows_apart(streams, beams)
        logits = torch.full((streams * beams, vocab), low, device="cuda", dtype=t)
        check(ops, logits, scores, end=3)
        logits[:, 5::7] = high
        check(ops, logits, scores, end=3)
        logits[:] = 0.0
        logits[:, vocab // 2:] = low
        logits[::2] = low
        check(ops, logits, scores)
        logits[:] = high
        logits[1::2, :9] = 0.0
        check(ops, logits, scores)


@pytest.mark.parametrize("vocab", VOCABS)
def test_even_rows_score_alike(ops, vocab):
    """Rows of equal logits have log(1 / V), wherever they lie: no row's totals are off against another's."""
    import torch
    at = torch.tensor([0.0, 1e4, -3e5, 1e7, 3e38, -3e38], device="cuda")
    got = ops.beam_select(at[:, None].repeat(1, vocab), torch.zeros(6, 1, device="cuda"))
    assert (got[0].view(-1) == got[0][0, 0]).all() and abs(float(got[0][0, 0]) + math.log(vocab)) <= 2e-6 + 4e-7 * math.log(vocab)
    assert (got[2] == 0).all()
