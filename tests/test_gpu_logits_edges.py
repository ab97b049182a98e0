"""Steered logits where their kernel's forms meet, against 64 bits: vocabularies next to a span's end, and histories at
which the spans and the counts change."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_decode import U, gen, ops, steered, torch_dtype, within  # noqa: E402, F401


def close(got, want, dtype):
    """Values below 64: up to 6 roundings in f32, and the output's own."""
    import torch
    finite = torch.where(torch.isfinite(want), want.abs(), torch.zeros_like(want))
    within(got, want, U[dtype] * finite + 6 * 2.0 ** -24 * 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [*range(4088, 4098), 8183, 8185, 8186, 8189, 8190, 8191, 8192, 12_287])
def test_vocabularies_next_to_a_span_s_end(ops, vocab, dtype):  # noqa: F811
    """A row's last span has one token, a few or none, by where the row begins."""
    import torch
    rows, at = 3, 5
    wide = (3 * torch.randn(rows, vocab + 9, device="cuda", generator=gen(vocab))).to(torch_dtype(dtype))
    history = torch.randint(-2, vocab + 2, (rows, 400), device="cuda", generator=gen(1)).int()
    history[:, 300:] = vocab - 1 - history[:, 300:].abs() % 8
    for x in (wide[:, :vocab].contiguous(), wide[:, at:at + vocab]):
        close(ops.adjust_logits(x, history=history, repetition=1.25, frequency=0.03125),
              steered(x, history, None, 1.25, 0.0, 0.03125, None, None, None), dtype)
    out = torch.full_like(wide, 9.0)
    ops.adjust_logits(wide[:, at:at + vocab], history=history, presence=0.5, out=out[:, at:at + vocab])
    assert torch.equal(out[:, at:at + vocab], ops.adjust_logits(wide[:, at:at + vocab].contiguous(), history=history, presence=0.5))
    assert (out[:, :at] == 9.0).all() and (out[:, at + vocab:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("most", [4096, 4097, 65_535, 65_536])
@pytest.mark.parametrize("bias", [False, True])
def test_long_histories(ops, most, bias, dtype):  # noqa: F811
    """Spans of 4,096 and 8,192 tokens, counts of 16 and 32 bits: a row that says one token throughout beside rows
    whose tokens are the neighbours of it, and rows of any tokens over all spans."""
    import torch
    vocab, rows = 20_011, 4
    g = gen(most)
    logits = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(torch_dtype(dtype))
    history = torch.randint(-2, vocab + 2, (rows, most), device="cuda", generator=g).int()
    history[0] = 8191                            # one token, a span's last
    history[1, 1::2], history[1, ::2] = 8192, 8193
    history[2, :most - 1], history[2, most - 1] = 12_288, 12_289
    lengths = torch.tensor([most, most, most + 5, most - 1], dtype=torch.int32, device="cuda")
    args = dict(history=history, lengths=lengths, repetition=1.25, presence=0.5, frequency=2.0 ** -13,
                bias=torch.randn(vocab, device="cuda", generator=g) if bias else None, allowed=None, states=None)
    want = steered(logits, **args)
    assert want.abs().max() < 64
    close(ops.adjust_logits(logits, **args), want, dtype)


@pytest.mark.parametrize("each", [False, True])
def test_quotients_that_overflow(ops, each):  # noqa: F811
    """f32 logits over a repetition below one: infinite where the quotient is past f32's largest, and the quotient up to it."""
    import numpy as np
    import torch
    big = float(np.finfo(np.float32).max)
    values = [big, 3e38, 1.7014118e38, np.float32(big) / 2, 1e38, 1.0, 0.0, -1.0, -3e38, -big, float("inf"), -float("inf"), 1e-45, 2.0 ** -130]
    for repetition in (0.5, 0.3, 0.7, 0.9999999, 1e-20, 2.0 ** -126, 1.5, 1e20, 3e38):
        rep = np.float32(repetition)
        with np.errstate(over="ignore", invalid="ignore", under="ignore"):
            edge = np.float32(big) * rep  # (quotients next to the largest number)
            x = np.array(values + [np.nextafter(edge, s * np.float32(np.inf)) for s in (1, -1)] + [edge], np.float32)
            want = np.where(x > 0, x / rep, x * rep)
        logits = torch.from_numpy(np.stack([x, x])).cuda()
        history = torch.arange(len(x), dtype=torch.int32, device="cuda").repeat(2, 1)
        got = ops.adjust_logits(logits, history=history, repetition=torch.full((2,), repetition, device="cuda") if each else repetition)
        for row in got.cpu().numpy():
            same = (row == want) | (np.isnan(row) & np.isnan(want))
            # (a quotient is right to a step, below the normal numbers to the least step)
            finite = np.isfinite(row) & np.isfinite(want)
            err = np.abs(np.where(finite, row, 0.0).astype(np.float64) - np.where(finite, want, 0.0))
            close_by = finite & (err <= 2.0 ** -23 * np.abs(want) + 2.0 ** -149)
            assert (same | close_by).all(), (repetition, x[~(same | close_by)], row[~(same | close_by)], want[~(same | close_by)])
