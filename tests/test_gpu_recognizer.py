"""The whole path of features, encoder and beam search against plain computations in 32 bits.

Tolerances: every sub-block rounds its normed input, projections, weights of the softmax and output
to bfloat16, about 6 roundings of at most 2^-9 of the value each, so a sub-block's part of the
residual is off by at most 1.2% and the sum of 2 x blocks of them, normed, by at most that
times their number in the mean square (3.5% for 4 blocks if they add like noise, 5% taken).  Logits of
deviation 2 are then off by up to 5% of it in the mean square: 0.1, and a step's log-probability by as
much; 0.2 a step is taken."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def recognizer():
    from scriptrs_amd.recognizer import Recognizer
    r = Recognizer()
    yield r
    r.close()


def rms(x, w):
    return x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w


def turn(x, positions):
    """Rotary positions of [rows, heads, dim], channel p with p + dim / 2."""
    import torch
    half = x.shape[-1] // 2
    angle = positions.double()[:, None] * 10_000.0 ** (-torch.arange(half, device=x.device).double() / half)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def attend(q, k, v, causal=False):
    import torch
    k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
    out = torch.empty_like(q)
    for h in range(q.shape[1]):
        x = q[:, h] @ k[:, h].T / math.sqrt(q.shape[2])
        if causal:
            x = x.masked_fill(torch.ones_like(x).triu(1).bool(), -math.inf)
        out[:, h] = torch.softmax(x, -1) @ v[:, h] if k.shape[0] else 0.0
    return out


def plain_encode(r, frames):
    import torch
    n, c = len(frames), r.config
    x = frames.float() @ r.encoder_in.float()
    positions = torch.arange(n, device=x.device)
    for b in r.encoder:
        q, k, v = (rms(x, b["norm"]) @ b["qkv"].float()).view(n, 3, c.heads, r.dim).unbind(1)
        x = x + attend(turn(q, positions), turn(k, positions), v).reshape(n, -1) @ b["out"].float()
        x = x + 0.5 * torch.nn.functional.silu(rms(x, b["norm_ff"]) @ b["up"].float()) @ b["down"].float()
    return rms(x, r.encoder_norm)


def plain_log_probs(r, encoded, tokens):
    """Log-probabilities [len(tokens), vocab] after each prefix of a transcript."""
    import torch
    c, n = r.config, len(tokens)
    kv = c.kv_heads * r.dim
    x = r.embedding[torch.cat([tokens.new_full((1,), r.end), tokens[:-1]])].float()
    positions = torch.arange(n, device=x.device)
    for b in r.decoder:
        qkv = rms(x, b["norm"]) @ b["qkv"].float()
        q, k, v = (t.reshape(n, -1, r.dim) for t in qkv.split([c.width, kv, kv], 1))
        x = x + attend(turn(q, positions), turn(k, positions), v, True).reshape(n, -1) @ b["out"].float()
        q = (rms(x, b["norm_cross"]) @ b["q"].float()).view(n, c.heads, r.dim)
        k, v = (encoded.float() @ b["kv"].float()).view(-1, 2, c.heads, r.dim).unbind(1)
        x = x + attend(q, k, v).reshape(n, -1) @ b["cross_out"].float()
        x = x + torch.nn.functional.silu(rms(x, b["norm_ff"]) @ b["up"].float()) @ b["down"].float()
    return torch.log_softmax(rms(x, r.decoder_norm) @ r.head.float(), -1)


def clips(lengths):
    import torch
    from scriptrs_amd.synth import sinusoids
    samples = np.concatenate([sinusoids(n, 3 + i) for i, n in enumerate(lengths)])
    return torch.from_numpy(samples).cuda(), np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


@pytest.mark.parametrize("lengths", [[160_000], [16_000, 800, 90_123, 1_300, 320_000]], ids=str)
def test_encoder(recognizer, lengths):
    r = recognizer
    frames, at = r.frames(*clips(lengths))
    got = r.encode(frames, at).float()
    assert at.tolist() == np.concatenate([[0], np.cumsum([(n // 160 + 1) // 8 for n in lengths])]).tolist()
    for a, b in zip(at[:-1], at[1:]):
        if b > a:
            want = plain_encode(r, frames[a:b])
            assert float((got[a:b] - want).norm() / want.norm()) < 0.05, (a, b)


@pytest.mark.parametrize("beams", [1, 4])
def test_transcripts_score_as_they_read(recognizer, beams):
    """A transcript's score is the sum of its tokens' log-probabilities: what its beam's cache
    held at each step was its own history."""
    import torch
    r, steps = recognizer, 12
    frames, at = r.frames(*clips([16_000, 800, 90_123, 48_000]))
    encoded = r.encode(frames, at)
    scores, tokens = r.decode(encoded, at, beams=beams, steps=steps)
    assert scores.shape == (4, beams) and tokens.shape == (4, beams, steps)
    assert torch.isfinite(scores).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    for s in range(4):
        for b in range(beams):
            t = tokens[s, b].long()
            ended = torch.nonzero(t == r.end)
            n = int(ended[0]) + 1 if len(ended) else steps
            assert (t[n:] == r.end).all()
            want = plain_log_probs(r, encoded[at[s]:at[s + 1]], t[:n]).gather(1, t[:n, None]).sum()
            assert abs(float(scores[s, b] - want)) < 0.2 * n, (s, b)


def test_greedy_follows_the_best_token(recognizer):
    """With one beam, each token is the most probable one within the logits' error."""
    import torch
    r = recognizer
    frames, at = r.frames(*clips([64_000]))
    encoded = r.encode(frames, at)
    _, tokens = r.decode(encoded, at, beams=1, steps=12)
    t = tokens[0, 0].long()
    ended = torch.nonzero(t == r.end)
    t = t[:int(ended[0]) + 1] if len(ended) else t
    probs = plain_log_probs(r, encoded, t)
    # (both the chosen one's and the best one's log-probability may be off by 0.2)
    assert (probs.gather(1, t[:, None])[:, 0] >= probs.amax(1) - 0.4).all()


def test_command(capsys, monkeypatch):
    from scriptrs_amd import recognizer as module
    monkeypatch.setattr("sys.argv", ["recognizer", "--clips", "3", "--steps", "4"])
    module.main()
    out = capsys.readouterr().out
    assert out.count("encoder frames") == 2 and "clip 2: score" in out
