"""The recogniser's decoder over a paged cache, with norms of heads, drafted trees and steered logits: against plain
computations in 32 bits, with tolerances as in test_gpu_recognizer.py (0.2 a step of log-probability).  The plain form keeps
its keys and values as the cache's type does; a code that goes the other way, since the 16-bit key did, is one step off in
one channel of 64, less than the key's other roundings together."""
import math

import numpy as np
import pytest
from test_gpu_decode import quantised
from test_gpu_recognizer import attend, clips, rms, turn

pytestmark = pytest.mark.gpu


def make(**config):
    from scriptrs_amd.recognizer import Recognizer, RecognizerConfig
    return Recognizer(RecognizerConfig(encoder_blocks=2, **config))


def kept(x, kind):
    return quantised(x.bfloat16(), kind).to(x.device)


def plain_logits(r, encoded, tokens):
    """Logits [len(tokens), vocab] that each token of a transcript is chosen from."""
    import torch
    c, n = r.config, len(tokens)
    kv = c.kv_heads * r.dim
    x = r.embedding[torch.cat([tokens.new_full((1,), r.end), tokens[:-1]])].float()
    positions = torch.arange(n, device=x.device)
    for b in r.decoder:
        qkv = rms(x, b["norm"]) @ b["qkv"].float()
        q, k, v = (t.reshape(n, -1, r.dim) for t in qkv.split([c.width, kv, kv], 1))
        if c.head_norm:
            q, k = rms(q, b["head_q"]), rms(k, b["head_k"])
        k, v = kept(turn(k, positions), c.cache or "bf16"), kept(v, c.cache or "bf16")
        x = x + attend(turn(q, positions), k, v, True).reshape(n, -1) @ b["out"].float()
        q = (rms(x, b["norm_cross"]) @ b["q"].float()).view(n, c.heads, r.dim)
        k, v = (encoded.float() @ b["kv"].float()).view(-1, 2, c.heads, r.dim).unbind(1)
        x = x + attend(q, k, v).reshape(n, -1) @ b["cross_out"].float()
        x = x + torch.nn.functional.silu(rms(x, b["norm_ff"]) @ b["up"].float()) @ b["down"].float()
    return rms(x, r.decoder_norm) @ r.head.float()


@pytest.mark.parametrize("kind,head_norm", [("bf16", False), ("e4m3", True), ("int8", True), (None, True)])
def test_transcripts_score_as_they_read(kind, head_norm):
    """A transcript's score is the sum of its tokens' log-probabilities over its own pages, reordered with its beam."""
    import torch
    r, steps = make(cache=kind, head_norm=head_norm), 20
    frames, at = r.frames(*clips([16_000, 800, 48_000]))
    encoded = r.encode(frames, at)
    scores, tokens = r.decode(encoded, at, beams=4, steps=steps)
    assert torch.isfinite(scores).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    for s in range(3):
        for b in range(4):
            t = tokens[s, b].long()
            ended = torch.nonzero(t == r.end)
            n = int(ended[0]) + 1 if len(ended) else steps
            want = torch.log_softmax(plain_logits(r, encoded[at[s]:at[s + 1]], t[:n]), -1).gather(1, t[:n, None]).sum()
            assert abs(float(scores[s, b] - want)) < 0.2 * n, (s, b)
    r.close()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_drafted_trees_are_scored_as_their_branches(kind):
    import torch
    r = make(cache=kind, head_norm=True)
    frames, at = r.frames(*clips([16_000, 90_123]))
    encoded = r.encode(frames, at)
    parents = [-1, 0, 1, 0, 3, 4, -1, 6, 2, 8, 9, 9]
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, r.end, (2, len(parents)), device="cuda", generator=g, dtype=torch.int32)
    got = r.draft_logits(encoded, at, tokens, parents).float()
    for s in range(2):
        for i in range(len(parents)):
            branch, p = [i], parents[i]
            while p >= 0:
                branch.insert(0, p)
                p = parents[p]
            want = plain_logits(r, encoded[at[s]:at[s + 1]], tokens[s, branch].long())[-1]
            # (logits of deviation 2, off by up to 5% of it in the mean square)
            assert float((got[s, i] - want).pow(2).mean().sqrt()) < 0.1, (s, i)
    r.close()


def test_steered_beams():
    """Only allowed tokens, and none twice where repeating costs more than anything gives."""
    import torch
    r = make(cache="int8")
    frames, at = r.frames(*clips([16_000, 48_000]))
    encoded = r.encode(frames, at)
    words = torch.zeros(1, (r.config.vocab + 31) // 32, dtype=torch.int64)
    for t in range(0, r.end, 3):
        words[0, t // 32] |= 1 << t % 32
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).int().cuda()
    _, tokens = r.decode(encoded, at, beams=4, steps=16, allowed=words)
    assert (tokens % 3 == 0).all() and (tokens < r.end).all()
    _, tokens = r.decode(encoded, at, beams=4, steps=16, frequency=1000.0, allowed=words)
    for row in tokens.view(-1, 16).tolist():
        assert len(set(row)) == 16 and all(t % 3 == 0 for t in row)
    free, _ = r.decode(encoded, at, beams=4, steps=16)
    same, _ = r.decode(encoded, at, beams=4, steps=16, allowed=torch.full_like(words, -1))
    assert torch.equal(free, same)
    r.close()


def test_a_step_as_a_graph():
    """Head norms, cache write, attention and steered logits of one step captured together: replays of a growing
    cache, with eager calls between them, give what eager calls give."""
    import torch
    from scriptrs_amd import KvCache, ModelOps, RotaryTable
    ops = ModelOps()
    H, K, D, rows, vocab = 8, 2, 64, 6, 1025
    table = RotaryTable(D)
    g = torch.Generator(device="cuda").manual_seed(1)
    caches = [KvCache(rows * 4, 16, K, D, dtype="e4m3") for _ in range(2)]
    pages = torch.randperm(rows * 4, device="cuda", generator=g).int().view(rows, 4)
    plan = ops.cache_plan(np.arange(rows + 1), H, K, D)
    lengths = torch.ones(rows, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(rows, H + 2 * K, D, device="cuda", dtype=torch.bfloat16)
    head = torch.randn(H * D, vocab, device="cuda", generator=g).bfloat16() * 0.05
    said = torch.zeros(rows, 64, dtype=torch.int32, device="cuda")

    def step(cache):
        q, k = ops.norm_rotary(table, lengths - 1, qkv[:, :H], qkv[:, H:H + K])
        ops.cache_write(plan, cache, pages, lengths, k, qkv[:, H + K:])
        y = ops.cache_attention(plan, cache, pages, lengths, q)
        logits = y.reshape(rows, H * D) @ head
        return y, ops.adjust_logits(logits, history=said, lengths=lengths, repetition=1.3)
    step(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    caches[0].data.zero_()
    for n in range(1, 60):
        lengths.fill_(n)
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g))
        said[:, n - 1] = torch.randint(0, vocab, (rows,), device="cuda", generator=g).int()
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = step(caches[1])
        assert torch.equal(caches[0].data, caches[1].data) and all(torch.equal(a, b) for a, b in zip(got, want)), n
    ops.close()


def test_command(capsys, monkeypatch):
    from scriptrs_amd import recognizer as module
    monkeypatch.setattr("sys.argv", ["recognizer", "--clips", "3", "--steps", "4", "--cache", "int8", "--head-norm",
                                     "--repetition", "1.2"])
    module.main()
    out = capsys.readouterr().out
    assert out.count("encoder frames") == 2 and "clip 2: score" in out
    assert math.isfinite(float(out.split("clip 0: score ")[1].split(",")[0]))
